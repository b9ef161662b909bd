"""The C ABI, the decoders and the test libraries build where torch is not installed (kaldi_decoder treats it
as optional); the torch binding of the operators over rows of logits is then left out."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIDE = """import sys
sys.modules["torch"] = None  # (find_spec then finds nothing)
"""


def _plan(env):
    return subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "kaldi-decoder_amd"), "--no-print-directory"],
                          capture_output=True, text=True, env=env)


def test_default_target_with_and_without_torch(tmp_path):
    env = dict(os.environ)
    env.pop("MAKEFLAGS", None)
    there = _plan(env)
    assert there.returncode == 0 and "_frames" in there.stdout and "torch/include" in there.stdout
    (tmp_path / "sitecustomize.py").write_text(HIDE)
    env["PYTHONPATH"] = str(tmp_path)
    gone = _plan(env)
    assert gone.returncode == 0, gone.stderr
    for lib in ("libkd_hip.so", "_kaldi_decoder", "libkd_hip_stress.so", "libkd_hip_jitter.so", "libkd_hip_jitter_full.so"):
        assert lib in gone.stdout, lib
    assert "Traceback" not in gone.stderr and "frames.cc" not in gone.stdout and "torch" in gone.stderr
    # asked for by name it is an error that says why
    one = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "kaldi-decoder_amd"), "frames"],
                         capture_output=True, text=True, env=env)
    assert one.returncode != 0 and "needs torch" in one.stderr


def test_build_imports_what_there_is(tmp_path):
    """What build() imports after the make, without torch: the package and the C ABI, not the binding."""
    (tmp_path / "sitecustomize.py").write_text(HIDE)
    code = ("import subprocess, sys\n"
            "subprocess.run = lambda *a, **k: None\n"
            "import __graft_entry__ as g\n"
            "g.build()\n"
            "assert 'kaldi_decoder.cabi' in sys.modules and 'kaldi_decoder.frames' not in sys.modules\n")
    env = dict(os.environ, PYTHONPATH=str(tmp_path))
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=env, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
