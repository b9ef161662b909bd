"""Host matrices with and without a gap between their rows: staged as one copy or row by row, decoded alike."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_rows_with_and_without_a_gap():
    from kaldi_decoder import cabi, synth
    V, T, B = 40, 30, 3
    g = synth.hlg_graph(V=V, n_words=200, n_hist=200, avg_succ=8, seed=4)
    G = cabi.Graph(g)
    dense = [synth.make_logprobs(T, V, i, peak=6.0, lexicon=g["lexicon"]) for i in range(B)]
    wide = [np.full((T, V + 7), np.nan, np.float32) for _ in range(B)]
    for w, d in zip(wide, dense):
        w[:, :V] = d
    results = []
    for mats, stride in ((dense, V), (wide, V + 7)):
        bt = cabi.Batch(G, max_batch=B, beam=10.0)
        bt.init_decoding()
        ptrs = bt._ptrs([m.ctypes.data for m in mats])
        for ready in (11, 12, T):  # (later rows of the same matrices: the copies start within them)
            rows = np.full(B, ready, np.int32)
            assert cabi.lib().kd_batch_advance(bt.h, ptrs, rows, None, V, stride, cabi.KD_MEM_HOST, -1) == 0
        results.append(bt.best_paths())
    import torch
    bt = cabi.Batch(G, max_batch=B, beam=10.0)
    bt.decode_tensor(torch.from_numpy(np.stack(dense)).cuda())
    results.append(bt.best_paths())
    for paths in results[1:]:
        for a, b in zip(results[0], paths):
            assert a.ok and b.ok and a.ilabel.tolist() == b.ilabel.tolist() and a.total_cost == b.total_cost
