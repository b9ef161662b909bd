// kaldi-decoder_amd/csrc/kd_frames.hip -- operators over a model's frame logits (include/kd_hip.h,
// "scores of given tokens" and "distillation"): kernels and their C entries.
//
// Everything here works on rows of V logits (f32, f16 or bf16), [batch][steps][V] with strides and
// optional lengths, the rows that the search itself is handed.  All of it is bound by the bytes of
// the logits, so the one rule is that a row is read once: a UNIT -- a whole row, or a segment of a
// long one -- is loaded into registers with 16-byte loads (NCH per lane, TPU = 64 or 256 threads)
// and every pass over it (maximum, sums, alternatives, gradient) runs over those registers.  A row
// of up to 8 KiB is one wave's, up to 32 KiB one workgroup's; a longer one is cut into segments
// whose partial results (maximum, sums, alternatives) a second kernel joins.
// Sums and statistics are f32; logits and gradients are rounded once, on the way in and out.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <string>

#include "kd_device.h"
#include "kd_hip.h"

namespace kd {
int SetError(int code, const std::string &msg);  // kd_api.hip
}

namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;
constexpr int kMaxTop = 64;       // alternatives a row
constexpr int kMaxSlots = 256;    // teacher's tokens a row
constexpr int kCap = 256;         // candidates a unit ranks (>= kMaxTop)
constexpr int64_t kMaxVocab = int64_t(1) << 24;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e+38f;

typedef uint32_t U4 __attribute__((ext_vector_type(4)));

// ---- element types ---------------------------------------------------------------------------
// kFill: what stands in for columns behind a row's end, -inf: it adds nothing to any sum, is no
// maximum and no alternative.
struct F32 {
  typedef float Store;
  typedef U4 Vec __attribute__((aligned(4)));
  static constexpr int kVec = 4;
  static constexpr uint32_t kFill = 0xff800000u;
  static __device__ float Get(const U4 &r, int j) { return __uint_as_float(r[j]); }
  static __device__ float Load(const Store *p) { return *p; }
  static __device__ Store Round(float v) { return v; }
  static __device__ U4 Pack(const float *v) {
    return U4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  }
};
template <class H, uint32_t FILL>
struct Half {
  typedef H Store;
  typedef U4 Vec __attribute__((aligned(2)));
  static constexpr int kVec = 8;
  static constexpr uint32_t kFill = FILL;
  static __device__ float Load(const Store *p) { return static_cast<float>(*p); }
  static __device__ Store Round(float v) { return static_cast<H>(v); }
  static __device__ U4 Pack(const float *v) {
    U4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      typedef H H2 __attribute__((ext_vector_type(2)));
      r[i] = __builtin_bit_cast(uint32_t, H2{static_cast<H>(v[2 * i]), static_cast<H>(v[2 * i + 1])});
    }
    return r;
  }
};
struct F16 : Half<_Float16, 0xfc00fc00u> {
  static __device__ float Get(const U4 &r, int j) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(r[j >> 1] >> (16 * (j & 1)))));
  }
};
struct BF16 : Half<__bf16, 0xff80ff80u> {
  static __device__ float Get(const U4 &r, int j) {
    return __uint_as_float((j & 1) ? (r[j >> 1] & 0xffff0000u) : (r[j >> 1] << 16));
  }
};

// ---- rows and units --------------------------------------------------------------------------
struct Rows {
  const void *x;           // logits
  const int32_t *lengths;  // [batch] valid rows, or null
  int64_t batch_stride, row_stride;
  uint32_t rows, steps;    // rows = batch * steps
  int32_t vocab;
  int32_t seg_len, nseg;   // a row's segments: [i * seg_len, min(vocab, (i + 1) * seg_len))
};

struct Unit {
  uint32_t row;
  int seg, lo, n;  // columns [lo, lo + n)
  int64_t b, t;
  bool skip;       // at or behind its utterance's length
};

// Unit `u`.  Its values are the same in all lanes of a wave.
__device__ inline Unit GetUnit(const Rows &r, uint32_t u) {
  Unit o;
  o.row = r.nseg == 1 ? u : u / static_cast<uint32_t>(r.nseg);
  o.seg = r.nseg == 1 ? 0 : static_cast<int>(u - o.row * static_cast<uint32_t>(r.nseg));
  o.lo = o.seg * r.seg_len;
  o.n = min(r.seg_len, r.vocab - o.lo);
  const uint32_t b = r.steps == r.rows ? 0u : o.row / r.steps;
  o.b = b;
  o.t = o.row - b * r.steps;
  o.skip = r.lengths && o.t >= r.lengths[b];
  return o;
}

template <class T>
__device__ inline const typename T::Store *RowPtr(const void *x, int64_t batch_stride, int64_t row_stride,
                                                  const Unit &u) {
  return static_cast<const typename T::Store *>(x) + u.b * batch_stride + u.t * row_stride;
}

// Lane `tid` of a unit holds columns [(c * TPU + tid) * kVec, + kVec) in r[c]: consecutive lanes
// load consecutive 16 bytes.  (Rows need no alignment beyond their element's: the loads are marked
// so and stay 16 bytes wide.)
template <class T, int NCH, int TPU>
__device__ inline void LoadUnit(const typename T::Store *p, int n, int tid, U4 (&r)[NCH]) {
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int e = (c * TPU + tid) * T::kVec;
    if (e + T::kVec <= n) {
      r[c] = *reinterpret_cast<const typename T::Vec *>(p + e);
    } else {
      r[c] = U4{T::kFill, T::kFill, T::kFill, T::kFill};
      if (e < n) {  // the row's end: at most kVec - 1 columns, one lane
        for (int j = 0; j < T::kVec - 1; ++j) {
          if (e + j >= n) break;
          if (T::kVec == 4) {
            const uint32_t v = __builtin_bit_cast(uint32_t, static_cast<float>(p[e + j]));
            if (j == 0) r[c][0] = v;
            if (j == 1) r[c][1] = v;
            if (j == 2) r[c][2] = v;
          } else {
            const uint32_t v = reinterpret_cast<const uint16_t *>(p)[e + j];
            const uint32_t old = j < 2 ? r[c][0] : j < 4 ? r[c][1] : j < 6 ? r[c][2] : r[c][3];
            const uint32_t now = (j & 1) ? (old & 0xffffu) | v << 16 : (old & 0xffff0000u) | v;
            if (j < 2) r[c][0] = now;
            else if (j < 4) r[c][1] = now;
            else if (j < 6) r[c][2] = now;
            else r[c][3] = now;
          }
        }
      }
    }
  }
}

// ---- reductions over a unit --------------------------------------------------------------------
// Wave level: five DPP steps inside rows of 16, then across them (lane 63 has the whole).
template <int CTRL, int ROW_MASK>
__device__ inline float Dpp(float identity, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(identity), __float_as_int(v), CTRL, ROW_MASK, 0xf,
                                                    false));
}
template <class OP>
__device__ inline float WaveReduce(float v, float identity, OP op) {
  v = op(v, Dpp<0x111, 0xf>(identity, v));  // row_shr:1
  v = op(v, Dpp<0x112, 0xf>(identity, v));
  v = op(v, Dpp<0x114, 0xf>(identity, v));
  v = op(v, Dpp<0x118, 0xf>(identity, v));
  v = op(v, Dpp<0x142, 0xa>(identity, v));  // row_bcast:15
  v = op(v, Dpp<0x143, 0xc>(identity, v));  // row_bcast:31
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ inline float WaveMax(float v) {
  return WaveReduce(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline float WaveSum(float v) {
  return WaveReduce(v, 0.0f, [](float a, float b) { return a + b; });
}

// A unit's scratch in LDS: of one wave (TPU 64, never synchronised with the others) or of the
// whole workgroup.
struct Scratch {
  float red[kWaves];
  int ired[kWaves];
  int count;
  float group_max[kBlock];
  float cand_v[kCap];
  int cand_i[kCap];
};

template <int TPU>
__device__ inline void UnitSync() {
  if (TPU > 64) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// (two barriers: `red` may be reused at once)
template <int TPU>
__device__ inline float UnitMax(float v, float *red) {
  v = WaveMax(v);
  if (TPU == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  return v;
}
template <int TPU>
__device__ inline float UnitSum(float v, float *red) {
  v = WaveSum(v);
  if (TPU == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (red[0] + red[1]) + (red[2] + red[3]);
  __syncthreads();
  return v;
}
// Sum over the unit of counts that every lane of a wave already agrees on.
template <int TPU>
__device__ inline int UnitCount(int wave_count, int *red) {
  if (TPU == 64) return wave_count;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = wave_count;
  __syncthreads();
  const int v = (red[0] + red[1]) + (red[2] + red[3]);
  __syncthreads();
  return v;
}
__device__ inline int Popc(uint64_t m) { return __popcll(m); }

// ---- the K largest -------------------------------------------------------------------------------
// Order: larger value first, then lower column.  -inf and NaN are no candidates.
//
// 1. A threshold: the K-th largest of the maxima of groups of a unit's elements (64 or 256 groups,
//    K <= 64 of them): at least K elements reach it, and of data in no particular order few more.
// 2. The elements that reach it are collected in LDS.  Where they are more than the list holds
//    (many equal values, or most of the large ones in few groups) the K-th element itself is found
//    by bisection, its value bit by bit and then, among equals, its column: exactly K are left.
// 3. Each candidate's place is the number of candidates ahead of it.

// A whole number that orders as the value does (-0 and +0 alike).
__device__ inline uint32_t OrderKey(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ inline float KeyValue(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// The k-th largest of 64 * G values of a wave (1 <= k <= 64 * G).
template <int G>
__device__ inline float KthLargest(const float (&v)[G], int k) {
  uint32_t key[G];
#pragma unroll
  for (int g = 0; g < G; ++g) key[g] = OrderKey(v[g]);
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = t | (1u << bit);
    int n = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) n += Popc(__ballot(key[g] >= c));
    if (n >= k) {
      t = c;
      if (n == k) break;
    }
  }
  // (broken off: every value from t upwards is among the k largest; t need not be one of them)
  return KeyValue(t);
}

// What a selection reads, as f(value, column) with all lanes of a wave in step: a unit's registers,
template <class T, int NCH, int TPU>
struct RegSource {
  const U4 (&r)[NCH];
  int lo, tid;
  template <class F>
  __device__ void Each(F f) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
#pragma unroll
      for (int j = 0; j < T::kVec; ++j) f(T::Get(r[c], j), lo + (c * TPU + tid) * T::kVec + j);
    }
  }
};
// the same unit from memory (for the bisection, which is rare: over the registers it would hold
// every unit's kernel to a copy of its code and theirs),
template <class T, int TPU>
struct MemSource {
  static constexpr int kLowBit = sizeof(typename T::Store) == 4 ? 0 : 13;  // an f16's or bf16's lower bits are 0
  const typename T::Store *p;
  int lo, n, tid;
  template <class F>
  __device__ void Each(F f) const {
    for (int base = 0; base < n; base += TPU) {
      const int k = base + tid;
      f(k < n ? T::Load(p + k) : -INFINITY, lo + k);
    }
  }
};
// or a list in memory (the alternatives of a row's segments).
struct ListSource {
  static constexpr int kLowBit = 0;
  const float *v;
  const int32_t *i;
  int n, tid;
  template <class F>
  __device__ void Each(F f) const {
    for (int base = 0; base < n; base += kBlock) {
      const int k = base + tid;
      f(k < n ? v[k] : -INFINITY, k < n ? i[k] : 0);
    }
  }
};

// Collects the elements that `pred` holds for; their number (all of them, kept or not).
template <int TPU, class SRC, class PRED>
__device__ inline int Collect(const SRC &src, Scratch &s, PRED pred) {
  const int lane = threadIdx.x & 63;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  int base = 0;
  if (TPU > 64) {
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
  }
  src.Each([&](float v, int i) {
    const bool mine = pred(v, i);
    const uint64_t m = __ballot(mine);
    if (m) {
      int at = base;
      if (TPU > 64) {
        int got = 0;
        if (lane == 0) got = atomicAdd(&s.count, Popc(m));
        at = __builtin_amdgcn_readfirstlane(got);
      }
      const int pos = at + Popc(m & below);
      if (mine && pos < kCap) {
        s.cand_v[pos] = v;
        s.cand_i[pos] = i;
      }
      base += Popc(m);
    }
  });
  UnitSync<TPU>();
  if (TPU > 64) {
    base = s.count;
    __syncthreads();
  }
  return base;
}

// The k-th element itself (value and column), among those that reach `floor_v`; at least k do.
template <int TPU, class SRC>
__device__ __noinline__ void KthElement(const SRC src, Scratch &s, float floor_v, int k, float *kv, int *ki) {
  uint32_t t = 0;
  for (int bit = 31; bit >= SRC::kLowBit; --bit) {
    const uint32_t c = t | (1u << bit);
    int n = 0;
    src.Each([&](float v, int) { n += Popc(__ballot(v >= floor_v && OrderKey(v) >= c)); });
    if (UnitCount<TPU>(n, s.ired) >= k) t = c;
  }
  const float val = KeyValue(t);
  int above = 0;
  src.Each([&](float v, int) { above += Popc(__ballot(v > val)); });
  const int need = k - UnitCount<TPU>(above, s.ired);  // of the equals, the first `need` columns
  int col = 0;  // (the largest column that fewer than `need` equals are in front of; columns < 2^24)
  for (int bit = 23; bit >= 0; --bit) {
    const int c = col | (1 << bit);
    int n = 0;
    src.Each([&](float v, int i) { n += Popc(__ballot(v == val && i < c)); });
    if (UnitCount<TPU>(n, s.ired) < need) col = c;
  }
  *kv = val;
  *ki = col;
}

// Puts the unit's K largest elements in order and hands (place, value, column) to `out`, once per
// place from some lane; places without an element get (-inf, -1).  `threshold`: at least k of the
// unit's elements reach it, or it is -inf.
template <int TPU, class SRC, class MEM, class OUT>
__device__ inline void SelectTop(const SRC &src, const MEM &mem, Scratch &s, float threshold, int k, OUT out) {
  const int tid = TPU == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const float floor_v = fmaxf(threshold, kLowest);  // (-inf is no alternative)
  int n = Collect<TPU>(src, s, [=](float v, int) { return v >= floor_v; });
  if (n > kCap) {
    float kv;
    int ki;
    KthElement<TPU>(mem, s, floor_v, k, &kv, &ki);
    n = Collect<TPU>(mem, s, [=](float v, int i) { return v > kv || (v == kv && i <= ki); });
    n = min(n, kCap);
  }
  for (int a = tid; a < n; a += TPU) {
    const float v = s.cand_v[a];
    const int i = s.cand_i[a];
    int place = 0;
    for (int b = 0; b < n; ++b) {
      const float w = s.cand_v[b];
      place += (w > v || (w == v && s.cand_i[b] < i)) ? 1 : 0;
    }
    if (place < k) out(place, v, i);
  }
  for (int a = n + tid; a < k; a += TPU) out(a, -INFINITY, -1);
}

// ---- scores ------------------------------------------------------------------------------------

struct Partial {  // a segment's part of a row's statistics: sums relative to its own maximum
  float m, s0, s1, pad;
};

struct ScoresArgs {
  Rows r;
  const void *tokens;  // int32 or int64 [rows], or null
  int32_t token64;
  int32_t k;           // alternatives
  float k2;            // log2(e) / temperature: e_j = exp2((x_j - m) * k2)
  float *logp, *entropy, *stats, *top_v;
  int32_t *top_i;
  Partial *part;       // split rows: [rows][nseg], and [rows][nseg][k] alternatives
  float *part_v;
  int32_t *part_i;
};

__device__ inline int64_t Token(const ScoresArgs &a, uint32_t row) {
  return a.token64 ? static_cast<const int64_t *>(a.tokens)[row] : static_cast<const int32_t *>(a.tokens)[row];
}

// A row's statistics are its maximum m and s = sum e_j.  (Not log s: 1 / s is what the gradient
// multiplies by, and a rounded log s of 10 would cost it 3 bits.)  A row without a finite value has
// m = -inf and s = 0; what is taken relative to its maximum is then taken relative to Base(m) = 0.
__device__ inline float Base(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ inline float LogSum(float s0) { return s0 == 0.0f ? 0.0f : logf(s0); }
// H = ls - sum e (x - m) / s: both terms are at least 0, nothing cancels.
__device__ inline float Entropy(float s0, float s1) { return s0 == 0.0f ? 0.0f : logf(s0) - s1 / s0; }

template <class T>
__device__ inline void WriteRowScores(const ScoresArgs &a, const Unit &u, const typename T::Store *x, float m,
                                      float s0, float s1) {
  const float ls = LogSum(s0);
  if (a.tokens) {
    const int64_t tok = Token(a, u.row);
    a.logp[u.row] = tok >= 0 && tok < a.r.vocab ? (T::Load(x + tok) - Base(m)) - ls : 0.0f;
  }
  a.entropy[u.row] = Entropy(s0, s1);
  a.stats[2 * static_cast<size_t>(u.row)] = m;
  a.stats[2 * static_cast<size_t>(u.row) + 1] = s0;
}

// Rows that are not read: zeros, and no alternatives.
template <int TPU>
__device__ inline void WriteRowNothing(const ScoresArgs &a, uint32_t row, int tid) {
  if (tid == 0) {
    if (a.tokens) a.logp[row] = 0.0f;
    a.entropy[row] = 0.0f;
    a.stats[2 * static_cast<size_t>(row)] = 0.0f;
    a.stats[2 * static_cast<size_t>(row) + 1] = 0.0f;
  }
  for (int i = tid; i < a.k; i += TPU) {
    a.top_v[static_cast<size_t>(row) * a.k + i] = -INFINITY;
    a.top_i[static_cast<size_t>(row) * a.k + i] = -1;
  }
}

struct TopWriter {
  float *v;
  int32_t *i;
  float base, ls;
  bool nan;  // the row's sum is NaN (NaN or +inf among its logits): no alternatives
  __device__ void operator()(int place, float val, int col) const {
    v[place] = nan ? ls : col < 0 ? -INFINITY : (val - base) - ls;
    i[place] = nan ? -1 : col;
  }
};

template <class T, int NCH, int TPU, bool SPLIT, bool ENT, bool TOP>
__global__ __launch_bounds__(kBlock) void ScoresKernel(const ScoresArgs a) {
  constexpr int kUnits = kBlock / TPU;
  __shared__ Scratch scratch[TOP || TPU > 64 ? kUnits : 1];
  const int tid = TPU == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const int which = TPU == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const uint32_t unit = blockIdx.x * kUnits + which;
  if (TPU == 64 && unit >= a.r.rows * static_cast<uint32_t>(a.r.nseg)) return;
  Scratch &s = scratch[TOP || TPU > 64 ? which : 0];
  const Unit u = GetUnit(a.r, unit);
  if (u.skip) {
    if (!SPLIT) WriteRowNothing<TPU>(a, u.row, tid);
    return;  // (split: the joining kernel writes, and reads no part of such a row)
  }
  const typename T::Store *x = RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u);
  U4 r[NCH];
  LoadUnit<T, NCH, TPU>(x + u.lo, u.n, tid, r);

  // the maxima of four groups of a lane's elements, and of all of them
  float gm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int j = 0; j < T::kVec; ++j) gm[j & 3] = fmaxf(gm[j & 3], T::Get(r[c], j));
  const float lane_max = fmaxf(fmaxf(gm[0], gm[1]), fmaxf(gm[2], gm[3]));
  if (TOP && TPU > 64) s.group_max[tid] = lane_max;
  const float m = UnitMax<TPU>(lane_max, s.red);
  const float base = Base(m);

  float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
#pragma unroll
    for (int j = 0; j < T::kVec; ++j) {
      const float d = T::Get(r[c], j) - base;
      const float e = __builtin_amdgcn_exp2f(d * a.k2);
      s0 += e;
      // (d is -inf for a masked column: 0 * -inf would be NaN)
      if (ENT) s1 = fmaf(e, fmaxf(d, kLowest), s1);
    }
  }
  s0 = UnitSum<TPU>(s0, s.red);
  if (ENT) s1 = UnitSum<TPU>(s1, s.red);

  if (SPLIT) {
    if (tid == 0) a.part[unit] = Partial{m, s0, s1, 0.0f};
  } else if (tid == 0) {
    WriteRowScores<T>(a, u, x, m, s0, s1);
  }
  if (TOP) {
    float threshold;
    if (TPU > 64) {
      const float g[4] = {s.group_max[tid & 63], s.group_max[64 + (tid & 63)], s.group_max[128 + (tid & 63)],
                          s.group_max[192 + (tid & 63)]};
      threshold = KthLargest<4>(g, a.k);
    } else if (a.k > 16) {
      threshold = KthLargest<4>(gm, a.k);
    } else {
      const float g[1] = {lane_max};
      threshold = KthLargest<1>(g, a.k);
    }
    const RegSource<T, NCH, TPU> src{r, u.lo, tid};
    const MemSource<T, TPU> mem{x + u.lo, u.lo, u.n, tid};
    const size_t at = (SPLIT ? static_cast<size_t>(unit) : static_cast<size_t>(u.row)) * a.k;
    if (SPLIT) {
      float *pv = a.part_v + at;
      int32_t *pi = a.part_i + at;
      SelectTop<TPU>(src, mem, s, threshold, a.k, [=](int place, float v, int i) {
        pv[place] = v;
        pi[place] = i;
      });
    } else {
      const float ls = LogSum(s0);
      SelectTop<TPU>(src, mem, s, threshold, a.k, TopWriter{a.top_v + at, a.top_i + at, base, ls, isnan(ls)});
    }
  }
}

// A row's statistics from its segments' (the whole workgroup; `red` is free again on return).
__device__ inline void JoinPartials(const Partial *part, int nseg, float k2, float *red, float *m_out, float *s0_out,
                                    float *s1_out) {
  float m = -INFINITY;
  for (int i = threadIdx.x; i < nseg; i += kBlock) m = fmaxf(m, part[i].m);
  m = UnitMax<kBlock>(m, red);
  const float base = Base(m);
  float s0 = 0.0f, s1 = 0.0f;
  for (int i = threadIdx.x; i < nseg; i += kBlock) {
    const Partial p = part[i];
    const float d = Base(p.m) - base, f = __builtin_amdgcn_exp2f(d * k2);
    // (a segment that adds nothing may have any maximum: its products are not formed)
    if (f != 0.0f && p.s0 != 0.0f) {
      s0 = fmaf(f, p.s0, s0);
      s1 += f * fmaf(d, p.s0, p.s1);
    }
  }
  *m_out = m;
  *s0_out = UnitSum<kBlock>(s0, red);
  *s1_out = UnitSum<kBlock>(s1, red);
}

template <class T, bool TOP>
__global__ __launch_bounds__(kBlock) void ScoresJoinKernel(const ScoresArgs a) {
  __shared__ Scratch s;
  const int tid = threadIdx.x;
  Unit u = GetUnit(a.r, blockIdx.x * static_cast<uint32_t>(a.r.nseg));
  if (u.skip) {
    WriteRowNothing<kBlock>(a, u.row, tid);
    return;
  }
  const int nseg = a.r.nseg;
  float m, s0, s1;
  JoinPartials(a.part + static_cast<size_t>(u.row) * nseg, nseg, a.k2, s.red, &m, &s0, &s1);
  const typename T::Store *x = RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u);
  if (tid == 0) WriteRowScores<T>(a, u, x, m, s0, s1);
  if (TOP) {
    const size_t n = static_cast<size_t>(nseg) * a.k;
    const ListSource src{a.part_v + u.row * n, a.part_i + u.row * n, static_cast<int>(n), tid};
    float mine = -INFINITY;
    src.Each([&](float v, int) { mine = fmaxf(mine, v); });
    s.group_max[tid] = mine;
    __syncthreads();
    const float g[4] = {s.group_max[tid & 63], s.group_max[64 + (tid & 63)], s.group_max[128 + (tid & 63)],
                        s.group_max[192 + (tid & 63)]};
    const float threshold = KthLargest<4>(g, a.k);
    const float ls = LogSum(s0);
    SelectTop<kBlock>(src, src, s, threshold, a.k,
                      TopWriter{a.top_v + static_cast<size_t>(u.row) * a.k, a.top_i + static_cast<size_t>(u.row) * a.k,
                                Base(m), ls, isnan(ls)});
  }
}

// ---- gradients -----------------------------------------------------------------------------------

struct GradOut {
  void *dx;
  int64_t batch_stride, row_stride;
};

// Writes f(value, column) for a unit's elements; a lane's columns as in LoadUnit.
template <class T, int NCH, int TPU, class F>
__device__ inline void StoreUnit(typename T::Store *p, int n, int tid, const U4 (&r)[NCH], F f) {
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int e = (c * TPU + tid) * T::kVec;
    if (e < n) {
      float g[T::kVec];
#pragma unroll
      for (int j = 0; j < T::kVec; ++j) g[j] = f(T::Get(r[c], j), e + j);
      if (e + T::kVec <= n) {
        *reinterpret_cast<typename T::Vec *>(p + e) = T::Pack(g);
      } else {
#pragma unroll
        for (int j = 0; j < T::kVec; ++j)
          if (e + j < n) p[e + j] = T::Round(g[j]);
      }
    }
  }
}
template <class T, int NCH, int TPU>
__device__ inline void StoreZeros(typename T::Store *p, int n, int tid) {
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int e = (c * TPU + tid) * T::kVec;
    if (e + T::kVec <= n) {
      *reinterpret_cast<typename T::Vec *>(p + e) = U4{0, 0, 0, 0};
    } else {
      for (int j = 0; j < T::kVec - 1; ++j)
        if (e + j < n) p[e + j] = T::Round(0.0f);
    }
  }
}

struct ScoresGradArgs {
  Rows r;
  GradOut o;
  const void *tokens;
  int32_t token64;
  const float *stats, *entropy;    // of the forward pass
  const float *g_logp, *g_entropy; // upstream, [rows] each, or null (0)
};

// dx_j = g_logp ([j = token] - p_j) - g_H p_j (log p_j + H) = p_j (A - g_H log p_j) + g_logp [j = token]
// with A = -g_logp - g_H H.
template <class T, int NCH, int TPU>
__global__ __launch_bounds__(kBlock) void ScoresGradKernel(const ScoresGradArgs a) {
  constexpr int kUnits = kBlock / TPU;
  const int tid = TPU == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const int which = TPU == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const uint32_t unit = blockIdx.x * kUnits + which;
  if (unit >= a.r.rows * static_cast<uint32_t>(a.r.nseg)) return;
  const Unit u = GetUnit(a.r, unit);
  typename T::Store *dx =
      const_cast<typename T::Store *>(RowPtr<T>(a.o.dx, a.o.batch_stride, a.o.row_stride, u)) + u.lo;
  const float m = a.stats[2 * static_cast<size_t>(u.row)], s0 = a.stats[2 * static_cast<size_t>(u.row) + 1];
  if (u.skip || s0 == 0.0f) {
    StoreZeros<T, NCH, TPU>(dx, u.n, tid);
    return;
  }
  const typename T::Store *x = RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u) + u.lo;
  U4 r[NCH];
  LoadUnit<T, NCH, TPU>(x, u.n, tid, r);
  int64_t tok = a.tokens ? (a.token64 ? static_cast<const int64_t *>(a.tokens)[u.row]
                                      : static_cast<const int32_t *>(a.tokens)[u.row])
                         : -1;
  if (tok < 0 || tok >= a.r.vocab) tok = -1;
  const float gl = a.g_logp && tok >= 0 ? a.g_logp[u.row] : 0.0f;
  const float gh = a.g_entropy ? a.g_entropy[u.row] : 0.0f;
  const float A = a.g_entropy ? -gl - gh * a.entropy[u.row] : -gl;
  const int at = tok < 0 ? -1 : static_cast<int>(tok) - u.lo;  // (outside the unit: matches no column)
  const float inv = 1.0f / s0, ls = logf(s0);
  StoreUnit<T, NCH, TPU>(dx, u.n, tid, r, [=](float v, int e) {
    const float d = v - m;
    const float p = __builtin_amdgcn_exp2f(d * kLog2e) * inv;
    const float lp = fmaxf(d - ls, -128.0f);  // (below -104 p is 0, and 0 times -inf would be NaN)
    const float g = p * fmaf(-gh, lp, A);
    return e == at ? g + gl : g;
  });
}

// ---- distillation ----------------------------------------------------------------------------------

struct DistillArgs {
  Rows r;
  GradOut o;              // dx null: no gradient
  const void *ids;        // int32 or int64 [rows][slots]
  const void *teacher;    // [rows][slots], teacher_dtype
  int32_t id64, teacher_dtype, slots;
  const float *weights;   // [rows] or null (1)
  const float *upstream;  // [rows] or null (1): times the weight, for the gradient only
  float inv_t, k2;        // 1 / temperature, log2(e) / temperature
  float *loss;            // [rows] or null
  float *stats;           // [rows][2] or null
  const Partial *part;    // split rows: [rows][nseg]
};

__device__ inline float TeacherValue(const DistillArgs &a, size_t at) {
  return a.teacher_dtype == KD_DTYPE_F32   ? static_cast<const float *>(a.teacher)[at]
         : a.teacher_dtype == KD_DTYPE_F16 ? static_cast<float>(static_cast<const _Float16 *>(a.teacher)[at])
                                           : static_cast<float>(static_cast<const __bf16 *>(a.teacher)[at]);
}

// A unit's teacher: lane `tid` holds slots tid, tid + TPU, ...; all of them also in LDS.
struct TeacherList {
  int id[kMaxSlots];
  float q[kMaxSlots];
};
template <int TPU>
struct Slots {
  static constexpr int kN = kMaxSlots / TPU;
  int id[kN];   // -1: empty
  float u[kN];  // (logit - largest) / temperature
  float q[kN];
  float log_usum;
  bool any;
};

template <int TPU>
__device__ inline void LoadSlots(const DistillArgs &a, uint32_t row, int tid, Slots<TPU> &t) {
#pragma unroll
  for (int i = 0; i < Slots<TPU>::kN; ++i) {
    t.id[i] = -1;
    t.u[i] = -INFINITY;
    const int k = i * TPU + tid;
    if (k < a.slots) {
      const size_t at = static_cast<size_t>(row) * a.slots + k;
      const int64_t id =
          a.id64 ? static_cast<const int64_t *>(a.ids)[at] : static_cast<const int32_t *>(a.ids)[at];
      if (id >= 0 && id < a.r.vocab) {
        t.id[i] = static_cast<int>(id);
        t.u[i] = TeacherValue(a, at);
      }
    }
  }
}
// q = softmax(u / temperature) over the filled slots.
template <int TPU>
__device__ inline void SoftmaxSlots(const DistillArgs &a, Slots<TPU> &t, TeacherList &list, float *red, int tid) {
  float um = -INFINITY, sum = 0.0f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < Slots<TPU>::kN; ++i) {
    um = fmaxf(um, t.u[i]);
    nan |= isnan(t.u[i]);
  }
  um = UnitMax<TPU>(nan ? INFINITY : um, red);  // (inf - inf below: NaN for the whole row)
  t.any = um != -INFINITY;
#pragma unroll
  for (int i = 0; i < Slots<TPU>::kN; ++i) {
    t.u[i] = (t.u[i] - Base(um)) * a.inv_t;
    t.q[i] = um == INFINITY && t.id[i] >= 0 ? NAN : expf(t.u[i]);
    sum += t.q[i];
  }
  sum = UnitSum<TPU>(sum, red);
  t.log_usum = logf(sum);
#pragma unroll
  for (int i = 0; i < Slots<TPU>::kN; ++i) {
    t.q[i] = t.q[i] / sum;
    const int k = i * TPU + tid;
    if (k < a.slots) {
      list.id[k] = t.id[i];
      list.q[k] = t.q[i];
    }
  }
  UnitSync<TPU>();
}

// sum_k q_k (log q_k - log p_k), log p_k = (x_k - m) / temperature - ls; xs: the students' logits at the slots.
template <int TPU>
__device__ inline float Divergence(const DistillArgs &a, const Slots<TPU> &t, const float (&xs)[Slots<TPU>::kN],
                                   float m, float ls, float *red) {
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < Slots<TPU>::kN; ++i) {
    // (the logit's product is formed with q / temperature: (lowest - m) / temperature alone may overflow)
    const float d = xs[i] - Base(m), each = (t.u[i] - t.log_usum) + ls;
    if (t.id[i] >= 0 && t.q[i] != 0.0f) sum += fmaf(t.q[i], each, -(t.q[i] * a.inv_t) * d);
  }
  return UnitSum<TPU>(sum, red);
}

// Writes a unit's gradient: coef (p_j - sum of the q of the slots that name column j).  The slots'
// columns are written again behind the others, by one lane each (slots that name one column write
// the same value).
template <class T, int NCH, int TPU>
__device__ inline void WriteDistillGrad(const DistillArgs &a, const Unit &u, const U4 (&r)[NCH], const Slots<TPU> &t,
                                        const float (&xs)[Slots<TPU>::kN], const TeacherList &list, float m, float s0,
                                        float coef, int tid) {
  typename T::Store *dx =
      const_cast<typename T::Store *>(RowPtr<T>(a.o.dx, a.o.batch_stride, a.o.row_stride, u)) + u.lo;
  // (a student without a finite logit gives nothing any probability)
  const float base = Base(m), k2 = a.k2, inv = s0 == 0.0f ? 0.0f : 1.0f / s0, scale = coef * inv;
  StoreUnit<T, NCH, TPU>(dx, u.n, tid, r,
                         [=](float v, int) { return scale * __builtin_amdgcn_exp2f((v - base) * k2); });
  UnitSync<TPU>();
#pragma unroll
  for (int i = 0; i < Slots<TPU>::kN; ++i) {
    if (i * TPU >= a.slots) break;
    const int at = t.id[i] - u.lo;
    const bool mine = t.id[i] >= 0 && at >= 0 && at < u.n;
    if (__ballot(mine)) {
      float q = 0.0f;
      for (int k = 0; k < a.slots; ++k) q += list.id[k] == t.id[i] ? list.q[k] : 0.0f;
      if (mine) dx[at] = T::Round(coef * (__builtin_amdgcn_exp2f((xs[i] - base) * k2) * inv - q));
    }
  }
}

// Whole rows: loss, and with GRAD the gradient from the registers that the statistics were taken of.
template <class T, int NCH, int TPU, bool GRAD>
__global__ __launch_bounds__(kBlock) void DistillKernel(const DistillArgs a) {
  constexpr int kUnits = kBlock / TPU;
  __shared__ TeacherList lists[kUnits];
  __shared__ float red[kWaves];
  const int tid = TPU == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const int which = TPU == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const uint32_t unit = blockIdx.x * kUnits + which;
  if (unit >= a.r.rows) return;
  const Unit u = GetUnit(a.r, unit);
  const float w = u.skip ? 0.0f : a.weights ? a.weights[u.row] : 1.0f;
  TeacherList &list = lists[which];
  Slots<TPU> t;
  t.any = false;
  if (w != 0.0f) {
    LoadSlots<TPU>(a, u.row, tid, t);
    SoftmaxSlots<TPU>(a, t, list, red, tid);
  }
  if (!t.any) {  // (the same in all lanes of the unit)
    if (tid == 0) {
      if (a.loss) a.loss[u.row] = 0.0f;
      if (a.stats) a.stats[2 * static_cast<size_t>(u.row)] = a.stats[2 * static_cast<size_t>(u.row) + 1] = 0.0f;
    }
    if (GRAD)
      StoreZeros<T, NCH, TPU>(
          const_cast<typename T::Store *>(RowPtr<T>(a.o.dx, a.o.batch_stride, a.o.row_stride, u)), u.n, tid);
    return;
  }
  const typename T::Store *x = RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u);
  U4 r[NCH];
  LoadUnit<T, NCH, TPU>(x, u.n, tid, r);
  float xs[Slots<TPU>::kN];
#pragma unroll
  for (int i = 0; i < Slots<TPU>::kN; ++i) xs[i] = t.id[i] >= 0 ? T::Load(x + t.id[i]) : 0.0f;
  float m = -INFINITY;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int j = 0; j < T::kVec; ++j) m = fmaxf(m, T::Get(r[c], j));
  m = UnitMax<TPU>(m, red);
  const float base = Base(m);
  float s0 = 0.0f;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int j = 0; j < T::kVec; ++j) s0 += __builtin_amdgcn_exp2f((T::Get(r[c], j) - base) * a.k2);
  s0 = UnitSum<TPU>(s0, red);
  const float ls = LogSum(s0);
  const float loss = Divergence<TPU>(a, t, xs, m, ls, red);
  if (tid == 0) {
    if (a.loss) a.loss[u.row] = w * loss;
    if (a.stats) {
      a.stats[2 * static_cast<size_t>(u.row)] = m;
      a.stats[2 * static_cast<size_t>(u.row) + 1] = s0;
    }
  }
  if (GRAD) {
    const float coef = w * a.inv_t * (a.upstream ? a.upstream[u.row] : 1.0f);
    WriteDistillGrad<T, NCH, TPU>(a, u, r, t, xs, list, m, s0, coef, tid);
  }
}

// Split rows: the statistics of a row from its segments', and its loss.
template <class T>
__global__ __launch_bounds__(kBlock) void DistillJoinKernel(const DistillArgs a) {
  __shared__ TeacherList list;
  __shared__ float red[kWaves];
  const int tid = threadIdx.x;
  const Unit u = GetUnit(a.r, blockIdx.x * static_cast<uint32_t>(a.r.nseg));
  const float w = u.skip ? 0.0f : a.weights ? a.weights[u.row] : 1.0f;
  Slots<kBlock> t;
  t.any = false;
  if (w != 0.0f) {
    LoadSlots<kBlock>(a, u.row, tid, t);
    SoftmaxSlots<kBlock>(a, t, list, red, tid);
  }
  float m = 0.0f, s0 = 0.0f, loss = 0.0f;
  if (t.any) {
    float s1;
    JoinPartials(a.part + static_cast<size_t>(u.row) * a.r.nseg, a.r.nseg, a.k2, red, &m, &s0, &s1);
    const float ls = LogSum(s0);
    const typename T::Store *x = RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u);
    const float xs[1] = {t.id[0] >= 0 ? T::Load(x + t.id[0]) : 0.0f};
    loss = Divergence<kBlock>(a, t, xs, m, ls, red);
  }
  if (tid == 0) {
    if (a.loss) a.loss[u.row] = t.any ? w * loss : 0.0f;
    a.stats[2 * static_cast<size_t>(u.row)] = m;
    a.stats[2 * static_cast<size_t>(u.row) + 1] = s0;
  }
}

// The gradient of rows or segments whose statistics are known.
template <class T, int NCH, int TPU>
__global__ __launch_bounds__(kBlock) void DistillGradKernel(const DistillArgs a) {
  constexpr int kUnits = kBlock / TPU;
  __shared__ TeacherList lists[kUnits];
  __shared__ float red[kWaves];
  const int tid = TPU == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const int which = TPU == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const uint32_t unit = blockIdx.x * kUnits + which;
  if (unit >= a.r.rows * static_cast<uint32_t>(a.r.nseg)) return;
  const Unit u = GetUnit(a.r, unit);
  const float w = u.skip ? 0.0f : a.weights ? a.weights[u.row] : 1.0f;
  TeacherList &list = lists[which];
  Slots<TPU> t;
  t.any = false;
  if (w != 0.0f) {
    LoadSlots<TPU>(a, u.row, tid, t);
    SoftmaxSlots<TPU>(a, t, list, red, tid);
  }
  if (!t.any) {
    StoreZeros<T, NCH, TPU>(
        const_cast<typename T::Store *>(RowPtr<T>(a.o.dx, a.o.batch_stride, a.o.row_stride, u)) + u.lo, u.n, tid);
    return;
  }
  const typename T::Store *x = RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u);
  U4 r[NCH];
  LoadUnit<T, NCH, TPU>(x + u.lo, u.n, tid, r);
  float xs[Slots<TPU>::kN];
#pragma unroll
  for (int i = 0; i < Slots<TPU>::kN; ++i) xs[i] = t.id[i] >= 0 ? T::Load(x + t.id[i]) : 0.0f;
  const float m = a.stats[2 * static_cast<size_t>(u.row)], s0 = a.stats[2 * static_cast<size_t>(u.row) + 1];
  const float coef = w * a.inv_t * (a.upstream ? a.upstream[u.row] : 1.0f);
  UnitSync<TPU>();  // (the gradient may be written over the logits: every lane has its slots' first)
  WriteDistillGrad<T, NCH, TPU>(a, u, r, t, xs, list, m, s0, coef, tid);
}

// ---- host side -----------------------------------------------------------------------------------

using kd::SetError;

// The tensors' device is made current for the launches, and the caller's put back.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    err_ = hipGetDevice(&old_);
    if (err_ == hipSuccess && old_ != device) {
      err_ = hipSetDevice(device);
      moved_ = err_ == hipSuccess;
    }
  }
  ~DeviceGuard() {
    if (moved_) (void)hipSetDevice(old_);
  }
  hipError_t error() const { return err_; }

 private:
  int old_ = 0;
  bool moved_ = false;
  hipError_t err_ = hipSuccess;
};

int HipFail(const char *what, hipError_t e) {
  return SetError(KD_E_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

template <class ARGS>
int Launch(void (*kernel)(ARGS), uint32_t blocks, const ARGS &args, void *stream) {
  if (!blocks) return KD_OK;
  void *argv[] = {const_cast<ARGS *>(&args)};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3(blocks), dim3(kBlock), argv, 0,
                                       static_cast<hipStream_t>(stream));
  return e == hipSuccess ? KD_OK : HipFail("launch", e);
}

int64_t ElemBytes(int dtype) { return dtype == KD_DTYPE_F32 ? 4 : 2; }

// How rows are dealt out (the comment at the top of this file): TPU threads a unit, NCH 16-byte
// loads each.
struct Plan {
  int tpu, nch, seg_len, nseg;
};
Plan MakePlan(int64_t vocab, int dtype) {
  const int64_t bytes = vocab * ElemBytes(dtype), vec = 16 / ElemBytes(dtype);
  Plan p;
  if (bytes <= 8192) {
    p = {64, 1, static_cast<int>(vocab), 1};
    while (64 * 16 * p.nch < bytes) p.nch *= 2;
  } else {
    const int64_t cap = kBlock * 16 * 8 / ElemBytes(dtype);  // columns of a unit of 32 KiB
    p.tpu = kBlock;
    p.nseg = static_cast<int>((vocab + cap - 1) / cap);
    // equal segments, whole vectors
    p.seg_len = static_cast<int>(((vocab + p.nseg - 1) / p.nseg + vec - 1) / vec * vec);
    p.nseg = static_cast<int>((vocab + p.seg_len - 1) / p.seg_len);
    p.nch = p.seg_len * ElemBytes(dtype) <= kBlock * 16 * 4 ? 4 : 8;
  }
  return p;
}

int CheckRows(const kd_frame_rows *r, Rows *out, Plan *plan, int64_t *rows) {
  if (!r || r->batch < 0 || r->steps < 0) return SetError(KD_E_INVALID, "bad argument: rows");
  if (r->dtype != KD_DTYPE_F32 && r->dtype != KD_DTYPE_F16 && r->dtype != KD_DTYPE_BF16)
    return SetError(KD_E_INVALID, "bad argument: dtype of the logits");
  if (r->vocab < 1 || r->vocab > kMaxVocab)
    return SetError(KD_E_INVALID, "bad argument: vocab must be between 1 and 2^24");
  if (r->batch > INT32_MAX || r->steps > INT32_MAX || r->batch * r->steps > INT32_MAX)
    return SetError(KD_E_INVALID, "bad argument: more than 2^31 - 1 rows");
  *rows = r->batch * r->steps;
  *plan = MakePlan(r->vocab, r->dtype);
  // (a grid has fewer than 2^32 threads)
  if (*rows * plan->nseg > ((int64_t(1) << 24) - 1) * (kBlock / plan->tpu))
    return SetError(KD_E_INVALID, "bad argument: rows x vocab is too large for one call");
  if (r->batch_stride < 0 || r->row_stride < 0) return SetError(KD_E_INVALID, "bad argument: negative stride");
  if (*rows && !r->logits) return SetError(KD_E_INVALID, "bad argument: logits is NULL");
  if (r->device < 0) return SetError(KD_E_INVALID, "bad argument: device");
  if (reinterpret_cast<uintptr_t>(r->logits) % ElemBytes(r->dtype))
    return SetError(KD_E_INVALID, "bad argument: logits are not aligned to their type");
  out->x = r->logits;
  out->lengths = r->lengths;
  out->batch_stride = r->batch_stride;
  out->row_stride = r->row_stride;
  out->rows = static_cast<uint32_t>(*rows);
  out->steps = static_cast<uint32_t>(r->steps);
  out->vocab = static_cast<int32_t>(r->vocab);
  out->seg_len = plan->seg_len;
  out->nseg = plan->nseg;
  return KD_OK;
}

// A gradient's rows must not lie over each other.
int CheckGrad(const kd_frame_rows *r, void *dx, int64_t batch_stride, int64_t row_stride, GradOut *o) {
  if (!dx) return SetError(KD_E_INVALID, "bad argument: grad is NULL");
  if (reinterpret_cast<uintptr_t>(dx) % ElemBytes(r->dtype))
    return SetError(KD_E_INVALID, "bad argument: grad is not aligned to its type");
  int64_t n[2] = {r->steps, r->batch}, s[2] = {row_stride, batch_stride};
  if (s[0] > s[1]) {
    std::swap(n[0], n[1]);
    std::swap(s[0], s[1]);
  }
  int64_t span = r->vocab;
  for (int i = 0; i < 2; ++i) {
    if (n[i] <= 1) continue;
    if (s[i] < span) return SetError(KD_E_INVALID, "bad argument: the gradient's rows overlap");
    span += (n[i] - 1) * s[i];
  }
  o->dx = dx;
  o->batch_stride = batch_stride;
  o->row_stride = row_stride;
  return KD_OK;
}

uint32_t Blocks(const Rows &r, const Plan &p) {
  const uint64_t units = static_cast<uint64_t>(r.rows) * r.nseg;
  return static_cast<uint32_t>(p.tpu == 64 ? (units + kWaves - 1) / kWaves : units);
}

// f(T{}, NCH, TPU as constants) for a plan.
template <int N>
struct Int {
  static constexpr int value = N;
};
template <class T, class F>
int ForPlan(const Plan &p, F f) {
  if (p.tpu == 64) {
    switch (p.nch) {
      case 1: return f(T{}, Int<1>{}, Int<64>{});
      case 2: return f(T{}, Int<2>{}, Int<64>{});
      case 4: return f(T{}, Int<4>{}, Int<64>{});
      default: return f(T{}, Int<8>{}, Int<64>{});
    }
  }
  return p.nch == 4 ? f(T{}, Int<4>{}, Int<kBlock>{}) : f(T{}, Int<8>{}, Int<kBlock>{});
}
template <class F>
int ForType(int dtype, F f) {
  return dtype == KD_DTYPE_F32 ? f(F32{}) : dtype == KD_DTYPE_F16 ? f(F16{}) : f(BF16{});
}

size_t Align(size_t n) { return (n + 255) & ~size_t(255); }

// No C++ exception leaves a C entry.
template <class F>
int Guarded(F f) {
  try {
    return f();
  } catch (const std::exception &) {
    return KD_E_INVALID;
  }
}

template <bool SPLIT, bool ENT, bool TOP>
int LaunchScores(const kd_frame_rows *rows, const ScoresArgs &a, const Plan &plan, void *stream) {
  return ForType(rows->dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (SPLIT) {
      return plan.nch == 4 ? Launch(ScoresKernel<T, 4, kBlock, true, ENT, TOP>, Blocks(a.r, plan), a, stream)
                           : Launch(ScoresKernel<T, 8, kBlock, true, ENT, TOP>, Blocks(a.r, plan), a, stream);
    } else {
      return ForPlan<T>(plan, [&](auto tt, auto nch, auto tpu) {
        return Launch(ScoresKernel<decltype(tt), decltype(nch)::value, decltype(tpu)::value, false, ENT, TOP>,
                      Blocks(a.r, plan), a, stream);
      });
    }
  });
}

}  // namespace

extern "C" {

size_t kd_token_scores_workspace(const kd_frame_rows *rows, int32_t top) {
  Rows r;
  Plan p;
  int64_t n;
  if (CheckRows(rows, &r, &p, &n) || top < 0 || top > kMaxTop || p.nseg == 1) return 0;
  const size_t units = static_cast<size_t>(n) * p.nseg;
  return Align(units * sizeof(Partial)) + (top ? Align(units * top * 4) * 2 : 0);
}

int kd_token_scores(const kd_frame_rows *rows, const void *tokens, int32_t token_bytes, int32_t top, float *logp,
                    float *entropy, float *stats, float *top_logp, int32_t *top_ids, void *workspace,
                    size_t workspace_bytes, void *stream) {
  return Guarded([&]() -> int {
    ScoresArgs a{};
    Plan p;
    int64_t n;
    if (int rc = CheckRows(rows, &a.r, &p, &n)) return rc;
    if (top < 0 || top > kMaxTop) return SetError(KD_E_INVALID, "bad argument: top must be between 0 and 64");
    if (tokens && token_bytes != 4 && token_bytes != 8)
      return SetError(KD_E_INVALID, "bad argument: token_bytes must be 4 or 8");
    if (!n) return KD_OK;
    if ((tokens && !logp) || !entropy || !stats || (top && (!top_logp || !top_ids)))
      return SetError(KD_E_INVALID, "bad argument: an output is NULL");
    const size_t need = kd_token_scores_workspace(rows, top);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
      return SetError(KD_E_INVALID, "bad argument: the workspace is too small (kd_token_scores_workspace) or unaligned");
    a.tokens = tokens;
    a.token64 = token_bytes == 8;
    a.k = top;
    a.k2 = kLog2e;
    a.logp = logp;
    a.entropy = entropy;
    a.stats = stats;
    a.top_v = top_logp;
    a.top_i = top_ids;
    DeviceGuard guard(rows->device);
    if (guard.error() != hipSuccess) return HipFail("hipSetDevice", guard.error());
    if (p.nseg == 1)
      return top ? LaunchScores<false, true, true>(rows, a, p, stream)
                 : LaunchScores<false, true, false>(rows, a, p, stream);
    const size_t units = static_cast<size_t>(n) * p.nseg;
    char *ws = static_cast<char *>(workspace);
    a.part = reinterpret_cast<Partial *>(ws);
    a.part_v = reinterpret_cast<float *>(ws + Align(units * sizeof(Partial)));
    a.part_i = reinterpret_cast<int32_t *>(ws + Align(units * sizeof(Partial)) + Align(units * top * 4));
    if (int rc = top ? LaunchScores<true, true, true>(rows, a, p, stream)
                     : LaunchScores<true, true, false>(rows, a, p, stream))
      return rc;
    return ForType(rows->dtype, [&](auto t) {
      using T = decltype(t);
      return top ? Launch(ScoresJoinKernel<T, true>, a.r.rows, a, stream)
                 : Launch(ScoresJoinKernel<T, false>, a.r.rows, a, stream);
    });
  });
}

int kd_token_scores_grad(const kd_frame_rows *rows, const void *tokens, int32_t token_bytes, const float *stats,
                         const float *entropy, const float *grad_logp, const float *grad_entropy, void *grad,
                         int64_t grad_batch_stride, int64_t grad_row_stride, void *stream) {
  return Guarded([&]() -> int {
    ScoresGradArgs a{};
    Plan p;
    int64_t n;
    if (int rc = CheckRows(rows, &a.r, &p, &n)) return rc;
    if (tokens && token_bytes != 4 && token_bytes != 8)
      return SetError(KD_E_INVALID, "bad argument: token_bytes must be 4 or 8");
    if (!n) return KD_OK;
    if (!stats || (grad_entropy && !entropy)) return SetError(KD_E_INVALID, "bad argument: stats / entropy is NULL");
    if (int rc = CheckGrad(rows, grad, grad_batch_stride, grad_row_stride, &a.o)) return rc;
    a.tokens = tokens;
    a.token64 = token_bytes == 8;
    a.stats = stats;
    a.entropy = entropy;
    a.g_logp = grad_logp;
    a.g_entropy = grad_entropy;
    DeviceGuard guard(rows->device);
    if (guard.error() != hipSuccess) return HipFail("hipSetDevice", guard.error());
    return ForType(rows->dtype, [&](auto t) {
      return ForPlan<decltype(t)>(p, [&](auto tt, auto nch, auto tpu) {
        return Launch(ScoresGradKernel<decltype(tt), decltype(nch)::value, decltype(tpu)::value>, Blocks(a.r, p), a,
                      stream);
      });
    });
  });
}

size_t kd_distill_loss_workspace(const kd_frame_rows *rows) {
  Rows r;
  Plan p;
  int64_t n;
  if (CheckRows(rows, &r, &p, &n) || p.nseg == 1) return 0;
  return Align(static_cast<size_t>(n) * p.nseg * sizeof(Partial)) + Align(static_cast<size_t>(n) * 8);
}

int kd_distill_loss(const kd_frame_rows *rows, const kd_teacher_rows *teacher, const float *weights, float temperature,
                    float *loss, float *stats, const float *upstream, void *grad, int64_t grad_batch_stride,
                    int64_t grad_row_stride, void *workspace, size_t workspace_bytes, void *stream) {
  return Guarded([&]() -> int {
    DistillArgs a{};
    Plan p;
    int64_t n;
    if (int rc = CheckRows(rows, &a.r, &p, &n)) return rc;
    if (!teacher || teacher->slots < 1 || teacher->slots > kMaxSlots)
      return SetError(KD_E_INVALID, "bad argument: a teacher lists between 1 and 256 tokens a row");
    if (teacher->id_bytes != 4 && teacher->id_bytes != 8)
      return SetError(KD_E_INVALID, "bad argument: id_bytes must be 4 or 8");
    if (teacher->dtype != KD_DTYPE_F32 && teacher->dtype != KD_DTYPE_F16 && teacher->dtype != KD_DTYPE_BF16)
      return SetError(KD_E_INVALID, "bad argument: dtype of the teacher's logits");
    if (!(temperature > 0.0f) || !std::isfinite(temperature) || !std::isfinite(kLog2e / temperature))
      return SetError(KD_E_INVALID, "bad argument: temperature must be positive and finite");
    if (!n) return KD_OK;
    if (!teacher->ids || !teacher->logits) return SetError(KD_E_INVALID, "bad argument: the teacher's list is NULL");
    if (!loss && !grad) return SetError(KD_E_INVALID, "bad argument: neither loss nor gradient asked for");
    // stats given and no loss asked for: the statistics of an earlier call, the gradient alone
    const bool known = !loss && stats;
    if (!loss && !stats) return SetError(KD_E_INVALID, "bad argument: a gradient alone needs the loss's stats");
    if (grad)
      if (int rc = CheckGrad(rows, grad, grad_batch_stride, grad_row_stride, &a.o)) return rc;
    const size_t need = known ? 0 : kd_distill_loss_workspace(rows);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
      return SetError(KD_E_INVALID, "bad argument: the workspace is too small (kd_distill_loss_workspace) or unaligned");
    a.ids = teacher->ids;
    a.id64 = teacher->id_bytes == 8;
    a.teacher = teacher->logits;
    a.teacher_dtype = teacher->dtype;
    a.slots = teacher->slots;
    a.weights = weights;
    a.upstream = upstream;
    a.inv_t = static_cast<float>(1.0 / static_cast<double>(temperature));
    a.k2 = static_cast<float>(1.44269504088896340736 / static_cast<double>(temperature));
    a.loss = loss;
    a.stats = stats;
    DeviceGuard guard(rows->device);
    if (guard.error() != hipSuccess) return HipFail("hipSetDevice", guard.error());
    if (p.nseg > 1 && !known) {
      ScoresArgs s{};
      s.r = a.r;
      s.k2 = a.k2;
      s.part = static_cast<Partial *>(workspace);
      if (!a.stats)
        a.stats = reinterpret_cast<float *>(static_cast<char *>(workspace) +
                                            Align(static_cast<size_t>(n) * p.nseg * sizeof(Partial)));
      a.part = s.part;
      if (int rc = LaunchScores<true, false, false>(rows, s, p, stream)) return rc;
      if (int rc = ForType(rows->dtype, [&](auto t) {
            return Launch(DistillJoinKernel<decltype(t)>, a.r.rows, a, stream);
          }))
        return rc;
      if (!grad) return KD_OK;
    }
    if (p.nseg > 1 || known) {
      return ForType(rows->dtype, [&](auto t) {
        return ForPlan<decltype(t)>(p, [&](auto tt, auto nch, auto tpu) {
          return Launch(DistillGradKernel<decltype(tt), decltype(nch)::value, decltype(tpu)::value>, Blocks(a.r, p), a,
                        stream);
        });
      });
    }
    return ForType(rows->dtype, [&](auto t) {
      return ForPlan<decltype(t)>(p, [&](auto tt, auto nch, auto tpu) {
        using T = decltype(tt);
        constexpr int N = decltype(nch)::value, TPU = decltype(tpu)::value;
        return grad ? Launch(DistillKernel<T, N, TPU, true>, Blocks(a.r, p), a, stream)
                    : Launch(DistillKernel<T, N, TPU, false>, Blocks(a.r, p), a, stream);
      });
    });
  });
}

}  // extern "C"
