// kaldi-decoder_amd/csrc/kd_frames.hip -- operators over a model's frame logits (include/kd_hip.h,
// "scores of given tokens" and "distillation"): kernels and their C entries.
//
// Everything here works on rows of V logits (f32, f16 or bf16), [batch][steps][V] with strides and
// optional lengths, the rows that the search itself is handed.  The operators are bound by the bytes of
// the logits, so the one rule is that a row is read once: a UNIT -- a whole row, or a segment of a
// long one -- is loaded into the registers of TPU lanes, up to NCH 16-byte loads each, and every pass
// over it (maximum, sums, alternatives, gradient) runs over those registers.  How rows are dealt out
// (MakePlan):
//
//   row           unit                                  one for all: the steps taken once a row
//   to 2 KiB      16 lanes, four rows a wave            ... serve four rows
//   to 8 KiB      a wave                                ... need no barrier
//   to 32 KiB     a workgroup of 256
//   to 64 KiB     a workgroup of 512 (values, and loss with gradient)
//   to 256 KiB    a workgroup of 1024, loss with gradient of many rows: read once, written once
//   longer, few   segments, whose partial results (maximum, sums, alternatives) a second kernel joins
//
// Sums and statistics are f32; logits and gradients are rounded once, on the way in and out.
// Figures below: one MI355X, kernels in a graph; large copies run at 4.9 TB/s there (read + write).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <initializer_list>
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
constexpr int64_t kMaxVocab = int64_t(1) << 24;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
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

template <int TPU>
constexpr int kThreads = TPU < kBlock ? kBlock : TPU;  // of a workgroup
// Waves a SIMD that a kernel is compiled for (1: as many as its registers allow).  Units of 512 lanes
// take two a SIMD, so 68 registers instead of 64 would cost one unit in four (38.0 instead of 42.0 us
// for 2048 rows of 32768 bf16 with 64 alternatives); units of 16 lanes hold 16 addresses a lane unless
// told not to (18.4 instead of 18.6 us for the loss and gradient of 24000 rows of 500 with 8 slots), but
// with four slots a lane loss and gradient together would spill registers (32 slots: 27.1 us, and 25.1 left
// alone).  SN: slots a lane, of such a kernel.
template <int TPU, int NCH, int SN = 1>
constexpr int kOccupancy = (TPU == 16 && SN == 1) || TPU == 512 || (TPU == 1024 && NCH <= 8) ? 8 : 1;
template <int TPU>
__device__ inline int UnitLane() {
  return TPU < kBlock ? (threadIdx.x & (TPU - 1)) : threadIdx.x;
}
// Which of a workgroup's units a lane belongs to, and the unit's number.  A wave's (TPU 64) is the
// same in all its lanes; 16 lanes (a DPP row) are the smallest unit.
template <int TPU>
__device__ inline int UnitInBlock() {
  return TPU == 16 ? threadIdx.x >> 4 : TPU == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
}
template <int TPU>
constexpr int kUnits = kThreads<TPU> / TPU;  // in a workgroup
template <int TPU>
__device__ inline uint32_t UnitNumber() {
  return blockIdx.x * kUnits<TPU> + UnitInBlock<TPU>();
}

// Lane `tid` of a unit holds 16 bytes of columns from (c * TPU + tid) * kVec on in r[c]: consecutive
// lanes load consecutive 16 bytes.  (Rows need no alignment beyond their element's: the loads are
// marked so and stay 16 bytes wide.)  Where those 16 bytes would reach over the row's end the lane
// holds the row's LAST 16 bytes, and the columns that are another lane's (or, further out, all of
// them) are replaced by kFill: no load depends on a branch, so all NCH are in flight at once.
template <class T>
__device__ inline int FirstCol(int e, int n) {
  return min(e, max(n - T::kVec, 0));
}
// Whether any lane of a unit of n columns has some in r[c] (passes leave out the others: the same
// for the whole unit, and one kernel for 8 16-byte loads a lane does the work of fewer as well).
template <class T, int TPU>
__device__ inline bool Used(int c, int n) {
  return c == 0 || c * TPU * T::kVec < n;
}
template <class T, int NCH, int TPU>
__device__ inline void LoadUnit(const typename T::Store *p, int n, int tid, U4 (&r)[NCH]) {
  if (n >= T::kVec) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (Used<T, TPU>(c, n))
        r[c] = *reinterpret_cast<const typename T::Vec *>(p + FirstCol<T>((c * TPU + tid) * T::kVec, n));
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if ((c + 1) * TPU * T::kVec <= n || !Used<T, TPU>(c, n)) continue;  // (no lane of this one reaches the end)
      const int e = (c * TPU + tid) * T::kVec, others = e - FirstCol<T>(e, n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (T::kVec == 4) {
          r[c][i] = i < others ? T::kFill : r[c][i];
        } else {
          uint32_t v = r[c][i];
          v = 2 * i < others ? (v & 0xffff0000u) | (T::kFill & 0xffffu) : v;
          r[c][i] = 2 * i + 1 < others ? (v & 0xffffu) | (T::kFill & 0xffff0000u) : v;
        }
      }
    }
  } else {  // a row of less than 16 bytes: all lane 0's
    r[0] = U4{T::kFill, T::kFill, T::kFill, T::kFill};
    if (tid == 0) {
#pragma unroll
      for (int j = 0; j < T::kVec - 1; ++j) {
        if (j >= n) break;
        if (T::kVec == 4) {
          r[0][j] = __builtin_bit_cast(uint32_t, static_cast<float>(p[j]));
        } else {
          const uint32_t v = reinterpret_cast<const uint16_t *>(p)[j];
          r[0][j >> 1] = (j & 1) ? (r[0][j >> 1] & 0xffffu) | v << 16 : (r[0][j >> 1] & 0xffff0000u) | v;
        }
      }
    }
  }
}
// Between two passes over a unit's registers: without it the compiler keeps the first pass's
// conversions for the second, two (f16, bf16: four) times the registers.
template <int NCH>
__device__ inline void NewPass(U4 (&r)[NCH]) {
#pragma unroll
  for (int c = 0; c < NCH; ++c) asm volatile("" : "+v"(r[c]));
}

// ---- reductions over a unit --------------------------------------------------------------------
// The larger of two; NaN if either is.  (fmaxf, which drops NaN, costs an instruction more for each
// operand that might be a signaling one; this is one v_maximum3, for three operands too.)
__device__ inline float Max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ inline float Min(float a, float b) { return __builtin_elementwise_minimum(a, b); }

template <int CTRL, int ROW_MASK, int BANK_MASK = 0xf>
__device__ inline float Dpp(float old, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL, ROW_MASK, BANK_MASK,
                                                    false));
}
// The same where every lane takes part: lanes without a source get 0.  (Nothing is kept of an old value,
// so the move becomes an operand of what uses it.)
template <int CTRL>
__device__ inline int MoveI(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ inline float Move(float v) {
  return __int_as_float(MoveI<CTRL>(__float_as_int(v)));
}
// Over 16 lanes (a DPP row), by rotations: every lane has the result.
constexpr int kRowRor = 0x120;
__device__ inline float RowMax(float v) {
  v = Max(v, Move<kRowRor + 8>(v));
  v = Max(v, Move<kRowRor + 4>(v));
  v = Max(v, Move<kRowRor + 2>(v));
  return Max(v, Move<kRowRor + 1>(v));
}
__device__ inline float RowSum(float v) {
  v += Move<kRowRor + 8>(v);
  v += Move<kRowRor + 4>(v);
  v += Move<kRowRor + 2>(v);
  return v + Move<kRowRor + 1>(v);
}
__device__ inline int RowSum(int v) {
  v += MoveI<kRowRor + 8>(v);
  v += MoveI<kRowRor + 4>(v);
  v += MoveI<kRowRor + 2>(v);
  return v + MoveI<kRowRor + 1>(v);
}
// Over a wave: rows 1 and 3 take over what row 0 and 2 have, then rows 2 and 3; lane 63 has all.
__device__ inline float Lane63(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }
__device__ inline float WaveMax(float v) {
  v = RowMax(v);
  v = Max(v, Dpp<0x142, 0xa>(v, v));  // row_bcast:15
  return Lane63(Max(v, Dpp<0x143, 0xc>(v, v)));  // row_bcast:31
}
__device__ inline float WaveSum(float v) {
  v = RowSum(v);
  v += Dpp<0x142, 0xa>(0.0f, v);
  return Lane63(v + Dpp<0x143, 0xc>(0.0f, v));
}

// A unit of a wave or less is never synchronised with the workgroup's others.
template <int TPU>
__device__ inline void UnitSync() {
  if (TPU > 64) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// `red`: one float a wave, not written again before the unit's next barrier but one.
template <int TPU>
__device__ inline float UnitMax(float v, float *red) {
  if (TPU == 16) return RowMax(v);
  v = WaveMax(v);
  if (TPU == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < TPU / 64; ++w) v = Max(v, red[w]);
  return v;
}
template <int TPU>
__device__ inline float SumOf(const float *red) {
  float v = red[0];
#pragma unroll
  for (int w = 1; w < TPU / 64; ++w) v += red[w];
  return v;
}
template <int TPU>
__device__ inline float UnitSum(float v, float *red) {
  if (TPU == 16) return RowSum(v);
  v = WaveSum(v);
  if (TPU == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return SumOf<TPU>(red);
}
// Sum over the unit of counts that every lane of a wave already agrees on.
template <int TPU>
__device__ inline int UnitCount(int wave_count, int *red) {
  if (TPU == 64) return wave_count;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = wave_count;
  __syncthreads();
  int v = 0;
#pragma unroll
  for (int w = 0; w < TPU / 64; ++w) v += red[w];
  __syncthreads();
  return v;
}
__device__ inline int Popc(uint64_t m) { return __popcll(m); }

// ---- sums of exponentials ------------------------------------------------------------------------
// e_j = exp2((x_j - m) k2) as exp2(fma(x_j, k2, -c)), c = m k2 rounded: one operation less an element
// than the difference times k2, and as exact -- what the rounding of c adds to every exponent is
// known (delta; at most 64) and taken out of the sums afterwards.  From |c| = 2^30 on (rows of the
// type's lowest value) any column that differs from m at all is 2^64 times smaller: there a power
// of two stands in for k2 that makes m k2 exact, about 2^40, and such columns' e 0.
// (1.5e-6 <= k2 <= 1.5e6, the range of the temperature.)
// The maximum's own e comes out as `one`, 2^delta rounded, the same bits wherever it is computed.  What is
// known to be 1 is therefore divided by it and not multiplied by another rounding of 2^-delta: a row that one
// token has nearly to itself would lose two roundings of 1 in s, and so in its log p and 1 - p.
struct Exponent {
  float k2, c, delta, one;
  __device__ Exponent(float base, float k2_) {
    const bool far = !(fabsf(base * k2_) < 0x1p30f) && base != INFINITY;
    k2 = far ? __uint_as_float(__float_as_uint(0x1p40f / fabsf(base)) & 0x7f800000u) : k2_;
    c = base * k2;
    delta = fmaf(base, k2, -c);  // exponents come out larger by this much
    one = __builtin_amdgcn_exp2f(delta);
  }
  __device__ float PerOne() const {  // 1 / one, within one step
    const float r = __builtin_amdgcn_rcpf(one);
    return fmaf(fmaf(-one, r, 1.0f), r, r);
  }
  __device__ float operator()(float x) const { return fmaf(x, k2, -c); }
};

// f(FIRST) + ... + f(FIRST + N - 1), in pairs: the 1 that a row's maximum brings in then takes part in a few
// additions of a lane's and not in all that follow it, each of which would round it.
template <int N, int FIRST = 0, class F>
__device__ inline float PairSum(const F &f) {
  if constexpr (N == 1) {
    return f(FIRST);
  } else {
    const float a = PairSum<N / 2, FIRST>(f);
    return a + PairSum<N / 2, FIRST + N / 2>(f);
  }
}

// ---- the K largest -------------------------------------------------------------------------------
// Order: larger value first, then lower column.  -inf and NaN are no candidates.
//
// 1. A threshold from the maxima of 64 or 128 groups of the unit's elements.
// 2. The elements that reach it are collected in LDS, each wave's in a list of its own.  Where they
//    are more than the lists hold (many equal values, or most of the large ones in few groups) the
//    K-th element itself is found by bisection, its value bit by bit and then, among equals, its
//    column: exactly K are left.
// 3. Each candidate's place is the number of candidates ahead of it.
constexpr int kCap = 128;       // candidates a wave's list holds; a unit of one wave: twice that
constexpr int kMaxRanked = 512; // candidates a unit ranks

template <int TPU>
struct Scratch {
  static constexpr int kW = TPU / 64;
  static constexpr int kList = kW == 1 ? 2 * kCap : kCap;
  float red[3][kW];
  int count[kW];
  float threshold;
  float group_max[kW == 1 ? 1 : 64 * kW];
  int place[kW == 1 ? 1 : kMaxRanked];
  uint64_t cand[kW][kList];  // Key
  U4 raw[kW][kList / 2];     // 16 bytes with a candidate among them, and whose they were
  uint16_t raw_of[kW][kList / 2];
};

// A whole number that orders as the value does (-0 and +0 alike).
__device__ inline uint32_t OrderKey(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ inline float KeyValue(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// A candidate as one number that orders as candidates do: larger value first, then lower column.
// (0: none.)
__device__ inline uint64_t Key(float v, int col) {
  return static_cast<uint64_t>(OrderKey(v)) << 32 | static_cast<uint32_t>(~col);
}
__device__ inline float ValueOf(uint64_t key) { return KeyValue(static_cast<uint32_t>(key >> 32)); }
__device__ inline int ColumnOf(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

// Values sorted over lanes, the largest first: bitonic sorts whose merges start with a mirrored
// exchange, so that every lane below its partner keeps the larger.
__device__ inline float Keep(float v, float o, bool below) { return below ? Max(v, o) : Min(v, o); }
template <int CTRL>
__device__ inline float Exchange(float v, bool below) {
  return Keep(v, Move<CTRL>(v), below);
}
__device__ inline float Exchange4(float v) {  // lane ^ 4: the lane 4 further or 4 before
  const float up = Dpp<0x104, 0xf, 0x5>(v, v);
  return Keep(v, Dpp<0x114, 0xf, 0xa>(up, v), !(threadIdx.x & 4));
}
__device__ inline float RowMerge8(float v) {  // 8 lanes' bitonic sequences
  const int l = threadIdx.x;
  v = Exchange4(v);
  v = Exchange<0x4e>(v, !(l & 2));  // lane ^ 2
  return Exchange<0xb1>(v, !(l & 1));
}
__device__ inline float RowMerge(float v) {  // 16 lanes'
  return RowMerge8(Exchange<kRowRor + 8>(v, !(threadIdx.x & 8)));
}
__device__ inline float RowSort(float v) {  // 16 lanes
  const int l = threadIdx.x;
  const bool b0 = !(l & 1), b1 = !(l & 2);
  v = Exchange<0xb1>(v, b0);
  v = Exchange<0x1b>(v, b1);  // lane ^ 3
  v = Exchange<0xb1>(v, b0);
  v = Exchange<0x141>(v, !(l & 4));  // lane ^ 7
  v = Exchange<0x4e>(v, b1);
  v = Exchange<0xb1>(v, b0);
  return RowMerge8(Exchange<0x140>(v, !(l & 8)));  // lane ^ 15
}
__device__ inline float OfLane(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_ds_bpermute(lane * 4, __float_as_int(v)));
}
__device__ inline float WaveSort(float v) {
  const int l = threadIdx.x & 63;
  v = RowSort(v);
  v = RowMerge(Keep(v, OfLane(v, l ^ 31), !(l & 16)));
  v = Keep(v, OfLane(v, l ^ 63), !(l & 32));
  return RowMerge(Keep(v, OfLane(v, l ^ 16), !(l & 16)));
}

// A value that at least k of a unit's elements reach, and few more than k do: about the k-th largest
// of the maxima of 64 groups of them (k <= 32; candidates of data in no particular order: 24 for 20)
// or of 128 (the 64th; 89 for 64).  `g`: a unit of one wave has its groups' maxima in its lanes; else
// they are in LDS, and one wave sorts while the others' issue slots are free for other units.
__device__ inline float WaveThreshold(float a, float b, int k) {
  if (k <= 32) {
    const float v = WaveSort(Max(a, b));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), k - 1));
  }
  a = WaveSort(a);
  b = WaveSort(b);
  // the 64 largest of both are the larger of the l-th and the (63 - l)-th
  return -WaveMax(-Max(a, OfLane(b, (threadIdx.x & 63) ^ 63)));
}
template <int TPU>
__device__ inline float GroupThreshold(const float (&g)[2], Scratch<TPU> &s, int k) {
  if (TPU == 64) return WaveThreshold(g[0], g[1], k);
  if (threadIdx.x < 64) {
    float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int w = 0; w < TPU / 64; ++w) m[w & 1] = Max(m[w & 1], s.group_max[64 * w + threadIdx.x]);
    const float t = WaveThreshold(m[0], m[1], k);
    if (threadIdx.x == 0) s.threshold = t;
  }
  __syncthreads();
  return s.threshold;
}

// What a selection reads, as f(value, column) with all lanes of a wave in step: a list in memory (the
// alternatives of a row's segments), in registers, or a unit's elements.  A unit in registers is
// collected in two steps (CollectUnit).
//
// A unit from memory, for the bisection, which is rare: over the registers it would make every
// kernel hold its code many times over.
template <class T, int TPU>
struct MemSource {
  static constexpr int kLowBit = sizeof(typename T::Store) == 4 ? 0 : 13;  // an f16's or bf16's lower bits are 0
  const typename T::Store *p;
  int lo, n, tid;
  template <class F>
  __device__ void Each(float, F f) const {
    for (int base = 0; base < n; base += TPU) {
      const int k = base + tid;
      f(k < n ? T::Load(p + k) : -INFINITY, lo + k);
    }
  }
};
// The sorted lists of a row's segments, in memory (the first of all, then the second of all, ...:
// a thread's share, whose maximum is one of the threshold's groups, has few of any one list's head).
struct ListSource {
  static constexpr int kLowBit = 0;
  const uint64_t *list;  // [nseg][k]
  int nseg, k, tid;
  template <class F>
  __device__ void Each(float, F f) const {
    int at = tid / nseg, seg = tid - at * nseg;
    const int ats = kBlock / nseg, segs = kBlock - ats * nseg;
    for (int base = 0; base < nseg * k; base += kBlock) {
      const uint64_t key = at < k ? list[static_cast<size_t>(seg) * k + at] : 0;  // (0: its value is a NaN)
      f(ValueOf(key), ColumnOf(key));
      at += ats;
      seg += segs;
      if (seg >= nseg) {
        seg -= nseg;
        ++at;
      }
    }
  }
};

// The same list in registers.
template <int N>
struct HeldSource {
  uint64_t key[N];
  __device__ void Load(const ListSource &l) {
    int at = l.tid / l.nseg, seg = l.tid - at * l.nseg;
    const int ats = kBlock / l.nseg, segs = kBlock - ats * l.nseg;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      key[i] = at < l.k ? l.list[static_cast<size_t>(seg) * l.k + at] : 0;
      at += ats;
      seg += segs;
      if (seg >= l.nseg) {
        seg -= l.nseg;
        ++at;
      }
    }
  }
  template <class F>
  __device__ void Each(float, F f) const {
#pragma unroll
    for (int i = 0; i < N; ++i) f(ValueOf(key[i]), ColumnOf(key[i]));
  }
};

// Collects a wave's elements that `pred` holds for (none below floor_v); their number, kept or not,
// in s.count[wave].
template <int TPU, class SRC, class PRED>
__device__ inline void Collect(const SRC &src, Scratch<TPU> &s, float floor_v, PRED pred) {
  const int lane = threadIdx.x & 63, w = TPU == 64 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int n = 0;
  src.Each(floor_v, [&](float v, int i) {
    const bool mine = pred(v, i);
    const uint64_t m = __ballot(mine);
    if (m) {
      const int pos = n + Popc(m & ((uint64_t(1) << lane) - 1));
      if (mine && pos < Scratch<TPU>::kList) s.cand[w][pos] = Key(v, i);
      n += Popc(m);
    }
  });
  if (lane == 0) s.count[w] = n;
}

// The same of a unit's registers, in two steps: the 16 bytes that have such an element (`cm`: a lane's
// maximum of each) are put into LDS, then a lane takes each and lists its elements -- a third of the
// instructions, and an eighth of the code, of looking at each register's elements in turn.
template <class T, int NCH, int TPU>
__device__ inline void CollectUnit(const U4 (&r)[NCH], const float (&cm)[NCH], int lo, int cols, Scratch<TPU> &s,
                                   float floor_v) {
  constexpr int kList = Scratch<TPU>::kList;
  const int lane = threadIdx.x & 63, w = TPU == 64 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint64_t below = (uint64_t(1) << lane) - 1;
  int held = 0;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const bool mine = cm[c] >= floor_v;
    const uint64_t m = __ballot(mine);
    if (m) {
      const int pos = held + Popc(m & below);
      if (mine && pos < kList / 2) {
        s.raw[w][pos] = r[c];
        s.raw_of[w][pos] = static_cast<uint16_t>(c * TPU + UnitLane<TPU>());
      }
      held += Popc(m);
    }
  }
  int n = held > kList / 2 ? kList + 1 : 0;  // (too many to hold: as too many candidates)
  if (!n) {
    UnitSync<64>();
    for (int base = 0; base < held; base += 64) {
      const bool have = base + lane < held;
      const U4 v = s.raw[w][have ? base + lane : 0];
      const int e = s.raw_of[w][have ? base + lane : 0] * T::kVec, first = FirstCol<T>(e, cols);
#pragma unroll
      for (int j = 0; j < T::kVec; ++j) {
        const float x = T::Get(v, j);
        const bool mine = have && first + j >= e && x >= floor_v;
        const uint64_t m = __ballot(mine);
        const int pos = n + Popc(m & below);
        if (mine && pos < kList) s.cand[w][pos] = Key(x, lo + first + j);
        n += Popc(m);
      }
    }
  }
  if (lane == 0) s.count[w] = n;
}

// The key of the k-th element itself, among those that reach `floor_v`; at least k do.
template <int TPU, class SRC>
__device__ __noinline__ uint64_t KthElement(const SRC src, int *red, float floor_v, int k) {
  uint32_t t = 0;
  for (int bit = 31; bit >= SRC::kLowBit; --bit) {
    const uint32_t c = t | (1u << bit);
    int n = 0;
    src.Each(floor_v, [&](float v, int) { n += Popc(__ballot(v >= floor_v && OrderKey(v) >= c)); });
    if (UnitCount<TPU>(n, red) >= k) t = c;
  }
  if (!(t & 0x80000000u)) t |= (1u << SRC::kLowBit) - 1;  // (a negative value's bits are inverted in its key)
  const float val = KeyValue(t);
  int above = 0;
  src.Each(floor_v, [&](float v, int) { above += Popc(__ballot(v > val)); });
  const int need = k - UnitCount<TPU>(above, red);  // of the equals, the first `need` columns
  int col = 0;  // (the largest column that fewer than `need` equals are in front of; columns < 2^24)
  for (int bit = 23; bit >= 0; --bit) {
    const int c = col | (1 << bit);
    int n = 0;
    src.Each(floor_v, [&](float v, int i) { n += Popc(__ballot(v == val && i < c)); });
    if (UnitCount<TPU>(n, red) < need) col = c;
  }
  return Key(val, col);
}

// (What alternatives cost beside the statistics, 2048 rows of 32768 bf16: 28 us with none, 31 with 1,
// 33 with 32, 38 with 64; a single row of 262144: 4.8 us with none, 9.6 with 20, most of it the steps that
// wait for each other in the two kernels.  The bisection reads a unit up to 57 times, with two barriers each
// time: constant rows, or rows where fewer than k columns are left above a mask of one finite value -- mask
// with -inf -- take 15 to 60 times as long: 32000 x 500 f32 with 8 alternatives 544 instead of 16.6 us, 64 x
// 131072 bf16 with 20 545 instead of 12.8, 2048 x 32768 bf16 with 64 2165 instead of 35.8.)
//
// Puts the unit's K largest elements in order and hands (place, key) to `out`, once per place from
// some lane; places without an element get key 0.  `threshold`: at least k of the unit's elements
// reach it, or it is -inf or NaN.  `collect`: Collect or CollectUnit of the elements that reach a value.
template <int TPU, class COLLECT, class MEM, class OUT>
__device__ inline void SelectTop(COLLECT collect, const MEM &mem, Scratch<TPU> &s, float threshold, int k, OUT out) {
  constexpr int kW = TPU / 64, kList = Scratch<TPU>::kList;
  const int tid = UnitLane<TPU>();
  const float floor_v = fmaxf(threshold, kLowest);  // (-inf is no alternative)
  collect(floor_v);
  if (TPU > 64)
    for (int a = tid; a < kMaxRanked; a += TPU) s.place[a] = 0;
  UnitSync<TPU>();
  int end[kW];  // of the waves' lists, one after the other
  auto count = [&] {
    bool over = false;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      end[w] = s.count[w] + (w ? end[w - 1] : 0);
      over |= s.count[w] > kList;
    }
    return over || end[kW - 1] > kMaxRanked;
  };
  if (count()) {
    UnitSync<TPU>();
    const uint64_t kth = KthElement<TPU>(mem, s.count, floor_v, k);
    Collect<TPU>(mem, s, floor_v, [=](float v, int i) { return v >= floor_v && Key(v, i) >= kth; });
    UnitSync<TPU>();
    count();
  }
  const int n = end[kW - 1];
  if (TPU == 64) {
    for (int a = tid; a < n; a += 64) {
      const uint64_t mine = s.cand[0][a];
      int place = 0;
#pragma unroll 4
      for (int b = 0; b < n; ++b) place += s.cand[0][b] > mine ? 1 : 0;
      if (place < k) out(place, mine);
    }
  } else {
    // each wave counts, for every candidate, those of its own list that are ahead
    const int lane = threadIdx.x & 63, own = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int own_n = s.count[own];
    auto candidate = [&](int a) {  // the a-th of all waves' lists
      int w = 0, first = 0;
#pragma unroll
      for (int x = 0; x < kW - 1; ++x) {
        w = a >= end[x] ? x + 1 : w;
        first = a >= end[x] ? end[x] : first;
      }
      return s.cand[w][a - first];
    };
    auto ahead = [&](uint64_t mine) {
      int place = 0;
#pragma unroll 4
      for (int b = 0; b < own_n; ++b) place += s.cand[own][b] > mine ? 1 : 0;
      return place;
    };
    if (n <= 64) {  // (nearly always, up to 32 alternatives: a candidate a lane)
      const uint64_t mine = lane < n ? candidate(lane) : 0;
      const int place = ahead(mine);
      if (place && lane < n) atomicAdd(&s.place[lane], place);
      __syncthreads();
      if (tid < n && s.place[tid] < k) out(s.place[tid], mine);
    } else {
      for (int a = lane; a < n; a += 64) {
        const int place = ahead(candidate(a));
        if (place) atomicAdd(&s.place[a], place);
      }
      __syncthreads();
      for (int a = tid; a < n; a += TPU)
        if (s.place[a] < k) out(s.place[a], candidate(a));
    }
  }
  for (int a = n + tid; a < k; a += TPU) out(a, 0);
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
  float k2;            // log2(e) / temperature
  float *logp, *entropy, *stats, *top_v;
  int32_t *top_i;
  Partial *part;       // split rows: [rows][nseg], and [rows][nseg][k] alternatives
  uint64_t *part_top;
  const float *weights;  // a loss's, [rows] or null: the statistics of rows of weight 0 are not wanted
};

__device__ inline int64_t IdAt(const void *ids, int32_t id64, size_t at) {
  return id64 ? static_cast<const int64_t *>(ids)[at] : static_cast<const int32_t *>(ids)[at];
}

// The row's token's logit: two loads that depend on each other, so they are issued with the row's own.
struct TokenLogit {
  bool there;
  float x;
};
template <class T>
__device__ inline TokenLogit LoadToken(const ScoresArgs &a, uint32_t row, const typename T::Store *x) {
  const int64_t tok = a.tokens ? IdAt(a.tokens, a.token64, row) : -1;
  const bool there = tok >= 0 && tok < a.r.vocab;
  return {there, there ? T::Load(x + tok) : 0.0f};
}

// A row's statistics are its maximum m and s = sum e_j.  (Not log s: 1 / s is what the gradient
// multiplies by, and a rounded log s of 10 would cost it 3 bits.)  A row without a finite value has
// m = -inf and s = 0; what is taken relative to its maximum is then taken relative to Base(m) = 0.
__device__ inline float Base(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ inline float LogSum(float s0) { return s0 == 0.0f ? 0.0f : logf(s0); }

// A unit's s0 and s1 = sum e_j log2(e_j) without what the rounding of the exponents' c added to them
// (Exponent).  With a finite maximum the sum is 1 for it and what the others add, so at least 1, and s1 at most 0:
// no log-probability above 0, no entropy below.  (NaN stays.)
__device__ inline float Corrected0(float s0, const Exponent &e, float m) {
  return m == -INFINITY ? s0 : fmaf(s0 - e.one, e.PerOne(), 1.0f);
}
__device__ inline float Corrected1(float s0, float s1, const Exponent &e) {
  return Min(fmaf(-e.delta, s0, s1) * e.PerOne(), 0.0f);
}

// H = log s - ln 2 s1 / s, two terms that are at least 0.  (What cancels is within s1: delta s0, where delta is
// at most 2^-24 of the maximum's own exponent.)
__device__ inline void WriteRowScores(const ScoresArgs &a, uint32_t row, TokenLogit tok, float m, float s0, float s1) {
  const float ls = LogSum(s0);
  if (a.tokens) a.logp[row] = tok.there ? (tok.x - Base(m)) - ls : 0.0f;
  a.entropy[row] = s0 == 0.0f ? 0.0f : ls - kLn2 * (s1 / s0);
  a.stats[2 * static_cast<size_t>(row)] = m;
  a.stats[2 * static_cast<size_t>(row) + 1] = s0;
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
  __device__ void operator()(int place, uint64_t key) const {
    v[place] = key ? (ValueOf(key) - base) - ls : -INFINITY;
    i[place] = key ? ColumnOf(key) : -1;
  }
};
// A row whose sum is NaN (NaN or +inf among its logits) has no alternatives.
template <int TPU>
__device__ inline void WriteNoTop(float *v, int32_t *i, float val, int k, int tid) {
  for (int a = tid; a < k; a += TPU) {
    v[a] = val;
    i[a] = -1;
  }
}

// Statistics, scores and alternatives of a unit: an element costs 1.5 operations for the maximum
// (v_maximum3 takes two, f16 and bf16 are unpacked first) and 7 (fma, exp2 -- a quarter of the rate --,
// two sums and their guard), so rows of bf16 keep the vector units busy for 62 % of a pass's cycles (86 % with
// 64 alternatives; profiles/frames_counters.csv): 268 M elements take 128 us, 4.2 TB/s, where a plain sum over the
// same bytes by the library runs at 4.0.
template <class T, int NCH, int TPU, bool SPLIT, bool ENT, bool TOP>
__global__ __launch_bounds__(kThreads<TPU>, (kOccupancy<TPU, NCH>)) void ScoresKernel(const ScoresArgs a) {
  __shared__ Scratch<TPU> scratch[TOP || TPU > 64 ? kUnits<TPU> : 1];
  const int tid = UnitLane<TPU>();
  const uint32_t unit = UnitNumber<TPU>();
  if (TPU < kBlock && unit >= a.r.rows) return;
  Scratch<TPU> &s = scratch[TOP || TPU > 64 ? UnitInBlock<TPU>() : 0];
  const Unit u = GetUnit(a.r, unit);
  if (u.skip) {
    if (!SPLIT) WriteRowNothing<TPU>(a, u.row, tid);
    return;  // (split: the joining kernel writes, and uses no part of such a row)
  }
  if (SPLIT && !ENT && a.weights && a.weights[u.row] == 0.0f) return;  // (a loss's statistics: as well)
  const typename T::Store *x = RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u);
  U4 r[NCH];
  LoadUnit<T, NCH, TPU>(x + u.lo, u.n, tid, r);
  TokenLogit tok{false, 0.0f};
  if (!SPLIT) tok = LoadToken<T>(a, u.row, x);

  // the maxima of a lane's 16 bytes, of its even and its odd columns, and of all
  float cm[NCH], g[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    cm[c] = -INFINITY;
    if (!Used<T, TPU>(c, u.n)) continue;
    float half[2] = {T::Get(r[c], 0), T::Get(r[c], 1)};
#pragma unroll
    for (int j = 2; j < T::kVec; ++j) half[j & 1] = Max(half[j & 1], T::Get(r[c], j));
    cm[c] = Max(half[0], half[1]);
    g[0] = Max(g[0], half[0]);
    g[1] = Max(g[1], half[1]);
  }
  const float lane_max = Max(g[0], g[1]);
  if (TOP && TPU > 64) s.group_max[tid] = lane_max;
  const float m = UnitMax<TPU>(lane_max, s.red[0]);
  const float base = Base(m);

  NewPass(r);
  const Exponent exponent(base, a.k2);
  float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    if (!Used<T, TPU>(c, u.n)) continue;
    s0 += PairSum<T::kVec>([&](int j) {
      const float t = exponent(T::Get(r[c], j)), e = __builtin_amdgcn_exp2f(t);
      // (t is -inf for a masked column: 0 * -inf would be NaN)
      if (ENT) s1 = fmaf(e, fmaxf(t, kLowest), s1);
      return e;
    });
  }
  s0 = WaveSum(s0);
  if (ENT) s1 = WaveSum(s1);
  if (TPU > 64) {
    if ((threadIdx.x & 63) == 0) {
      s.red[1][threadIdx.x >> 6] = s0;
      if (ENT) s.red[2][threadIdx.x >> 6] = s1;
    }
    __syncthreads();
    s0 = SumOf<TPU>(s.red[1]);
    if (ENT) s1 = SumOf<TPU>(s.red[2]);
  }
  if (ENT) s1 = Corrected1(s0, s1, exponent);
  s0 = Corrected0(s0, exponent, m);

  if (SPLIT) {
    if (tid == 0) a.part[unit] = Partial{m, s0, s1, 0.0f};
  } else if (tid == TPU - 1) {  // (not the wave that the threshold is up to)
    WriteRowScores(a, u.row, tok, m, s0, s1);
  }
  if (TOP) {
    const size_t at = (SPLIT ? static_cast<size_t>(unit) : static_cast<size_t>(u.row)) * a.k;
    if (isnan(s0)) {  // (the same in all lanes of the unit; split: the joining kernel sees the sum)
      if (!SPLIT) WriteNoTop<TPU>(a.top_v + at, a.top_i + at, s0, a.k, tid);
      return;
    }
    NewPass(r);
    const float threshold = GroupThreshold<TPU>(g, s, a.k);
    auto collect = [&](float floor_v) { CollectUnit<T, NCH, TPU>(r, cm, u.lo, u.n, s, floor_v); };
    const MemSource<T, TPU> mem{x + u.lo, u.lo, u.n, tid};
    if (SPLIT) {
      uint64_t *list = a.part_top + at;
      SelectTop<TPU>(collect, mem, s, threshold, a.k, [=](int place, uint64_t key) { list[place] = key; });
    } else {
      SelectTop<TPU>(collect, mem, s, threshold, a.k, TopWriter{a.top_v + at, a.top_i + at, base, LogSum(s0)});
    }
  }
}

// A row's statistics from its segments' (the whole workgroup).  `mine`: the thread's first part, loaded
// before (or one that adds nothing).
__device__ inline Partial FirstPartial(const Partial *part, int nseg) {
  return static_cast<int>(threadIdx.x) < nseg ? part[threadIdx.x] : Partial{-INFINITY, 0.0f, 0.0f, 0.0f};
}
__device__ inline void JoinPartials(const Partial *part, Partial mine, int nseg, float k2, float (*red)[kWaves],
                                    float *m_out, float *s0_out, float *s1_out) {
  float m = mine.m;
  for (int i = threadIdx.x + kBlock; i < nseg; i += kBlock) m = Max(m, part[i].m);
  m = UnitMax<kBlock>(m, red[0]);
  const float base = Base(m);
  float s0 = 0.0f, s1 = 0.0f;
  auto add = [&](const Partial &p) {
    const float t = (Base(p.m) - base) * k2, f = __builtin_amdgcn_exp2f(t);
    // (a segment that adds nothing may have any maximum: its products are not formed)
    if (f != 0.0f && p.s0 != 0.0f) {
      s0 = fmaf(f, p.s0, s0);
      s1 += f * fmaf(t, p.s0, p.s1);
    }
  };
  add(mine);
  for (int i = threadIdx.x + kBlock; i < nseg; i += kBlock) add(part[i]);
  s0 = WaveSum(s0);
  s1 = WaveSum(s1);
  if ((threadIdx.x & 63) == 0) {
    red[1][threadIdx.x >> 6] = s0;
    red[2][threadIdx.x >> 6] = s1;
  }
  __syncthreads();
  *m_out = m;
  *s0_out = SumOf<kBlock>(red[1]);
  *s1_out = SumOf<kBlock>(red[2]);
}

// One workgroup a row.  It is as long as the loads that wait for each other, so the parts, the token's
// logit and (up to kHeld a thread) the lists are all loaded at once.
constexpr int kHeld = 8;
template <class T, bool TOP>
__global__ __launch_bounds__(kBlock) void ScoresJoinKernel(const ScoresArgs a) {
  __shared__ Scratch<kBlock> s;
  const int tid = threadIdx.x;
  const Unit u = GetUnit(a.r, blockIdx.x * static_cast<uint32_t>(a.r.nseg));
  if (u.skip) {
    WriteRowNothing<kBlock>(a, u.row, tid);
    return;
  }
  const int nseg = a.r.nseg, k = a.k;
  const Partial *part = a.part + static_cast<size_t>(u.row) * nseg;
  const Partial mine = FirstPartial(part, nseg);
  const ListSource list{a.part_top + static_cast<size_t>(u.row) * nseg * k, nseg, k, tid};
  HeldSource<kHeld> held;
  const bool hold = nseg * k <= kHeld * kBlock;
  if (TOP && hold) held.Load(list);
  const TokenLogit tok = LoadToken<T>(a, u.row, RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u));
  if (TOP) {
    float most = -INFINITY;
    auto more = [&](float v, int) { most = fmaxf(most, v); };
    if (hold) {
      held.Each(0.0f, more);
    } else {
      list.Each(0.0f, more);
    }
    s.group_max[tid] = most;
  }
  float m, s0, s1;
  JoinPartials(part, mine, nseg, a.k2, s.red, &m, &s0, &s1);
  if (tid == 0) WriteRowScores(a, u.row, tok, m, s0, s1);
  if (TOP) {
    float *tv = a.top_v + static_cast<size_t>(u.row) * k;
    int32_t *ti = a.top_i + static_cast<size_t>(u.row) * k;
    if (isnan(s0)) {
      WriteNoTop<kBlock>(tv, ti, s0, k, tid);
      return;
    }
    const float none[2] = {};
    const float threshold = GroupThreshold<kBlock>(none, s, k);
    const TopWriter out{tv, ti, Base(m), LogSum(s0)};
    SelectTop<kBlock>(
        [&](float floor_v) {
          auto reaches = [=](float v, int) { return v >= floor_v; };
          if (hold) {
            Collect<kBlock>(held, s, floor_v, reaches);
          } else {
            Collect<kBlock>(list, s, floor_v, reaches);
          }
        },
        list, s, threshold, k, out);
  }
}

// ---- scores of short rows --------------------------------------------------------------------
// Rows of up to 2 KiB: a wave takes four, 16 lanes (one DPP row) each.  What such a row costs is not
// its bytes but the steps that are taken once a row -- reductions, threshold, ranking --, and these
// serve four rows here: 24000 rows of 500 f32 with 8 alternatives 14.5 us (10.5 without), and 21.4 (12.4)
// with a wave a row.  More than 16 alternatives need the 64 groups of a whole wave (21.0 us with 17).

// The k-th largest (k <= 16) of 16 lanes' pairs, in all lanes.
__device__ inline float RowKthLargest(float a, float b, int k) {
  a = RowSort(a);
  b = RowSort(b);
  // the 16 largest of both are the larger of the l-th and the (15 - l)-th: a bitonic sequence
  a = RowMerge(Max(a, Move<0x140>(b)));
  return OfLane(a, (threadIdx.x & 48) + k - 1);
}

constexpr int kShortTop = 16;  // alternatives
constexpr int kShortCap = 64;  // candidates a row

// KthElement for 16 lanes (a row's lanes are active together or not at all).
template <class T>
__device__ __noinline__ uint64_t ShortKthElement(const typename T::Store *p, int n, float floor_v, int k) {
  const int l = threadIdx.x & 15;
  auto count = [&](auto pred) {
    int c = 0;
    for (int i = l; i < n; i += 16) c += pred(T::Load(p + i), i) ? 1 : 0;
    return RowSum(c);
  };
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = t | (1u << bit);
    if (count([=](float v, int) { return v >= floor_v && OrderKey(v) >= c; }) >= k) t = c;
  }
  const float val = KeyValue(t);
  const int need = k - count([=](float v, int) { return v > val; });
  int col = 0;
  for (int bit = 11; bit >= 0; --bit) {  // (columns < 2^11)
    const int c = col | (1 << bit);
    if (count([=](float v, int i) { return v == val && i < c; }) < need) col = c;
  }
  return Key(val, col);
}
// Sum over a row's lanes up to and with one's own.
__device__ inline int RowPrefix(int v) {
  v += MoveI<0x111>(v);  // row_shr:1
  v += MoveI<0x112>(v);
  v += MoveI<0x114>(v);
  return v + MoveI<0x118>(v);
}

template <class T, int NCH, bool TOP>
__global__ __launch_bounds__(kBlock) void ScoresShortKernel(const ScoresArgs a) {
  __shared__ uint64_t lists[TOP ? kBlock / 16 : 1][TOP ? kShortCap : 1];
  __shared__ uint8_t chunk_lists[TOP ? kBlock / 16 : 1][TOP ? kShortCap : 1];
  const int l = UnitLane<16>();
  const uint32_t row = UnitNumber<16>();
  if (row >= a.r.rows) return;
  const Unit u = GetUnit(a.r, row);
  if (u.skip) {
    WriteRowNothing<16>(a, row, l);
    return;
  }
  const typename T::Store *x = RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u);
  const int n = a.r.vocab;
  U4 r[NCH];
  LoadUnit<T, NCH, 16>(x, n, l, r);
  const TokenLogit tok = LoadToken<T>(a, row, x);
  // the maxima of a lane's 16 bytes, and of the even and the odd ones of these
  float cm[NCH], half[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    cm[c] = -INFINITY;
    if (!Used<T, 16>(c, n)) continue;
    cm[c] = T::Get(r[c], 0);
#pragma unroll
    for (int j = 1; j < T::kVec; ++j) cm[c] = Max(cm[c], T::Get(r[c], j));
    half[c & 1] = Max(half[c & 1], cm[c]);
  }
  const float lane_max = Max(half[0], half[1]);
  const float m = RowMax(lane_max), base = Base(m);
  NewPass(r);
  const Exponent exponent(base, a.k2);
  float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    if (!Used<T, 16>(c, n)) continue;
    const U4 v = r[c];  // (the array itself, caught by reference, would stay in memory)
    s0 += PairSum<T::kVec>([&](int j) {
      const float t = exponent(T::Get(v, j)), e = __builtin_amdgcn_exp2f(t);
      s1 = fmaf(e, fmaxf(t, kLowest), s1);
      return e;
    });
  }
  s0 = RowSum(s0);
  s1 = RowSum(s1);
  s1 = Corrected1(s0, s1, exponent);
  s0 = Corrected0(s0, exponent, m);
  const float ls = LogSum(s0);
  if (l == 0) WriteRowScores(a, row, tok, m, s0, s1);
  if (!TOP) return;

  const int k = a.k;
  const TopWriter out{a.top_v + static_cast<size_t>(row) * k, a.top_i + static_cast<size_t>(row) * k, base, ls};
  if (isnan(s0)) {
    WriteNoTop<16>(out.v, out.i, s0, k, l);
    return;
  }
  // The lane's 16 bytes with a candidate among them, listed; then one lane takes each, from memory
  // (a register cannot be chosen at run time), and lists its candidates.
  const float floor_v = Max(RowKthLargest(half[0], half[1], k), kLowest);
  uint64_t *list = lists[threadIdx.x >> 4];
  uint32_t hit = 0;
#pragma unroll
  for (int c = 0; c < NCH; ++c) hit |= cm[c] >= floor_v ? 1u << c : 0u;
  const int hits = __popc(hit), upto = RowPrefix(hits), listed = RowSum(hits);
  int count = 0;
  if (listed <= kShortCap) {
    uint8_t *chunks = chunk_lists[threadIdx.x >> 4];
    for (int at = upto - hits; hit; hit &= hit - 1, ++at) chunks[at] = static_cast<uint8_t>((__ffs(hit) - 1) * 16 + l);
    UnitSync<64>();
    for (int i = 0; i < listed; i += 16) {  // (mostly once)
      const bool have = i + l < listed;
      const int e = (have ? chunks[i + l] : 0) * T::kVec, first = FirstCol<T>(e, n);
      // (a row of less than 16 bytes: lane 0 has it all)
      const U4 raw = n >= T::kVec ? *reinterpret_cast<const typename T::Vec *>(x + first) : r[0];
      uint32_t in = 0;
#pragma unroll
      for (int j = 0; j < T::kVec; ++j)
        in |= have && first + j >= e && T::Get(raw, j) >= floor_v ? 1u << j : 0u;
      const int some = __popc(in);
      int at = count + RowPrefix(some) - some;
#pragma unroll
      for (int j = 0; j < T::kVec; ++j) {
        if (in & (1u << j)) {
          if (at < kShortCap) list[at] = Key(T::Get(raw, j), first + j);
          ++at;
        }
      }
      count += RowSum(some);
    }
  }
  if (listed > kShortCap || count > kShortCap) {  // many equal values: exactly the k, found by bisection
    const uint64_t kth = ShortKthElement<T>(x, n, floor_v, k);
    UnitSync<64>();
    int pos = 0;
    for (int i0 = 0; i0 < n; i0 += 16) {
      const float v = i0 + l < n ? T::Load(x + i0 + l) : -INFINITY;
      const uint64_t key = Key(v, i0 + l);
      const int in = v >= floor_v && key >= kth ? 1 : 0;
      const int upto_me = RowPrefix(in);  // (all of the row's lanes take part)
      if (in) list[pos + upto_me - 1] = key;
      pos += RowSum(in);
    }
    count = k;
  }
  UnitSync<64>();
  for (int b = l; b < count; b += 16) {
    const uint64_t mine = list[b];
    int place = 0;
#pragma unroll 4
    for (int o = 0; o < count; ++o) place += list[o] > mine ? 1 : 0;
    if (place < k) out(place, mine);
  }
  for (int b = count + l; b < k; b += 16) out(b, 0);
}

// ---- gradients -----------------------------------------------------------------------------------

struct GradOut {
  void *dx;
  int64_t batch_stride, row_stride;
};

// Writes g[0 .. kVec) = f(r[c], first column in the unit) for a unit's elements.
template <class T, int NCH, int TPU, class F>
__device__ inline void StoreUnit(typename T::Store *p, int n, int tid, const U4 (&r)[NCH], F f) {
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    if (!Used<T, TPU>(c, n)) continue;
    const int e = (c * TPU + tid) * T::kVec;
    if (e < n) {
      const int first = FirstCol<T>(e, n);
      float g[T::kVec];
      f(r[c], first, g);
      if (e + T::kVec <= n) {
        *reinterpret_cast<typename T::Vec *>(p + e) = T::Pack(g);
      } else {  // (the columns in front are another lane's)
#pragma unroll
        for (int j = 0; j < T::kVec; ++j)
          if (first + j >= e && first + j < n) p[first + j] = T::Round(g[j]);
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

// dx_j = g_logp ([j = token] - p_j) - g_H p_j (log p_j + H).  With p_j = e_j / s, log p_j = ln 2 t_j -
// log s (t_j the exponent) that is e_j (A + B t_j) + g_logp [j = token]: A = (-g_logp - g_H (H - log s)) / s,
// B = -ln 2 g_H / s.  Bound by memory: 4096 rows of 65536 bf16 are read and written at 5.9 TB/s.
template <class T, int NCH, int TPU>
__global__ __launch_bounds__(kThreads<TPU>, (kOccupancy<TPU, NCH>)) void ScoresGradKernel(const ScoresGradArgs a) {
  const int tid = UnitLane<TPU>();
  const uint32_t unit = UnitNumber<TPU>();
  if (TPU < kBlock && unit >= a.r.rows) return;
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
  int64_t tok = a.tokens ? IdAt(a.tokens, a.token64, u.row) : -1;
  if (tok < 0 || tok >= a.r.vocab) tok = -1;
  const float gl = a.g_logp && tok >= 0 ? a.g_logp[u.row] : 0.0f;
  const float gh = a.g_entropy ? a.g_entropy[u.row] : 0.0f;
  const int at = tok < 0 ? -T::kVec : static_cast<int>(tok) - u.lo;  // (may be outside the unit)
  const Exponent exponent(m, kLog2e);
  const float inv = 1.0f / (exponent.one * s0), ls = logf(s0);
  const float B = -kLn2 * gh * inv;
  const float A = (a.g_entropy ? -gl - gh * (a.entropy[u.row] - ls) : -gl) * inv - B * exponent.delta;
  StoreUnit<T, NCH, TPU>(dx, u.n, tid, r, [=](const U4 &v, int first, float *g) {
#pragma unroll
    for (int j = 0; j < T::kVec; ++j) {
      const float t = exponent(T::Get(v, j));
      // (below -150 e is 0, and 0 times -inf would be NaN)
      g[j] = __builtin_amdgcn_exp2f(t) * fmaf(B, fmaxf(t, -256.0f), A);
    }
    if (static_cast<uint32_t>(at - first) < static_cast<uint32_t>(T::kVec)) {
#pragma unroll
      for (int j = 0; j < T::kVec; ++j) g[j] += first + j == at ? gl : 0.0f;
    }
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
// (SN slots a lane: 256 in a unit of a wave or more, 16 or 64 in one of 16 lanes.)
template <int TPU, int SN>
constexpr int kListed = TPU * SN < kMaxSlots ? TPU * SN : kMaxSlots;
template <int TPU, int SN>
struct TeacherList {
  int2 slot[kListed<TPU, SN>];  // id, and the bits of q
  float red[5][TPU < 64 ? 1 : TPU / 64];
};
template <int TPU, int SN>
struct Slots {
  int id[SN];   // -1: empty
  float u[SN];  // (logit - largest) / temperature
  float q[SN];
  float log_usum;
  bool any;
};

template <int TPU, int SN>
__device__ inline void LoadSlots(const DistillArgs &a, uint32_t row, int tid, Slots<TPU, SN> &t) {
#pragma unroll
  for (int i = 0; i < SN; ++i) {
    t.id[i] = -1;
    t.u[i] = -INFINITY;
    const int k = i * TPU + tid;
    if (k < a.slots) {
      const size_t at = static_cast<size_t>(row) * a.slots + k;
      const int64_t id = IdAt(a.ids, a.id64, at);
      if (id >= 0 && id < a.r.vocab) {
        t.id[i] = static_cast<int>(id);
        t.u[i] = TeacherValue(a, at);
      }
    }
  }
}
// q = softmax(u / temperature) over the filled slots.
template <int TPU, int SN>
__device__ inline void SoftmaxSlots(const DistillArgs &a, Slots<TPU, SN> &t, TeacherList<TPU, SN> &list, int tid) {
  float um = -INFINITY, sum = 0.0f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < SN; ++i) {
    um = fmaxf(um, t.u[i]);
    nan |= isnan(t.u[i]);
  }
  um = UnitMax<TPU>(nan ? INFINITY : um, list.red[0]);  // (inf - inf below: NaN for the whole row)
  t.any = um != -INFINITY;
#pragma unroll
  for (int i = 0; i < SN; ++i) {
    t.u[i] = (t.u[i] - Base(um)) * a.inv_t;
    t.q[i] = um == INFINITY && t.id[i] >= 0 ? NAN : expf(t.u[i]);
    sum += t.q[i];
  }
  sum = UnitSum<TPU>(sum, list.red[1]);
  t.log_usum = logf(sum);
#pragma unroll
  for (int i = 0; i < SN; ++i) {
    t.q[i] = t.q[i] / sum;
    const int k = i * TPU + tid;
    if (k < a.slots) {
      list.slot[k] = int2{t.id[i], __float_as_int(t.q[i])};
    }
  }
  UnitSync<TPU>();
}

// w sum_k q_k (log q_k - log p_k), log p_k = (x_k - m) / temperature - ls; xs: the students' logits at the slots.
template <int TPU, int SN>
__device__ inline float Divergence(const DistillArgs &a, const Slots<TPU, SN> &t, const float (&xs)[SN], float m,
                                   float ls, float w, float *red) {
  // No product of two or three of the factors stays in f32's range (a logit of the type's lowest value times
  // 1 / temperature, a small weight times a small q -- and that product must not be 0 where the student rules
  // the token out, d = -inf).  So w is taken apart, (log q - log p) carries 2^-64 and q 2^40, exactly: the
  // first is below 2^85 then and the second at least 2^-110, and one ldexp rounds the term.
  const float w40 = __builtin_amdgcn_frexp_mantf(w) * 0x1p40f, inv_t64 = a.inv_t * 0x1p-64f;
  const int exponent = __builtin_amdgcn_frexp_expf(w) + 24;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < SN; ++i) {
    const float d = xs[i] - Base(m), each = (t.u[i] - t.log_usum) + ls;
    if (t.id[i] >= 0 && t.q[i] != 0.0f)
      sum += __builtin_amdgcn_ldexpf(w40 * t.q[i] * fmaf(-inv_t64, d, each * 0x1p-64f), exponent);
  }
  return UnitSum<TPU>(sum, red);
}

// weight upstream / temperature of a row: the product of two of them may leave f32's range where that of all
// three does not, so it is formed in 64 bits.
__device__ inline float GradFactor(const DistillArgs &a, uint32_t row, float w) {
  const float up = a.upstream ? a.upstream[row] : 1.0f;
  return static_cast<float>(static_cast<double>(w) * a.inv_t * up);
}

// Writes a unit's gradient: coef (p_j - sum of the q of the slots that name column j).  The slots'
// columns are written again behind the others, by one lane each (slots that name one column write
// the same value).
template <class T, int NCH, int TPU, int SN>
__device__ inline void WriteDistillGrad(const DistillArgs &a, const Unit &u, const U4 (&r)[NCH], const Slots<TPU, SN> &t,
                                        const float (&xs)[SN], const TeacherList<TPU, SN> &list, float m,
                                        float s0, float coef, int tid) {
  typename T::Store *dx =
      const_cast<typename T::Store *>(RowPtr<T>(a.o.dx, a.o.batch_stride, a.o.row_stride, u)) + u.lo;
  const Exponent exponent(Base(m), a.k2);
  // (a student without a finite logit gives nothing any probability)
  const float inv = s0 == 0.0f ? 0.0f : 1.0f / (exponent.one * s0), scale = coef * inv;
  StoreUnit<T, NCH, TPU>(dx, u.n, tid, r, [=](const U4 &v, int, float *g) {
#pragma unroll
    for (int j = 0; j < T::kVec; ++j) g[j] = scale * __builtin_amdgcn_exp2f(exponent(T::Get(v, j)));
  });
  UnitSync<TPU>();
  bool mine[SN], any = false;
  float q[SN];
#pragma unroll
  for (int i = 0; i < SN; ++i) {
    const int at = t.id[i] - u.lo;
    mine[i] = t.id[i] >= 0 && at >= 0 && at < u.n;
    any |= mine[i];
    q[i] = 0.0f;
  }
  if (!__ballot(any)) return;
#pragma unroll 4
  for (int k = 0; k < a.slots; ++k) {
    const int2 slot = list.slot[k];
#pragma unroll
    for (int i = 0; i < SN; ++i) q[i] += slot.x == t.id[i] ? __int_as_float(slot.y) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < SN; ++i)
    if (mine[i]) dx[t.id[i] - u.lo] = T::Round(coef * (__builtin_amdgcn_exp2f(exponent(xs[i])) * inv - q[i]));
}

// The students' logits at a lane's slots.
template <class T, int TPU, int SN>
__device__ inline void LoadAtSlots(const typename T::Store *x, const Slots<TPU, SN> &t, float (&xs)[SN]) {
#pragma unroll
  for (int i = 0; i < SN; ++i) xs[i] = t.id[i] >= 0 ? T::Load(x + t.id[i]) : 0.0f;
}

// Whole rows: loss, and with GRAD the gradient from the registers that the statistics were taken of:
// 4096 rows of 131072 bf16 in 470 us, 4.6 TB/s of one read and one write, where statistics and gradient
// in two kernels, three passes over memory, take 622.  (A row of 256 KiB fills half a CU's registers, so
// its loads, sums and stores do not overlap with another's on the same CU; other CUs' do.)
template <class T, int NCH, int TPU, int SN, bool GRAD>
__global__ __launch_bounds__(kThreads<TPU>, (kOccupancy<TPU, NCH, GRAD ? SN : 1>)) void DistillKernel(const DistillArgs a) {
  __shared__ TeacherList<TPU, SN> lists[kUnits<TPU>];
  const int tid = UnitLane<TPU>();
  const uint32_t unit = UnitNumber<TPU>();
  if (TPU < kBlock && unit >= a.r.rows) return;
  const Unit u = GetUnit(a.r, unit);
  const float w = u.skip ? 0.0f : a.weights ? a.weights[u.row] : 1.0f;
  TeacherList<TPU, SN> &list = lists[UnitInBlock<TPU>()];
  Slots<TPU, SN> t;
  t.any = false;
  const typename T::Store *x = RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u);
  U4 r[NCH];
  float xs[SN];
  if (w != 0.0f) {
    LoadSlots<TPU, SN>(a, u.row, tid, t);
    LoadUnit<T, NCH, TPU>(x, u.n, tid, r);
    LoadAtSlots<T, TPU, SN>(x, t, xs);
    SoftmaxSlots<TPU, SN>(a, t, list, tid);
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
  float m = -INFINITY;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    if (!Used<T, TPU>(c, u.n)) continue;
#pragma unroll
    for (int j = 0; j < T::kVec; ++j) m = Max(m, T::Get(r[c], j));
  }
  m = UnitMax<TPU>(m, list.red[2]);
  NewPass(r);
  const Exponent exponent(Base(m), a.k2);
  float s0 = 0.0f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    if (!Used<T, TPU>(c, u.n)) continue;
    s0 += PairSum<T::kVec>([&](int j) { return __builtin_amdgcn_exp2f(exponent(T::Get(r[c], j))); });
  }
  s0 = Corrected0(UnitSum<TPU>(s0, list.red[3]), exponent, m);
  const float ls = LogSum(s0);
  const float loss = Divergence<TPU, SN>(a, t, xs, m, ls, w, list.red[4]);
  if (tid == 0) {
    if (a.loss) a.loss[u.row] = loss;
    if (a.stats) {
      a.stats[2 * static_cast<size_t>(u.row)] = m;
      a.stats[2 * static_cast<size_t>(u.row) + 1] = s0;
    }
  }
  if (GRAD) {
    NewPass(r);
    const float coef = GradFactor(a, u.row, w);
    WriteDistillGrad<T, NCH, TPU, SN>(a, u, r, t, xs, list, m, s0, coef, tid);
  }
}

// Split rows: the statistics of a row from its segments', and its loss.
template <class T>
__global__ __launch_bounds__(kBlock) void DistillJoinKernel(const DistillArgs a) {
  __shared__ TeacherList<kBlock, 1> list;
  __shared__ float red[3][kWaves];
  const int tid = threadIdx.x;
  const Unit u = GetUnit(a.r, blockIdx.x * static_cast<uint32_t>(a.r.nseg));
  const float w = u.skip ? 0.0f : a.weights ? a.weights[u.row] : 1.0f;
  const Partial *part = a.part + static_cast<size_t>(u.row) * a.r.nseg;
  const Partial mine = FirstPartial(part, a.r.nseg);
  Slots<kBlock, 1> t;
  t.any = false;
  float xs[1];
  if (w != 0.0f) {
    LoadSlots<kBlock, 1>(a, u.row, tid, t);
    LoadAtSlots<T, kBlock, 1>(RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u), t, xs);
    SoftmaxSlots<kBlock, 1>(a, t, list, tid);
  }
  float m = 0.0f, s0 = 0.0f, loss = 0.0f;
  if (t.any) {
    float s1;
    JoinPartials(part, mine, a.r.nseg, a.k2, red, &m, &s0, &s1);
    loss = Divergence<kBlock, 1>(a, t, xs, m, LogSum(s0), w, list.red[4]);
  }
  if (tid == 0) {
    if (a.loss) a.loss[u.row] = t.any ? loss : 0.0f;
    a.stats[2 * static_cast<size_t>(u.row)] = m;
    a.stats[2 * static_cast<size_t>(u.row) + 1] = s0;
  }
}

// The gradient of rows or segments whose statistics are known.
template <class T, int NCH, int TPU, int SN>
__global__ __launch_bounds__(kThreads<TPU>, (kOccupancy<TPU, NCH>)) void DistillGradKernel(const DistillArgs a) {
  __shared__ TeacherList<TPU, SN> lists[kUnits<TPU>];
  const int tid = UnitLane<TPU>();
  const uint32_t unit = UnitNumber<TPU>();
  if (TPU < kBlock && unit >= a.r.rows) return;
  const Unit u = GetUnit(a.r, unit);
  const float w = u.skip ? 0.0f : a.weights ? a.weights[u.row] : 1.0f;
  TeacherList<TPU, SN> &list = lists[UnitInBlock<TPU>()];
  Slots<TPU, SN> t;
  t.any = false;
  const typename T::Store *x = RowPtr<T>(a.r.x, a.r.batch_stride, a.r.row_stride, u);
  U4 r[NCH];
  float xs[SN];
  if (w != 0.0f) {
    LoadSlots<TPU, SN>(a, u.row, tid, t);
    LoadUnit<T, NCH, TPU>(x + u.lo, u.n, tid, r);
    LoadAtSlots<T, TPU, SN>(x, t, xs);
    // (its barriers stand between every lane's loads of the slots' logits and the first stores: the
    // gradient may be written over the logits)
    SoftmaxSlots<TPU, SN>(a, t, list, tid);
  }
  if (!t.any) {
    StoreZeros<T, NCH, TPU>(
        const_cast<typename T::Store *>(RowPtr<T>(a.o.dx, a.o.batch_stride, a.o.row_stride, u)) + u.lo, u.n, tid);
    return;
  }
  const float m = a.stats[2 * static_cast<size_t>(u.row)], s0 = a.stats[2 * static_cast<size_t>(u.row) + 1];
  const float coef = GradFactor(a, u.row, w);
  WriteDistillGrad<T, NCH, TPU, SN>(a, u, r, t, xs, list, m, s0, coef, tid);
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
int Launch(void (*kernel)(ARGS), uint32_t blocks, const ARGS &args, void *stream, int threads = kBlock) {
  if (!blocks) return KD_OK;
  void *argv[] = {const_cast<ARGS *>(&args)};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3(blocks), dim3(threads), argv, 0,
                                       static_cast<hipStream_t>(stream));
  return e == hipSuccess ? KD_OK : HipFail("launch", e);
}

int64_t ElemBytes(int dtype) { return dtype == KD_DTYPE_F32 ? 4 : 2; }

// How rows are dealt out: TPU lanes a unit, up to NCH 16-byte loads each.  Both sides of each rule, in
// us (D: loss and gradient of bf16 rows with 64 slots; S: scores with 20 alternatives):
//   whole to 64 KiB         S 1 x 32768 7.2, in segments 9.2; D 8 x 32768 8.6 and 10.6; D 4096 x 32768
//                           115 and 176
//   1024 lanes, 128 KiB     D 64 x 65536 13.3, in segments 15.3; 16 x 65536 12.0 and 11.2; 4096 x 65536 219 and 334
//   1024 lanes, 256 KiB     D 256 x 131072 32.2, in segments 43.1; 128 x 131072 25.1 and 25.2; 64: 22.4 and 19.5
//                           (values alone are read once either way: 512 x 131072 41.7 and 29.4)
//   smaller segments for    S 8 x 131072 9.8 with 256 units and more, 10.7 with 64; D 8 x 131072 11.2 and 12.5; S 1 x
//   few rows                262144 9.6 and 10.3 (from 1024 units on the joining kernel's share grows: 16 x 131072
//                           10.1 with 512, 10.8 with 1024).  That kernel holds at most kHeld x 256
//                           alternatives in registers (1 x 262144 with 64: 14.1 with 32 units, 18.9 with 64)
struct Plan {
  int tpu, nch, seg_len, nseg;
};
enum Purpose {
  kValues,  // statistics, alternatives, losses
  kFused,   // loss and gradient
  kPieces,  // a gradient whose statistics are known: any part of a row by itself
};
Plan MakePlan(int64_t vocab, int dtype, int64_t rows, Purpose what, int top, bool narrow) {
  const int64_t bytes = vocab * ElemBytes(dtype), vec = 16 / ElemBytes(dtype);
  const int whole = static_cast<int>(vocab);
  // Short rows, four to a wave (the lists of a longer teacher take a wave's lanes: `narrow`).
  if (bytes <= 2048 && narrow) return {16, bytes <= 512 ? 2 : 8, whole, 1};
  if (bytes <= 2048) return {64, 2, whole, 1};
  if (bytes <= 8192) return {64, 8, whole, 1};
  if (bytes <= 32768) return {kBlock, 8, whole, 1};
  if (what != kPieces && bytes <= 65536) return {512, 8, whole, 1};
  if (what == kFused && bytes <= 131072 && rows >= 32) return {1024, 8, whole, 1};
  if (what == kFused && bytes <= 262144 && rows >= 128) return {1024, 16, whole, 1};
  Plan p{kBlock, 8, 0, 0};
  int64_t cap = 32768;
  while (cap > 4096 && rows * ((bytes + cap - 1) / cap) < 256 && 2 * top * ((bytes + cap - 1) / cap) <= kHeld * kBlock)
    cap /= 2;
  cap /= ElemBytes(dtype);
  p.nseg = static_cast<int>((vocab + cap - 1) / cap);
  // equal segments, whole vectors
  p.seg_len = static_cast<int>(((vocab + p.nseg - 1) / p.nseg + vec - 1) / vec * vec);
  p.nseg = static_cast<int>((vocab + p.seg_len - 1) / p.seg_len);
  return p;
}

int64_t NumBlocks(int64_t units, const Plan &p) {
  const int64_t per = std::max(kBlock / p.tpu, 1);
  return (units + per - 1) / per;
}

int CheckRows(const kd_frame_rows *r, Purpose what, Rows *out, Plan *plan, int64_t *rows, int top, bool narrow) {
  if (!r || r->batch < 0 || r->steps < 0) return SetError(KD_E_INVALID, "bad argument: rows");
  if (r->dtype != KD_DTYPE_F32 && r->dtype != KD_DTYPE_F16 && r->dtype != KD_DTYPE_BF16)
    return SetError(KD_E_INVALID, "bad argument: dtype of the logits");
  if (r->vocab < 1 || r->vocab > kMaxVocab)
    return SetError(KD_E_INVALID, "bad argument: vocab must be between 1 and 2^24");
  if (r->batch > INT32_MAX || r->steps > INT32_MAX || r->batch * r->steps > INT32_MAX)
    return SetError(KD_E_INVALID, "bad argument: more than 2^31 - 1 rows");
  *rows = r->batch * r->steps;
  *plan = MakePlan(r->vocab, r->dtype, *rows, what, top, narrow);
  // (a grid has fewer than 2^32 threads, those of its last workgroup included)
  if (NumBlocks(*rows * plan->nseg, *plan) * std::max(plan->tpu, kBlock) > (int64_t(1) << 32) - 1)
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

// Rows in memory, in bytes from `base` on: n[1] groups, s[1] apart, of n[0] runs of `width`, s[0] apart.
// (Strides may be anything: 128 bits hold what they add up to.)
typedef __int128 Wide;
struct Region {
  uintptr_t base;
  int64_t n[2];
  Wide s[2], width;

  Region(const void *p, const kd_frame_rows *r, int64_t batch_stride, int64_t row_stride)
      : base(reinterpret_cast<uintptr_t>(p)), n{r->steps, r->batch}, width(r->vocab * ElemBytes(r->dtype)) {
    s[0] = Wide(row_stride) * ElemBytes(r->dtype);
    s[1] = Wide(batch_stride) * ElemBytes(r->dtype);
    for (int i = 0; i < 2; ++i)
      if (n[i] <= 1) s[i] = 0;  // (a stride that is never taken)
    if (n[0] <= 1 || (n[1] > 1 && s[0] > s[1])) {
      std::swap(n[0], n[1]);
      std::swap(s[0], s[1]);
    }
  }
  // Runs that touch or lie over each other are one.
  void Merge() {
    for (int i = 0; i < 2 && n[0] > 1 && s[0] <= width; ++i) {
      width += (n[0] - 1) * s[0];
      n[0] = n[1];
      s[0] = s[1];
      n[1] = 1;
      s[1] = 0;
    }
  }
  Wide Inner() const { return width + (n[0] - 1) * s[0]; }  // of a group
  Wide Span() const { return Inner() + (n[1] - 1) * s[1]; }
};
Wide FloorDiv(Wide a, Wide b) { return a / b - (a % b < 0); }  // (b > 0)
// First and last of the 0 <= i < n with lo < i * s + width and i * s < hi; none: first > last.
void Hits(Wide lo, Wide hi, Wide s, Wide width, int64_t n, Wide *first, Wide *last) {
  *first = n > 1 ? std::max(FloorDiv(lo - width, s) + 1, Wide(0)) : Wide(lo < width ? 0 : 1);
  *last = n > 1 ? std::min(FloorDiv(hi - 1, s), Wide(n - 1)) : Wide(hi > 0 ? 0 : -1);
}
// Whether bytes [at, at + bytes) meet any run of `g`, whose runs and groups lie one behind the other.
bool Meets(const Region &g, uintptr_t at, Wide bytes) {
  if (bytes <= 0) return false;
  const Wide lo = Wide(at) - Wide(g.base), hi = lo + bytes;
  Wide first, last, run, end;
  Hits(lo, hi, g.s[1], g.Inner(), g.n[1], &first, &last);
  if (first != last) return first < last;  // (none, or all that is between two groups' starts)
  Hits(lo - first * g.s[1], hi - first * g.s[1], g.s[0], g.width, g.n[0], &run, &end);
  return run <= end;
}
// Whether any byte of `x` is one of `g`, whose runs and groups lie one behind the other.
bool Meets(const Region &g, const Region &x) {
  if (Wide(x.base) + x.Span() <= Wide(g.base) || Wide(g.base) + g.Span() <= Wide(x.base)) return false;
  if (g.n[0] == x.n[0] && g.n[1] == x.n[1] && g.s[0] == x.s[0] && g.s[1] == x.s[1] && g.width == x.width) {
    // side by side in one tensor: some whole number of strides must lead from one to within the other
    const Wide delta = Wide(x.base) - Wide(g.base), inner = g.Inner();
    Wide j = 0, last = 0;
    if (g.n[1] > 1) {
      j = std::max(FloorDiv(-delta - inner, g.s[1]), Wide(1 - g.n[1]));
      last = std::min(FloorDiv(inner - delta, g.s[1]) + 1, Wide(g.n[1] - 1));
    }
    for (; j <= last; ++j) {
      const Wide off = delta + j * g.s[1];  // wanted: -width < off + i s < width, |i| < n
      Wide i = 0;
      if (g.n[0] > 1) i = std::min(std::max(FloorDiv(-g.width - off, g.s[0]) + 1, Wide(1 - g.n[0])), Wide(g.n[0] - 1));
      if (off + i * g.s[0] > -g.width && off + i * g.s[0] < g.width) return true;
    }
    return false;
  }
  for (int64_t j = 0; j < x.n[1]; ++j)
    for (int64_t i = 0; i < x.n[0]; ++i)
      if (Meets(g, static_cast<uintptr_t>(Wide(x.base) + j * x.s[1] + i * x.s[0]), x.width)) return true;
  return false;
}

struct Read {  // an array that a gradient's kernel reads
  const void *p;
  int64_t bytes;
  const char *what;
};

// A gradient's rows must not lie over each other, nor over anything that other units read while they are written.
// The logits themselves, element for element, will do: a unit has loaded its own before it stores, and nothing
// that it loads of another's is used.
int CheckGrad(const kd_frame_rows *r, void *dx, int64_t batch_stride, int64_t row_stride,
              std::initializer_list<Read> reads, GradOut *o) {
  if (!dx) return SetError(KD_E_INVALID, "bad argument: grad is NULL");
  if (reinterpret_cast<uintptr_t>(dx) % ElemBytes(r->dtype))
    return SetError(KD_E_INVALID, "bad argument: grad is not aligned to its type");
  Region g(dx, r, batch_stride, row_stride), x(r->logits, r, r->batch_stride, r->row_stride);
  if ((g.n[0] > 1 && g.s[0] < g.width) || (g.n[1] > 1 && g.s[1] < g.Inner()))
    return SetError(KD_E_INVALID, "bad argument: the gradient's rows overlap");
  g.Merge();
  x.Merge();
  // (each row in its own logits' place: regions that are alike may have their dimensions the other way round)
  const bool itself = dx == r->logits && (r->batch <= 1 || batch_stride == r->batch_stride) &&
                      (r->steps <= 1 || row_stride == r->row_stride);
  if (!itself) {
    if (Meets(g, x))
      return SetError(KD_E_INVALID, "bad argument: the gradient lies across the logits (some memory location is another "
                                    "element of theirs)");
  }
  for (const Read &a : reads)
    if (a.p && Meets(g, reinterpret_cast<uintptr_t>(a.p), a.bytes))
      return SetError(KD_E_INVALID, std::string("bad argument: the gradient lies across ") + a.what);
  o->dx = dx;
  o->batch_stride = batch_stride;
  o->row_stride = row_stride;
  return KD_OK;
}

uint32_t Blocks(const Rows &r, const Plan &p) {
  return static_cast<uint32_t>(NumBlocks(static_cast<int64_t>(r.rows) * r.nseg, p));
}

// f(T{}, NCH, TPU as constants) for a plan.
template <int N>
struct Int {
  static constexpr int value = N;
};
// Which units of short rows a kernel is made for.
enum ShortUnits { kNone, kBySixteen, kByWave, kByBoth };
template <Purpose WHAT, ShortUnits SHORT, class T, class F>
int ForPlan(const Plan &p, F f) {
  if constexpr (SHORT == kBySixteen || SHORT == kByBoth)
    if (p.tpu == 16) return p.nch == 2 ? f(T{}, Int<2>{}, Int<16>{}) : f(T{}, Int<8>{}, Int<16>{});
  if constexpr (SHORT == kByWave || SHORT == kByBoth)
    if (p.tpu == 64 && p.nch == 2) return f(T{}, Int<2>{}, Int<64>{});
  if (p.tpu == 64) return f(T{}, Int<8>{}, Int<64>{});
  if constexpr (WHAT != kPieces)
    if (p.tpu == 512) return f(T{}, Int<8>{}, Int<512>{});
  if constexpr (WHAT == kFused)
    if (p.tpu == 1024) return p.nch == 8 ? f(T{}, Int<8>{}, Int<1024>{}) : f(T{}, Int<16>{}, Int<1024>{});
  return f(T{}, Int<8>{}, Int<kBlock>{});
}
// f(SN as a constant): slots a lane.
constexpr int kShortSlots = 64;  // of a teacher of short rows
template <int TPU, class F>
int ForSlots(int slots, F f) {
  if constexpr (TPU == 16) return slots <= 16 ? f(Int<1>{}) : f(Int<4>{});
  else return f(Int<(TPU < kMaxSlots ? kMaxSlots / TPU : 1)>{});
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
      return Launch(ScoresKernel<T, 8, kBlock, true, ENT, TOP>, Blocks(a.r, plan), a, stream);
    } else {
      // (short rows of few alternatives are LaunchShort's: without alternatives no wave takes one)
      constexpr ShortUnits kShort = TOP ? kByWave : kNone;
      return ForPlan<kValues, kShort, T>(plan, [&](auto tt, auto nch, auto tpu) {
        return Launch(ScoresKernel<decltype(tt), decltype(nch)::value, decltype(tpu)::value, false, ENT, TOP>,
                      Blocks(a.r, plan), a, stream, kThreads<decltype(tpu)::value>);
      });
    }
  });
}

template <bool TOP>
int LaunchShort(const kd_frame_rows *rows, const ScoresArgs &a, const Plan &plan, void *stream) {
  return ForType(rows->dtype, [&](auto t) {
    using T = decltype(t);
    return plan.nch == 2 ? Launch(ScoresShortKernel<T, 2, TOP>, Blocks(a.r, plan), a, stream)
                         : Launch(ScoresShortKernel<T, 8, TOP>, Blocks(a.r, plan), a, stream);
  });
}

}  // namespace

extern "C" {

size_t kd_token_scores_workspace(const kd_frame_rows *rows, int32_t top) {
  Rows r;
  Plan p;
  int64_t n;
  if (top < 0 || top > kMaxTop || Guarded([&] { return CheckRows(rows, kValues, &r, &p, &n, top, top <= kShortTop); }) ||
      p.nseg == 1)
    return 0;
  const size_t units = static_cast<size_t>(n) * p.nseg;
  return Align(units * sizeof(Partial)) + units * top * sizeof(uint64_t);
}

int kd_token_scores(const kd_frame_rows *rows, const void *tokens, int32_t token_bytes, int32_t top, float *logp,
                    float *entropy, float *stats, float *top_logp, int32_t *top_ids, void *workspace,
                    size_t workspace_bytes, void *stream) {
  return Guarded([&]() -> int {
    ScoresArgs a{};
    Plan p;
    int64_t n;
    if (int rc = CheckRows(rows, kValues, &a.r, &p, &n, std::max(top, 0), top <= kShortTop)) return rc;
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
    if (p.tpu == 16) return top ? LaunchShort<true>(rows, a, p, stream) : LaunchShort<false>(rows, a, p, stream);
    if (p.nseg == 1)
      return top ? LaunchScores<false, true, true>(rows, a, p, stream)
                 : LaunchScores<false, true, false>(rows, a, p, stream);
    const size_t units = static_cast<size_t>(n) * p.nseg;
    char *ws = static_cast<char *>(workspace);
    a.part = reinterpret_cast<Partial *>(ws);
    a.part_top = reinterpret_cast<uint64_t *>(ws + Align(units * sizeof(Partial)));
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
    if (int rc = CheckRows(rows, kPieces, &a.r, &p, &n, 0, true)) return rc;
    if (tokens && token_bytes != 4 && token_bytes != 8)
      return SetError(KD_E_INVALID, "bad argument: token_bytes must be 4 or 8");
    if (!n) return KD_OK;
    if (!stats || (grad_entropy && !entropy)) return SetError(KD_E_INVALID, "bad argument: stats / entropy is NULL");
    if (int rc = CheckGrad(rows, grad, grad_batch_stride, grad_row_stride,
                           {{rows->lengths, 4 * rows->batch, "lengths"},
                            {tokens, n * token_bytes, "tokens"},
                            {stats, n * 8, "stats"},
                            {entropy, n * 4, "entropy"},
                            {grad_logp, n * 4, "grad_logp"},
                            {grad_entropy, n * 4, "grad_entropy"}},
                           &a.o))
      return rc;
    a.tokens = tokens;
    a.token64 = token_bytes == 8;
    a.stats = stats;
    a.entropy = entropy;
    a.g_logp = grad_logp;
    a.g_entropy = grad_entropy;
    DeviceGuard guard(rows->device);
    if (guard.error() != hipSuccess) return HipFail("hipSetDevice", guard.error());
    return ForType(rows->dtype, [&](auto t) {
      return ForPlan<kPieces, kBySixteen, decltype(t)>(p, [&](auto tt, auto nch, auto tpu) {
        return Launch(ScoresGradKernel<decltype(tt), decltype(nch)::value, decltype(tpu)::value>, Blocks(a.r, p), a,
                      stream, kThreads<decltype(tpu)::value>);
      });
    });
  });
}

size_t kd_distill_loss_workspace(const kd_frame_rows *rows, int32_t with_grad) {
  Rows r;
  Plan p;
  int64_t n;
  if (Guarded([&] { return CheckRows(rows, with_grad ? kFused : kValues, &r, &p, &n, 0, false); }) || p.nseg == 1)
    return 0;
  return Align(static_cast<size_t>(n) * p.nseg * sizeof(Partial)) + Align(static_cast<size_t>(n) * 8);
}

int kd_distill_loss(const kd_frame_rows *rows, const kd_teacher_rows *teacher, const float *weights, float temperature,
                    float *loss, float *stats, const float *upstream, void *grad, int64_t grad_batch_stride,
                    int64_t grad_row_stride, void *workspace, size_t workspace_bytes, void *stream) {
  return Guarded([&]() -> int {
    DistillArgs a{};
    Plan p;
    int64_t n;
    // stats given and no loss asked for: the statistics of an earlier call, the gradient alone
    const bool known = !loss && stats;
    if (int rc = CheckRows(rows, known ? kPieces : grad ? kFused : kValues, &a.r, &p, &n, 0, teacher && teacher->slots <= kShortSlots)) return rc;
    if (!teacher || teacher->slots < 1 || teacher->slots > kMaxSlots)
      return SetError(KD_E_INVALID, "bad argument: a teacher lists between 1 and 256 tokens a row");
    if (teacher->id_bytes != 4 && teacher->id_bytes != 8)
      return SetError(KD_E_INVALID, "bad argument: id_bytes must be 4 or 8");
    if (teacher->dtype != KD_DTYPE_F32 && teacher->dtype != KD_DTYPE_F16 && teacher->dtype != KD_DTYPE_BF16)
      return SetError(KD_E_INVALID, "bad argument: dtype of the teacher's logits");
    if (!(temperature >= 1e-6f && temperature <= 1e6f))
      return SetError(KD_E_INVALID, "bad argument: temperature must be between 1e-6 and 1e6");
    if (!n) return KD_OK;
    if (!teacher->ids || !teacher->logits) return SetError(KD_E_INVALID, "bad argument: the teacher's list is NULL");
    if (!loss && !grad) return SetError(KD_E_INVALID, "bad argument: neither loss nor gradient asked for");
    if (!loss && !stats) return SetError(KD_E_INVALID, "bad argument: a gradient alone needs the loss's stats");
    const size_t need = known ? 0 : kd_distill_loss_workspace(rows, grad != nullptr);
    if (grad)
      if (int rc = CheckGrad(rows, grad, grad_batch_stride, grad_row_stride,
                             {{rows->lengths, 4 * rows->batch, "lengths"},
                              {teacher->ids, n * teacher->slots * teacher->id_bytes, "the teacher's ids"},
                              {teacher->logits, n * teacher->slots * ElemBytes(teacher->dtype), "the teacher's logits"},
                              {weights, n * 4, "weights"},
                              {upstream, n * 4, "upstream"},
                              {loss, n * 4, "loss"},
                              {stats, n * 8, "stats"},
                              {workspace, static_cast<int64_t>(need), "the workspace"}},
                             &a.o))
        return rc;
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
      s.weights = weights;
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
        return ForPlan<kPieces, kByBoth, decltype(t)>(p, [&](auto tt, auto nch, auto tpu) {
          return ForSlots<decltype(tpu)::value>(a.slots, [&](auto sn) {
            return Launch(DistillGradKernel<decltype(tt), decltype(nch)::value, decltype(tpu)::value, decltype(sn)::value>,
                          Blocks(a.r, p), a, stream);
          });
        });
      });
    }
    auto whole = [&](auto what, auto with_grad) {
      return ForType(rows->dtype, [&](auto t) {
        return ForPlan<static_cast<Purpose>(decltype(what)::value), kByBoth, decltype(t)>(p, [&](auto tt, auto nch, auto tpu) {
          constexpr int TPU = decltype(tpu)::value;
          return ForSlots<TPU>(a.slots, [&](auto sn) {
            return Launch(DistillKernel<decltype(tt), decltype(nch)::value, TPU, decltype(sn)::value,
                                        decltype(with_grad)::value != 0>,
                          Blocks(a.r, p), a, stream, kThreads<TPU>);
          });
        });
      });
    };
    return grad ? whole(Int<kFused>{}, Int<1>{}) : whole(Int<kValues>{}, Int<0>{});
  });
}

}  // extern "C"
