// Sampling from next-token logits (gfx950): the truncated softmax of a row and the accept rule of a
// sampled speculative round, both from 16-bit logits x[0..V).
//
//   w_v = exp((x_v - max x) / T), 0 where x_v is -inf or NaN (max = +inf: 1 where x_v = +inf, else 0)
//   K   = the top_k largest logits (all without top_k), Z_K the sum of w over K
//   N   = the tokens of K, in falling order, before which less than top_p * Z_K lies
//   p_v = w_v / Z on N with Z the sum of w over N, else 0; equal logits are ordered by index
//   accept draft i:  u_i * q_i(x_i) < p_i(x_i)        (q = 1 at the drafted token without draft_probs)
//   n = the first draft refused (or the number of drafts); the token after them is drawn from
//   r_v = max(p_v - q_v, 0) of row n, from p of row n where there was no draft or r is zero throughout:
//   the first v whose running sum of r passes u_last times the whole sum.
//
// Every weight is formed and summed in 64 bits, in an order that depends on the sizes alone: which
// token a random number falls on is decided by differences that fp32 sums over 1e5 tokens do not hold
// (a token of probability 1e-5 is 1e2 units of an fp32 sum of 1 wide). An fp64 instruction takes 8 cycles a
// wave here; a weight takes 16 of them, of which 10 are its polynomial.
//
// A row is cut into segments of 512 logits, one wave load of 16 bytes a lane. The first pass leaves the
// maximum of each segment and its sum of weights against that maximum; whatever follows works on these
// few hundred values and re-reads single segments:
//   - the normaliser of a row is the join of its segments;
//   - a cut needs a threshold. 16-bit logits have at most 2^16 values, so the weight mass above a value is
//     a sum over distinct values of count * weight: integer counts in LDS, joined in falling order. Only
//     segments whose maximum can reach the threshold are read: for top_k the k-th largest segment
//     maximum bounds it from below, for top_p the weight (1 - top_p) S / V (what lies below all
//     together weighs less than (1 - top_p) S);
//   - the drawn token is found by a scan over segments, then inside one.
// Segments start at 16-byte addresses, not at the row's start: a row of odd length behind another one
// still loads 16 bytes a lane, and only its first and last 8 logits element by element.
#pragma once

#include "dspark_common.h"

namespace dspark {

constexpr int kSegVals = 512;          // logits of a segment
constexpr int kMaxSegs = 1024;         // segments of a row: one LDS slot each in the kernels of a row
constexpr int kMaxDraft = 255;         // drafts of a sequence
constexpr int kBins = 30720;           // distinct logit values counted at a time: most of the LDS
// Distinct values joined first, four times as many after them: the goal is mostly in the first (35 rows of 32003 in fp16: 29.1
// us at 4096, 32.0 at 8192, 43.1 at 2048, which it lies beyond; 5 rows of 151936 in bf16: 21.8 at 1024, 22.4 at 2048, 25 at 4096).
template <bool HALF>
constexpr int kChunk = HALF ? 4096 : 1024;     // 4 octaves of fp16, 8 of bf16
constexpr int kRowThreads = 1024;      // threads of the kernels that work on one row or sequence
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kListed = 256;           // candidates of a row that are sorted instead of counted

constexpr int kNoTies = -8;            // a cut below every index, those before a row's first logit too

struct SampleArgs {
  const u16* x;                        // logits
  long ldb, ldr;                       // strides of a sequence, of a row inside it
  int rows, per, V, nseg;              // rows in all, rows of a sequence
  double c;                            // log2(e) / T
  double top_p;
  int top_k;                           // 0: none
  int parts;                           // of a segment, whose maxima bound the top_k (0: whole segments)
  float* segm;                         // [rows][nseg] segment maxima
  double* segs;                        // [rows][nseg] segment sums
  int* arrived;                        // [sequences], [rows]: workgroups that are done, cleared by the first launch
};

struct RowInfo {                       // what is sampled from of a row
  double z;                            // sum of the kept weights (0: nothing to draw from)
  double px;                           // the drafted token's probability
  float m;                             // the row's maximum
  int thr, cut;                        // kept: key > thr, or key == thr and index <= cut
  int pad;
};

struct VerifyIn {
  const int32_t* draft;                // [sequences][per - 1]
  const float* q;                      // draft probabilities, or null
  long qb, qr;                         // strides of a sequence, of a draft
  const int32_t* lens;                 // drafts of each sequence, or null
  const void* u;                       // uniforms [sequences][per]
  int u64;                             // uniforms in 64 bits
  int32_t* n;                          // accepted
  int32_t* tokens;                     // [sequences][per]
  float* px;                           // [sequences][per - 1]
};

// ---------------------------------------------------------------- values and keys

template <bool HALF>
__device__ __forceinline__ float val(u32 bits) {
  if constexpr (HALF) return (float)__builtin_bit_cast(_Float16, (u16)bits);
  else return bf2f(bits);
}

template <bool HALF>
constexpr u32 kInfBits = HALF ? 0x7C00u : 0x7F80u;

// The order of the logits as integers: the magnitude's bits with their sign, so +0 and -0 are equal. A NaN lies
// outside [kLowKey, -kLowKey], the keys of the infinities.
template <bool HALF>
constexpr int kLowKey = -(int)kInfBits<HALF>;
template <bool HALF>
__device__ __forceinline__ float val_of_key(int k) {
  return val<HALF>(k < 0 ? 0x8000u | (u32)-k : (u32)k);
}
template <bool HALF>
__device__ __forceinline__ int key_of_float(float f) {
  int b;
  if constexpr (HALF) b = (int16_t)__builtin_bit_cast(u16, (_Float16)f);
  else b = (int16_t)f2bf(f);
  return b < 0 ? -(b & 0x7FFF) : b;
}

// The keys of a lane's 8 logits, two at a time.
typedef int16_t i16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void keys8(const u32x4_t& v, int (&k)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32 two = v[i];              // a value of its own: the cast of a vector's element takes the first one
    const i16x2_t b = __builtin_bit_cast(i16x2_t, two), s = b >> (int16_t)15;
    const i16x2_t r = ((b & (int16_t)0x7FFF) ^ s) - s;
    k[2 * i] = r[0];
    k[2 * i + 1] = r[1];
  }
}

// 2^d for d < 1024: the interpolation of 2^f on [-1/2, 1/2] in 11 Chebyshev nodes, its coefficients formed in 70 digits
// (within 3.2e-16 of itself and exact at 0; its steps' roundings another 1.5e-16), times a power of two; 0 below 2^-1075.
// A weight's argument, x c - m c, is off by 2^-53 of m c beside that.
__device__ __forceinline__ double exp2_neg(double d) {
  d = __builtin_fmax(d, -1080.0);
  const double n = __builtin_rint(d), f = d - n;
  double p = 7.0725859492692234e-09;
  p = __builtin_fma(p, f, 1.0208690299958306e-07);
  p = __builtin_fma(p, f, 1.3215442587921689e-06);
  p = __builtin_fma(p, f, 1.5252657260200837e-05);
  p = __builtin_fma(p, f, 0.0001540353044173605);
  p = __builtin_fma(p, f, 0.0013333558230164974);
  p = __builtin_fma(p, f, 0.0096181291076068882);
  p = __builtin_fma(p, f, 0.055504108664447722);
  p = __builtin_fma(p, f, 0.24022650695910097);
  p = __builtin_fma(p, f, 0.69314718055994995);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// The weight of a logit against a maximum m over -inf (1 where they are equal, infinities too; a NaN logit's
// NaN argument is taken for the smaller operand: 0); mc = -m c. Straight code: the weights of a lane's 8
// logits overlap.
__device__ __forceinline__ double weight(float x, float m, double c, double mc) {
  return exp2_neg(x == m ? 0.0 : __builtin_fma((double)x, c, mc));
}
__device__ __forceinline__ double weight(float x, float m, double c) { return weight(x, m, c, -(double)m * c); }

// ---------------------------------------------------------------- wave reductions (DPP)

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_d(double v) {
  const u32x2_t b = __builtin_bit_cast(u32x2_t, v);
  u32x2_t r;
  r[0] = (u32)__builtin_amdgcn_update_dpp(0, (int)b[0], CTRL, ROWS, 0xF, true);
  r[1] = (u32)__builtin_amdgcn_update_dpp(0, (int)b[1], CTRL, ROWS, 0xF, true);
  return __builtin_bit_cast(double, r);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_i(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_max(float v) {  // max with the shifted value, -inf where there is none
  const int lo = __builtin_bit_cast(int, -INFINITY);
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(lo, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false)));
}

// The value of the lane before (0 in lane 0): a shift of the whole wave by one.
__device__ __forceinline__ double lane_before(double v) { return dpp_d<0x138, 0xF>(v); }
__device__ __forceinline__ int lane_before(int v) { return dpp_i<0x138, 0xF>(v); }

// Running sums over the lanes of a wave: shifts inside rows of 16 lanes, then the last lane of row 0
// and 2 into the next row, then that of the lower half into the upper.
__device__ __forceinline__ double wave_scan(double v) {
  v += dpp_d<0x111, 0xF>(v);
  v += dpp_d<0x112, 0xF>(v);
  v += dpp_d<0x114, 0xF>(v);
  v += dpp_d<0x118, 0xF>(v);
  v += dpp_d<0x142, 0xA>(v);
  v += dpp_d<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_i<0x111, 0xF>(v);
  v += dpp_i<0x112, 0xF>(v);
  v += dpp_i<0x114, 0xF>(v);
  v += dpp_i<0x118, 0xF>(v);
  v += dpp_i<0x142, 0xA>(v);
  v += dpp_i<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ double lane_value(double v, int lane) {
  const u32x2_t b = __builtin_bit_cast(u32x2_t, v);
  u32x2_t r;
  r[0] = (u32)__builtin_amdgcn_readlane((int)b[0], lane);
  r[1] = (u32)__builtin_amdgcn_readlane((int)b[1], lane);
  return __builtin_bit_cast(double, r);
}
__device__ __forceinline__ double wave_total(double v) { return lane_value(wave_scan(v), 63); }
__device__ __forceinline__ float wave_max(float v) {
  v = dpp_max<0x111, 0xF>(v);
  v = dpp_max<0x112, 0xF>(v);
  v = dpp_max<0x114, 0xF>(v);
  v = dpp_max<0x118, 0xF>(v);
  v = dpp_max<0x142, 0xA>(v);
  v = dpp_max<0x143, 0xC>(v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Running sums over the threads of a workgroup, in thread order: what lies before a thread (returned) and up
// to it (`upto`), the whole in `total`. `waves`: a slot a wave, free again after the next barrier.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* waves, V& upto, V& total) {
  const int w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const V in = wave_scan(v);
  if ((threadIdx.x & 63) == 63) waves[w] = in;
  __syncthreads();
  V before = 0, all = 0;
  for (int i = 0; i < nw; ++i) {
    if (i == w) before = all;
    all += waves[i];
  }
  __syncthreads();
  total = all;
  upto = before + in;
  return before + lane_before(in);
}

// ---------------------------------------------------------------- between workgroups of a launch

// Written through to, and read from, where every XCD sees it.
template <typename V>
__device__ __forceinline__ void put_far(V* p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename V>
__device__ __forceinline__ V get_far(const V* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// True in every thread of the workgroup that arrives last of `n`; what the others put before it is there to get.
__device__ __forceinline__ bool arrives_last(int* counter, int n, int* slot) {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");     // this thread's stores are complete
  __syncthreads();
  if (threadIdx.x == 0) *slot = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
  __syncthreads();
  return *slot;
}

// ---------------------------------------------------------------- segments

// Where a row's first logit lies inside its first 16 bytes: logit v is value v + off of the segments.
__device__ __forceinline__ int row_off(const u16* row) { return (int)((reinterpret_cast<uintptr_t>(row) >> 1) & 7); }

// The 8 logits of a lane of segment `seg` (first index v0 = 512 seg + 8 lane - off), -inf outside the row.
template <bool HALF>
__device__ __forceinline__ u32x4_t load8(const u16* row, int v0, int V) {
  if (v0 >= 0 && v0 + 8 <= V) return ldg128(row + v0);
  u32 b[8];                            // a row's ends: each on its own, from inside the row
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = row[min(max(v0 + i, 0), V - 1)];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = v0 + i >= 0 && v0 + i < V ? b[i] : 0x8000u | kInfBits<HALF>;
  return u32x4_t{b[0] | b[1] << 16, b[2] | b[3] << 16, b[4] | b[5] << 16, b[6] | b[7] << 16};
}
__device__ __forceinline__ u32 bits_of(const u32x4_t& v, int j) { return (v[j >> 1] >> (16 * (j & 1))) & 0xFFFFu; }

// The largest of a segment's logits (NaN: none), in every lane.
template <bool HALF>
__device__ __forceinline__ float max8_wave(const u32x4_t& v) {
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, val<HALF>(bits_of(v, j)));
  return wave_max(m);
}

__device__ __forceinline__ const u16* row_ptr(const SampleArgs& a, int seq, int i) { return a.x + seq * a.ldb + i * a.ldr; }

// Maximum and normaliser of a row without a cut, the join of its segments, by one wave: eight values a lane at once.
__device__ __forceinline__ double join_wave(const float* segm, const double* segs, int nseg, double c, float& m) {
  constexpr int kAtOnce = 8;
  const int lane = threadIdx.x & 63;
  float mx = -INFINITY;                // of this lane so far; z against it
  double z = 0;
  for (int s0 = lane; s0 < nseg; s0 += 64 * kAtOnce) {
    float sm[kAtOnce], to = mx;
    double ss[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int s = s0 + 64 * i;
      sm[i] = s < nseg ? segm[s] : -INFINITY;
      ss[i] = s < nseg ? segs[s] : 0.0;
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) to = fmaxf(to, sm[i]);
    z *= weight(mx, to, c);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (s0 - lane + 64 * i < nseg) z += ss[i] * weight(sm[i], to, c);
    mx = to;
  }
  m = wave_max(mx);
  const double all = wave_total(m > -INFINITY ? z * weight(mx, m, c) : 0.0);
  return all;
}

}  // namespace dspark
