// Log probabilities of given tokens, the entropy of their distributions and the best alternatives (gfx950).
//
// With z = (x - max x) / temperature over a row's logits, S = sum e^z and U = sum z e^z:
//   log p(token) = z_token - ln S,   entropy = ln S - U / S,   alternatives: the largest x, equal ones by index.
// One pass: every lane keeps its running maximum with S and U relative to it (U' = f (U + delta S) where the maximum
// rises by -delta in the exponent), in fp32 and units of log 2; ln S and the differences that leave the call are fp64. NaN
// counts as -inf; with infinite logits those share all of it; a row of nothing has -inf everywhere and no entropy.
//
// The alternatives come out of the same pass. A candidate is a 64-bit key, value before inverted index, so that no two are
// equal and the order is total. A wave keeps a list of candidates in LDS and a least key, under which k better ones are
// known; a lane's values of a step are compared by their maximum, which the sums need anyway, and looked at only where it
// reaches the least key (passes it, once the wave is behind the least key's index: rows of equal values, as of forbidden
// tokens, cost no more). The least key starts as the k-th of the 64 lanes' maxima, rises when a full list is cut to its k best,
// and is shared by the workgroup's waves.
//
// Bound by the bytes of the logits, with the exponential (a quarter of the rate) and about 6 more instructions a value
// close behind. Many rows: a workgroup of four waves a row; few: up to 64 waves a row, a workgroup each, joined by a second
// launch. bf16, 900 rows of 128255 with the best 5: 59 us (3.9 TB/s; 66 with loads that fill the caches, 61 and 72 with 16
// and 48 values a lane's step instead of 32); one row of 151936: 6 us, 13 with the best 20, of which the list takes its time
// from a wave that has nothing beside it on its SIMD.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dspark_common.h"

namespace dspark {
namespace {

using u64 = unsigned long long;

constexpr int kScoreWaves = 4;                 // of a workgroup that takes a whole row
constexpr int kMostTop = 64;
constexpr int kList = 192;                     // candidates of a wave: 1.5 times the most, 16, and a key of every lane
constexpr int kMostSegments = 64;              // of a row: a lane each where they are joined
constexpr float kScoreLowest = -3.402823466e38f;
constexpr float kNothing = -1e4f;              // an exponent whose power of two is 0, times which 0 is 0

struct ScoreArgs {
  const char* x;
  long ld;                                     // row stride in elements
  int rows, V, top, segments;
  float c;                                     // log2(e) / temperature
  double temperature;
  const void* tokens;
  int tokens64;
  float* given;
  float* entropy;
  int* ids;                                    // [rows][top]
  float* best;
  float* stats;                                // [rows][segments][3]
  u64* keys;                                   // [rows][segments][top], falling; 0: none
};

template <int DT> struct Logit;
template <> struct Logit<DSPARK_DTYPE_BF16> {
  using t = u16;
  static __device__ __forceinline__ float get(u16 v) { return bf2f(v); }
};
template <> struct Logit<DSPARK_DTYPE_F16> {
  using t = u16;
  static __device__ __forceinline__ float get(u16 v) { return (float)__builtin_bit_cast(_Float16, v); }
};
template <> struct Logit<DSPARK_DTYPE_F32> {
  using t = float;
  static __device__ __forceinline__ float get(float v) { return v; }
};

// A key falls with the value, then with the index; NaN as -inf, -0 as 0. Never 0.
__device__ __forceinline__ u64 key_of(float x, int i) {
  x = x == x ? x + 0.f : -__builtin_inff();
  const u32 b = __builtin_bit_cast(u32, x);
  return (u64)(b ^ ((int)b < 0 ? 0xFFFFFFFFu : 0x80000000u)) << 32 | (u32)~i;
}
__device__ __forceinline__ float value_of(u64 k) {
  const u32 b = (u32)(k >> 32);
  return __builtin_bit_cast(float, b ^ ((int)b < 0 ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ int index_of(u64 k) { return (int)~(u32)k; }

__device__ __forceinline__ u64 lane_key(u64 k, int l) {
  return (u64)(u32)__builtin_amdgcn_readlane((int)(k >> 32), l) << 32 | (u32)__builtin_amdgcn_readlane((int)(u32)k, l);
}
struct Stats {
  float m, s, u;                               // maximum, sum of 2^d, sum of d 2^d, d = (x - m) c
};

__device__ __forceinline__ Stats join(Stats a, Stats b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float da = fmaxf((a.m - m) * c, kNothing), db = fmaxf((b.m - m) * c, kNothing);
  const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  return Stats{m, fa * a.s + fb * b.s, fa * (a.u + da * a.s) + fb * (b.u + db * b.s)};
}
__device__ __forceinline__ Stats join_wave(Stats s, float c) {
#pragma unroll
  for (int x = 1; x < 64; x *= 2) s = join(s, Stats{shfl_xor(s.m, x), shfl_xor(s.s, x), shfl_xor(s.u, x)}, c);
  return s;
}

// The k best of a wave's list of n (up to 64 N), in order at its start; how many there are
template <int N>
__device__ __forceinline__ int cut_list(u64* list, int n, int k) {
  const int lane = __lane_id();
  u64 mine[N];
  int rank[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    mine[i] = 64 * i + lane < n ? list[64 * i + lane] : 0;
    rank[i] = 0;
  }
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const u64 o = list[j];
#pragma unroll
    for (int i = 0; i < N; ++i) rank[i] += o > mine[i] ? 1 : 0;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (mine[i] && rank[i] < k) list[rank[i]] = mine[i];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return min(n, k);
}

// Infinite logits of a row, counted by one wave
template <int DT>
__device__ __forceinline__ int infinite_logits(const ScoreArgs& a, long row) {
  using T = typename Logit<DT>::t;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld;
  int n = 0;
#pragma unroll 1
  for (int i = __lane_id(); i < a.V; i += 64) n += Logit<DT>::get(x[i]) == __builtin_inff() ? 1 : 0;
#pragma unroll 1
  for (int d = 1; d < 64; d *= 2) n += __builtin_amdgcn_ds_bpermute((__lane_id() ^ d) << 2, n);
  return n;
}

// What a row's sums and keys (falling, in LDS or memory) come to; by one wave
template <int DT>
__device__ __forceinline__ void finish_row(const ScoreArgs& a, long row, Stats s, u64 mine) {
  using T = typename Logit<DT>::t;
  const int lane = __lane_id();
  double log_sum = log((double)s.s), entropy = log_sum - 0.69314718055994531 * ((double)s.u / (double)s.s);
  const bool infinite = s.m == __builtin_inff();
  if (infinite) entropy = log_sum = log((double)infinite_logits<DT>(a, row));
  const bool none = !infinite && !(s.s > 0.f);
  auto log_p = [&](float x) {
    if (infinite) return x == s.m ? (float)-log_sum : -__builtin_inff();
    if (none || x != x) return -__builtin_inff();
    return (float)(((double)x - (double)s.m) / a.temperature - log_sum);
  };
  if (lane == 0) {
    const int64_t t = a.tokens64 ? static_cast<const int64_t*>(a.tokens)[row] : (int64_t)static_cast<const int32_t*>(a.tokens)[row];
    a.given[row] = t >= 0 && t < a.V ? log_p(Logit<DT>::get((reinterpret_cast<const T*>(a.x) + row * a.ld)[t])) : -__builtin_inff();
    a.entropy[row] = none ? 0.f : (float)(entropy > 0. ? entropy : 0.);
  }
  if (lane < a.top) {
    a.ids[row * a.top + lane] = index_of(mine);
    a.best[row * a.top + lane] = log_p(value_of(mine));
  }
}

// Keys of a wave's list, and the least one under which k better ones are known
struct List {
  u64* keys;
  int n, top, full;
  u64 least;
  u64* shared;                                 // the workgroup's least key (null: one wave)

  __device__ __forceinline__ void raise(u64 k) {
    if (k <= least) return;
    least = k;
    if (shared && __lane_id() == 0) atomicMax(shared, k);
  }
  // Where 64 lanes' best keys come to k of at least some key, that is a least key
  __device__ __forceinline__ void raise_by(u64 best) {
    keys[n + __lane_id()] = best;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < 64; ++j) rank += keys[n + j] > best ? 1 : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const u64 kth = __builtin_amdgcn_ballot_w64(rank == top - 1 && best != 0);
    if (kth) raise(lane_key(best, __builtin_ctzll(kth)));
  }
  // A key of every lane (0: none)
  __device__ __forceinline__ void push(u64 k) {
    const u64 in = __builtin_amdgcn_ballot_w64(k != 0 && k >= least);
    if (!in) return;
    if (k != 0 && k >= least) keys[n + __builtin_popcountll(in & ((1ull << __lane_id()) - 1))] = k;
    n = uniform(n + __builtin_popcountll(in));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (n > full) cut();
  }
  __device__ __forceinline__ void cut() {
    n = uniform(n <= 64 ? cut_list<1>(keys, n, top) : cut_list<kList / 64>(keys, n, top));
    if (n == top) raise(keys[top - 1]);
  }
};
__device__ __forceinline__ List new_list(u64* keys, int top, u64* shared) {
  return List{keys, 0, top, top + top / 2 + 16, 0, shared};
}

// Values of a lane's step. A wave that has a row's part for itself is alone on its SIMD, and what counts is how many
// instructions it issues until it is done: one step for most vocabularies.
template <int WAVES> constexpr int kPerLane = WAVES == 1 ? 40 : 32;

template <int DT, bool TOP, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void score_kernel(const ScoreArgs a) {
  using T = typename Logit<DT>::t;
  constexpr int kPer = kPerLane<WAVES>;
  constexpr int E = 16 / sizeof(T), NL = kPer / E;           // values of a 16-byte load, loads of a step
  constexpr int STEP = 64 * NL;                              // 16-byte chunks of a wave's step
  struct alignas(16) Vec { T v[E]; };
  __shared__ u64 lists[WAVES][TOP ? kList : 1];
  __shared__ float staged[WAVES][TOP ? kPer * 64 : 1];
  __shared__ u64 least_of_all;
  __shared__ Stats parts[WAVES];
  __shared__ int counts[WAVES];
  const int lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : uniform((int)(threadIdx.x >> 6));
  const long row = blockIdx.x / a.segments;
  const int seg = blockIdx.x - (int)row * a.segments;
  const T* const x0 = reinterpret_cast<const T*>(a.x) + row * a.ld;
  // 16-byte chunks from the one that the row starts in: value i is number i + off of them
  const int off = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
  const Vec* const chunks = reinterpret_cast<const Vec*>(x0 - off);
  const int nc = (int)(((long)a.V + off + E - 1) / E), per = (nc + a.segments - 1) / a.segments;
  const int c0 = (int)min((long)seg * per, (long)nc), c1 = min(c0 + per, nc);
  const int w0 = off ? 1 : 0, w1 = min(c1, (int)(((long)a.V + off) / E));      // chunks that are all the row's
  List list = new_list(lists[wave], a.top, WAVES > 1 ? &least_of_all : nullptr);
  if (TOP && WAVES > 1) {
    if (threadIdx.x == 0) least_of_all = 0;
    __syncthreads();
  }

  auto whole = [&](int c) { return c >= w0 && c + STEP <= w1; };
  auto load = [&](Vec (&v)[NL], int c) {
    if (whole(c)) {
      const Vec* p = chunks + c + lane;
#pragma unroll
      for (int j = 0; j < NL; ++j) v[j] = __builtin_bit_cast(Vec, ldg128_nt(p + 64 * j));
      return;
    }
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int k = c + 64 * j + lane;
      if (k >= w0 && k < w1) {
        v[j] = chunks[k];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const long i = (long)k * E + e - off;
          T t;
          if constexpr (sizeof(T) == 4) t = __builtin_nanf("");
          else t = 0x7FFF;                                   // NaN: nothing
          if (k < c1 && i >= 0 && i < a.V) t = x0[i];
          v[j].v[e] = t;
        }
      }
    }
  };

  Stats st{kScoreLowest, 0.f, 0.f};
  int c = c0 + wave * STEP;
  Vec next[NL];
  if (c < c1) load(next, c);
  while (c < c1) {
    u64 shared = 0;
    if (TOP && WAVES > 1) shared = *(volatile u64*)&least_of_all;
    float x[kPer];
#pragma unroll
    for (int j = 0; j < NL; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) x[j * E + e] = Logit<DT>::get(next[j].v[e]);
    const int cur = c;
    c += WAVES * STEP;
    if (c < c1) load(next, c);
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kPer; ++i) top = fmaxf(top, x[i]);
    const float m = fmaxf(st.m, top);
    const float d0 = fmaxf((st.m - m) * a.c, kNothing), f = __builtin_amdgcn_exp2f(d0);
    st.u = f * (st.u + d0 * st.s);
    st.s *= f;
    st.m = m;
    float s1 = 0.f, u1 = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float d = fmaxf((x[i] - m) * a.c, kNothing), e = __builtin_amdgcn_exp2f(d);
      (i & 1 ? s1 : st.s) += e;
      if (i & 1) u1 = __builtin_fmaf(e, d, u1);
      else st.u = __builtin_fmaf(e, d, st.u);
    }
    st.s += s1;
    st.u += u1;
    if constexpr (TOP) {
      list.least = shared > list.least ? shared : list.least;
      // what a value has to reach: the least key's, or the next one up where all of the step's indices lie behind its
      auto needed = [&] {
        if (!list.least) return -__builtin_inff();
        const bool behind = (long)cur * E - off > (long)index_of(list.least);
        return value_of(behind ? list.least + (1ull << 32) : list.least);
      };
      const u64 some = __builtin_amdgcn_ballot_w64(top >= needed());
      if (!some) continue;
      const bool all = whole(cur);
      auto index = [&](int i) { return (int)((long)(cur + 64 * (i / E) + lane) * E + i % E - off); };
      auto there = [&](int i) {
        const int at = index(i);
        return all || (at >= 0 && at < a.V && cur + 64 * (i / E) + lane < c1);
      };
      if (__builtin_popcountll(some) >= max(a.top, 16)) {
        u64 best = 0;                                        // the lane's: the first of its largest
#pragma unroll
        for (int i = kPer - 1; i >= 0; --i)
          if ((x[i] == top || top == -__builtin_inff()) && there(i)) best = (u32)~index(i);
        if (best) best |= key_of(top, 0) & 0xFFFFFFFF00000000ull;
        list.raise_by(best);
      }
      // Bit i: value i reaches the least key's (NaN counts as -inf). They are listed out of LDS, where a lane finds value i:
      // one copy of the code, where one for every value would not fit the instruction cache
      using Mask = std::conditional_t<(kPer > 32), u64, u32>;
      const float least_value = needed();
      Mask mask = 0;
#pragma unroll
      for (int i = kPer - 1; i >= 0; --i) mask = mask + mask + (x[i] >= least_value ? 1u : 0u);
      if (least_value == -__builtin_inff()) mask = ~Mask(0) >> (8 * sizeof(Mask) - kPer);
      float* const mine = &staged[wave][lane];
      if (mask) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) mine[64 * i] = x[i];
      }
      while (__builtin_amdgcn_ballot_w64(mask != 0)) {
        const int i = mask ? __builtin_ctzll(mask) : 0, at = index(i);
        u64 k = 0;
        if (mask && at >= 0 && at < a.V && cur + 64 * (i / E) + lane < c1) k = key_of(mine[64 * i], at);
        mask &= mask - 1;
        list.push(k);
      }
    }
  }

  st = join_wave(st, a.c);
  if (TOP) list.cut();
  if constexpr (WAVES > 1) {
    if (lane == 0) {
      parts[wave] = st;
      counts[wave] = list.n;
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll 1
    for (int w = 1; w < WAVES; ++w) {
      st = join(st, parts[w], a.c);
      if (TOP) list.push(lane < counts[w] ? lists[w][lane] : 0);
    }
    if (TOP) list.cut();
  }
  const u64 mine = TOP && lane < list.n ? list.keys[lane] : 0;
  if (a.segments == 1) {
    finish_row<DT>(a, row, st, mine);
    return;
  }
  if (lane == 0) {
    float* to = a.stats + 3 * (row * a.segments + seg);
    to[0] = st.m, to[1] = st.s, to[2] = st.u;
  }
  if (TOP && lane < a.top) a.keys[(row * a.segments + seg) * a.top + lane] = mine;
}

// A row's segments together, by one wave: a lane has a segment's sums, and its keys, which fall
template <int DT>
__global__ __launch_bounds__(64) void join_scores_kernel(const ScoreArgs a) {
  __shared__ u64 keys[kList];
  const long row = blockIdx.x;
  const int lane = __lane_id();
  Stats s{kScoreLowest, 0.f, 0.f};
  if (lane < a.segments) {
    const float* from = a.stats + 3 * (row * a.segments + lane);
    s = Stats{from[0], from[1], from[2]};
  }
  u64 mine = 0;
  if (a.top) {
    List list = new_list(keys, a.top, nullptr);
    const u64* from = a.keys + (row * a.segments + min(lane, a.segments - 1)) * a.top;
    u64 k = lane < a.segments ? from[0] : 0;
    if (a.segments >= a.top) list.raise_by(k);
#pragma unroll 1
    for (int i = 1; __builtin_amdgcn_ballot_w64(k != 0 && k >= list.least); ++i) {
      const u64 next = lane < a.segments && i < a.top ? from[i] : 0;
      list.push(k);
      k = next;
    }
    list.cut();
    if (lane < list.n) mine = keys[lane];
  }
  finish_row<DT>(a, row, join_wave(s, a.c), mine);
}

// Segments of a row: 1 from 512 rows on, a workgroup each; fewer rows are dealt to 2048 waves, of whole steps
int score_segments(int64_t rows, int64_t V) {
  if (rows >= 512) return 1;
  constexpr int64_t step = 64 * kPerLane<1>;
  const int64_t n = std::min<int64_t>((2048 + rows - 1) / rows, kMostSegments), steps = (V + n * step - 1) / (n * step);
  return (int)((V + steps * step - 1) / (steps * step));
}

template <int DT, bool TOP>
int launch_score(const ScoreArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows * (long)a.segments));
  if (a.segments == 1) hipLaunchKernelGGL((score_kernel<DT, TOP, kScoreWaves>), grid, dim3(64 * kScoreWaves), 0, s, a);
  else hipLaunchKernelGGL((score_kernel<DT, TOP, 1>), grid, dim3(64), 0, s, a);
  const int st = check_launch("token_logprobs");
  if (st || a.segments == 1) return st;
  hipLaunchKernelGGL((join_scores_kernel<DT>), dim3((unsigned)a.rows), dim3(64), 0, s, a);
  return check_launch("token_logprobs(join)");
}
template <int DT>
int launch_score(const ScoreArgs& a, hipStream_t s) {
  return a.top ? launch_score<DT, true>(a, s) : launch_score<DT, false>(a, s);
}

}  // namespace
}  // namespace dspark

using namespace dspark;

extern "C" size_t dspark_token_logprobs_workspace(int64_t rows, int64_t V, int64_t top) {
  if (rows < 1 || rows > (1 << 20) || V < 1 || V > (1 << 28) || top < 0 || top > kMostTop || top > V) return 0;
  const int64_t n = score_segments(rows, V);
  return n == 1 ? 256 : (size_t)(rows * n * (8 * top + 12) + 256);
}

extern "C" int dspark_token_logprobs(const dspark_token_logprobs_args* p, dspark_stream stream) {
  const char* what = "token_logprobs";
  if (!p || !p->logits || !p->tokens || !p->logprobs || !p->entropy || !p->workspace || (p->top && (!p->top_tokens || !p->top_logprobs)))
    return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  const size_t need = dspark_token_logprobs_workspace(p->rows, p->V, p->top);
  if (!need)
    return fail(DSPARK_ERR_SHAPE, "%s: %ld rows (up to 2^20) of %ld logits (up to 2^28), the best %ld (up to %d and all)", what,
                (long)p->rows, (long)p->V, (long)p->top, kMostTop);
  if (!aligned(p->tokens, p->tokens_i64 ? 8 : 4)) return fail(DSPARK_ERR_ALIGN, "%s: tokens need the alignment of their type", what);
  if (!(p->temperature >= 1e-30 && p->temperature <= 1e30)) return fail(DSPARK_ERR_ARG, "%s: temperature %g", what, p->temperature);
  const int es = p->dtype == DSPARK_DTYPE_F32 ? 4 : 2;
  if (!aligned(p->logits, es)) return fail(DSPARK_ERR_ALIGN, "%s: logits need the alignment of their type", what);
  if (!aligned(p->workspace, 16) || (size_t)p->workspace_bytes < need)
    return fail(DSPARK_ERR_WORKSPACE, "%s: workspace %ld < %zu bytes, or not 16-byte aligned", what, (long)p->workspace_bytes, need);
  ScoreArgs a = {};
  a.x = static_cast<const char*>(p->logits);
  a.ld = p->ld;
  a.rows = (int)p->rows;
  a.V = (int)p->V;
  a.top = (int)p->top;
  a.segments = score_segments(p->rows, p->V);
  a.c = (float)(1.44269504088896340736 / p->temperature);
  a.temperature = p->temperature;
  a.tokens = p->tokens;
  a.tokens64 = p->tokens_i64 != 0;
  a.given = p->logprobs;
  a.entropy = p->entropy;
  a.ids = p->top_tokens;
  a.best = p->top_logprobs;
  a.keys = static_cast<u64*>(p->workspace);
  a.stats = reinterpret_cast<float*>(a.keys + p->rows * a.segments * p->top);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (p->dtype) {
    case DSPARK_DTYPE_BF16: return launch_score<DSPARK_DTYPE_BF16>(a, s);
    case DSPARK_DTYPE_F16: return launch_score<DSPARK_DTYPE_F16>(a, s);
    case DSPARK_DTYPE_F32: return launch_score<DSPARK_DTYPE_F32>(a, s);
    default: return fail(DSPARK_ERR_UNSUPPORTED, "%s: dtype %ld", what, (long)p->dtype);
  }
}
