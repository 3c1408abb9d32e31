// The kernels and entry points of dspark_sampling.h: the truncated softmax of a row
// (dspark_sampling_probs) and the accept rule of a sampled round (dspark_speculative_verify).
//
// The first launch leaves every segment's maximum and sum. Then
//   verify, a small top_k: a workgroup a row selects and draws, the last of a sequence accepts;
//   verify, else: one launch selects where something is cut, one of workgroups over a sequence's segments joins its
//   rows where nothing is, accepts, sums r over the row drawn from, and its last workgroup draws;
//   probabilities: a launch selects where something is cut, one writes.
// A small top_k of rows that are not long, without drafts, is one launch: a workgroup takes its row whole.
#include <cmath>

#include "dspark_sampling.h"

namespace dspark {
namespace {

// ---------------------------------------------------------------- segments of every row

constexpr int kStatThreads = 256;
// Segments of a wave in the first pass: its sums are fp64 work that many waves share better (15 rows of 151936 cut by a
// mass: 24.7 us at 2, 26.3 at 4, 24.9 at 1; 128 rows uncut in fp16: 47.2, 47.7, 48.3). Writing probabilities: 4 where a
// wave joins its row first (128 rows: 49.7 us at 2), 2 behind a cut, which has joined it (15 rows: 26.6 us at 4).
constexpr int kSegWave = 2, kProbWave = 4, kProbCutWave = 2;

// Maximum and sum of weights of every segment: a wave takes SPW segments, their loads first.
template <bool HALF, int SPW, bool SUM>
__global__ __launch_bounds__(kStatThreads) void sample_segments_kernel(const SampleArgs a) {
  const int lane = threadIdx.x & 63, seq = blockIdx.z;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (blockIdx.y == 0) a.arrived[seq] = 0;
    a.arrived[gridDim.z + (long)seq * a.per + blockIdx.y] = 0;
  }
  const int s0 = (blockIdx.x * (kStatThreads / 64) + uniform(threadIdx.x >> 6)) * SPW;
  const u16* x = row_ptr(a, seq, blockIdx.y);
  const int off = row_off(x);
  u32x4_t v[SPW];
#pragma unroll
  for (int i = 0; i < SPW; ++i) v[i] = load8<HALF>(x, (s0 + i) * kSegVals + 8 * lane - off, a.V);
#pragma unroll
  for (int i = 0; i < SPW; ++i) {
    if (s0 + i >= a.nseg) return;
    const float m = max8_wave<HALF>(v[i]);
    const long at = ((long)seq * a.per + blockIdx.y) * a.nseg + s0 + i;
    if constexpr (SUM) {
      const double mc = -(double)m * a.c;
      double s = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += weight(val<HALF>(bits_of(v[i], j)), m, a.c, mc);
      s = wave_total(s);
      if (lane == 0) a.segs[at] = m > -INFINITY ? s : 0.0;
    }
    if (lane == 0) a.segm[at] = m;
  }
}

// The same over many segments of bf16 logits, uncut: a value's weight against 0, 2^(c x), from a table in LDS.
// bf16 has 128 values an octave; 22 octaves, 2^-14 to 2^8, and both signs are 45 KB, formed once by each workgroup
// (one a CU, its waves then walk through the segments). A look-up and its sum are 6 instructions, one of them fp64;
// the weight itself is 16, nearly all fp64, and bounds the pass above (76032 segments: 37 us; the table's: 21).
// The sums stand against 0, so no maximum is looked for. A value the table does not have turns the sum into NaN, one
// below -256 counts as none; a segment of either kind, or too light for what was left out, is summed plainly.
constexpr int kTabLow = (127 - 14) << 7, kTabHalf = 22 << 7;
constexpr int kTabSlots = kTabHalf + 2;               // of one sign: below, the values, above
constexpr int kTabThreads = 1024, kTabAhead = 3;
constexpr double kTabMaxC = 3.5;       // 2^(c 256) stays far below the largest double

typedef u16 u16x2_t __attribute__((ext_vector_type(2)));

__global__ __launch_bounds__(kTabThreads) void sample_table_kernel(const SampleArgs a, const int total, const int steps) {
  __shared__ double tab[2 * kTabSlots];
  const int t = threadIdx.x, lane = t & 63;
  if (blockIdx.x == 0)
    for (int i = t; i < a.rows / a.per; i += kTabThreads) a.arrived[i] = 0;
  // a run of segments a wave, one row after another; the first loads before the table
  const int g0 = (blockIdx.x * (kTabThreads / 64) + uniform(t >> 6)) * steps, g1 = min(g0 + steps, total);
  int row = g0 / a.nseg, s = g0 - row * a.nseg, ahead = g0;            // of the next load
  const u16* x = row_ptr(a, row / a.per, row % a.per);
  const auto load = [&]() {
    const u32x4_t v = ahead < g1 ? load8<false>(x, s * kSegVals + 8 * lane - row_off(x), a.V) : u32x4_t{};
    ++ahead;
    if (++s == a.nseg) {
      s = 0;
      ++row;
      if (ahead < g1) x = row_ptr(a, row / a.per, row % a.per);
    }
    return v;
  };
  u32x4_t v[kTabAhead];
#pragma unroll
  for (int i = 0; i < kTabAhead; ++i) v[i] = load();
  if (t < 2 * kTabHalf / 8) {           // 8 values a thread, inside an octave: one after another by a ratio
    const int sign = t >= kTabHalf / 8, i0 = 8 * t - (sign ? kTabHalf : 0);
    const u32 b = (u32)(kTabLow + i0) | (sign ? 0x8000u : 0u);
    double w = exp2_neg((double)bf2f(b) * a.c);
    const double ratio = exp2_neg(((double)bf2f(b + 1) - (double)bf2f(b)) * a.c);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      tab[sign * kTabSlots + 1 + i0 + i] = w;
      w *= ratio;
    }
  }
  if (t < 4) tab[(t >> 1) * kTabSlots + (t & 1) * (kTabHalf + 1)] = t == 3 ? 0.0 : __builtin_nan("");
  __syncthreads();
  const double light = __builtin_ldexp(1.0, (int)(80.0 - 256.0 * a.c));      // V values below -256 weigh nothing beside it
  for (int g = g0; g < g1; g += kTabAhead) {
#pragma unroll
    for (int i = 0; i < kTabAhead; ++i) {
      if (g + i >= g1) break;
      const u32x4_t now = v[i];
      double sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32 two = now[j];
        const u16x2_t b = __builtin_bit_cast(u16x2_t, two);
        const u16x2_t sign = (b >> (u16)15) * (u16)kTabSlots;
        const u16x2_t slot = __builtin_elementwise_min(__builtin_elementwise_sub_sat((u16x2_t)(b & (u16)0x7FFF), (u16x2_t)(u16)(kTabLow - 1)),
                                                       (u16x2_t)(u16)(kTabHalf + 1)) + sign;
        sum += tab[slot[0]];
        sum += tab[slot[1]];
      }
      v[i] = load();
      sum = wave_total(sum);
      float m = 0;
      if (!(sum >= light)) {            // also NaN
        m = max8_wave<false>(now);
        sum = 0;
        if (m > -INFINITY) {
          const double mc = -(double)m * a.c;
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            const u32 two = j == 0 ? now[0] : j == 1 ? now[1] : j == 2 ? now[2] : now[3];
            sum += weight(bf2f(two & 0xFFFFu), m, a.c, mc);
            sum += weight(bf2f(two >> 16), m, a.c, mc);
          }
          sum = wave_total(sum);
        }
      }
      if (lane == 0) {
        a.segs[g + i] = sum;            // [rows][nseg], the order of the walk
        a.segm[g + i] = m;
      }
    }
  }
}

// ---------------------------------------------------------------- what is kept of a row

constexpr int kAhead = 4;              // segments of a wave whose loads are out together

struct RowState {
  int skey[kMaxSegs];                  // key of each segment's maximum
  int list[kMaxSegs];                  // the segments that may hold a kept token, in no order
  int cnt[kMaxSegs];
  double red_d[kRowWaves];
  float red_f[kRowWaves];
  int red_i[kRowWaves];
  int owner, key, keep, ties, cut, nlist, ncand, last, token;
  double z;
};

// Most segments of a row that a workgroup takes whole, without a launch before it (a token drawn from one row of 70000: 9.9
// us, 10.6 in two launches; of 100000: 11.1, 10.6; from each of 600 rows of 50257: 29.6, 35.9).
constexpr int kWholeSegs = 160;
static_assert(kWholeSegs <= kListed, "one room");

struct Few {                           // a few candidates, one by one
  uint64_t cand[kListed];              // (key + 2^15) << 32 | ~index: the larger the earlier in falling order
  uint64_t sorted[kListed];
  double w[kListed], r[kListed];       // weights in falling order; what is drawn from, by index
  union {
    int order[kListed];                // the kept tokens by index
    float segm[kWholeSegs];            // before that: the segments' maxima
  };
};

struct RowShared : RowState {
  union {
    int bins[kBins];
    Few few;
  };
};

// The bin, of 256 in falling order, that the k-th of what they count lies in; k: which of that bin's it is. Every
// wave for itself, four bins a lane.
__device__ __forceinline__ int nth_bin(const int* hist, int& k) {
  const int lane = threadIdx.x & 63;
  int c[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum += c[i] = hist[4 * lane + i];
  const int upto = wave_scan(sum);
  int before = upto - sum, at = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (at == i && before + c[i] < k) {
      before += c[i];
      at = i + 1;
    }
  const int owner = __ffsll(__ballot(upto >= k)) - 1;
  k -= __builtin_amdgcn_readlane(before, owner);
  return 4 * owner + __builtin_amdgcn_readlane(at, owner);
}

// The largest key that at least k of the threads' keys reach (`in`: a thread that has one; there are at least k):
// counts of the high bytes in falling order, then of the low bytes of the one the k-th lies in. `hist`: 512 zeros.
__device__ __forceinline__ int kth_key(bool in, int key, int k, int* hist) {
  const u32 u = (u32)(key + (1 << 15));
  int high = 0, low = 0;
  for (int round = 0; round < 2; ++round) {
    const int bin = 255 - (round ? (int)(u & 255) : (int)(u >> 8));
    if (in && (!round || (int)(u >> 8) == high)) atomicAdd(&hist[256 * round + bin], 1);
    __syncthreads();
    const int got = 255 - nth_bin(hist + 256 * round, k);
    if (round == 0) high = got;
    else low = got;
  }
  return (high << 8 | low) - (1 << 15);
}

// The segments of s0 .. s1 whose maximum reaches `lo`, into sh.list; their number in sh.nlist (0 on entry).
__device__ __forceinline__ int list_segments(RowState& sh, int s0, int s1, int lo) {
  const int t = threadIdx.x, lane = t & 63;
  const bool f = t >= s0 && t < s1 && sh.skey[t] >= lo;        // kMaxSegs <= kRowThreads
  const unsigned long long on = __ballot(f);
  int base = 0;
  if (on) {
    if (lane == 0) base = atomicAdd(&sh.nlist, __popcll(on));
    base = __builtin_amdgcn_readfirstlane(base);
    if (f) sh.list[base + __popcll(on & ((1ull << lane) - 1))] = t;
  }
  __syncthreads();
  return sh.nlist;
}

// Calls f(segment, its 8 logits of this lane) for every listed segment, a wave at a time.
template <bool HALF, typename F>
__device__ __forceinline__ void each_listed(const SampleArgs& a, const u16* x, int off, const int* list, int nlist, F&& f) {
  const int lane = threadIdx.x & 63;
  for (int i0 = uniform(threadIdx.x >> 6); i0 < nlist; i0 += kAhead * kRowWaves) {
    u32x4_t v[kAhead];
    int s[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * kRowWaves;
      s[u] = i < nlist ? uniform(list[i]) : -1;
      if (s[u] >= 0) v[u] = load8<HALF>(x, s[u] * kSegVals + 8 * lane - off, a.V);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (s[u] < 0) break;
      f(s[u], v[u]);
    }
  }
}

// Counts 8 logits of a lane by key, bin hi - key for lo <= key <= hi; PAIRS: two bins of 16 bits an int.
template <bool HALF, bool PAIRS>
__device__ __forceinline__ void count_seg(const u32x4_t& v, int* bins, int hi, int lo) {
  int k[8];
  keys8(v, k);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const u32 b = (u32)(hi - k[j]);
    if (b <= (u32)(hi - lo)) atomicAdd(&bins[PAIRS ? b >> 1 : b], PAIRS ? 1 << (16 * (b & 1)) : 1);
  }
}

// All logits of the listed segments.
template <bool HALF>
__device__ __forceinline__ void count_keys(const SampleArgs& a, const u16* x, int off, RowShared& sh, int nlist, int hi,
                                           int lo) {
  for (int i = threadIdx.x; i <= hi - lo; i += kRowThreads) sh.bins[i] = 0;
  __syncthreads();
  each_listed<HALF>(a, x, off, sh.list, nlist, [&](int, const u32x4_t& v) { count_seg<HALF, false>(v, sh.bins, hi, lo); });
  __syncthreads();
}

// The weights of falling keys, one after another: inside an octave the values are evenly spaced, so each weight is
// the one before times a constant. A power of two is formed anew at each octave's end.
template <bool HALF>
struct FallingWeights {
  int key, left;
  double w, ratio;
  __device__ __forceinline__ void start(int k, float m, double c, double mc) {
    constexpr int kOctave = HALF ? 1024 : 128;
    const float x = val_of_key<HALF>(k);
    key = k;
    w = weight(x, m, c, mc);
    left = k > 0 ? ((k - 1) & (kOctave - 1)) + 1 : kOctave - (-k & (kOctave - 1));
    ratio = exp2_neg(((double)val_of_key<HALF>(k - 1) - (double)x) * c);
  }
  __device__ __forceinline__ void next(float m, double c, double mc) {
    if (--left == 0) start(key - 1, m, c, mc);
    else {
      w *= ratio;
      --key;
    }
  }
};

// p of a token of logit x (-inf for one outside the vocabulary)
template <bool HALF>
__device__ __forceinline__ double px_of(const SampleArgs& a, const RowInfo& r, int v, float x) {
  if (!(x > -INFINITY && r.z > 0)) return 0;          // NaN too
  const int k = key_of_float<HALF>(x);
  return k > r.thr || (k == r.thr && v <= r.cut) ? weight(x, r.m, a.c) / r.z : 0;
}

// Four values a lane, in thread order over the 256 of one wave: their running sums' start and the whole.
__device__ __forceinline__ double scan4(const double (&v)[4], double& total) {
  const double in = wave_scan((v[0] + v[1]) + (v[2] + v[3]));
  total = lane_value(in, 63);
  return lane_before(in);
}

enum { kDrawRow = 0, kDrawRest = 1, kDrawOther = 2 };   // r = p, max(p - q, 0), p without one token

struct DrawIn {                        // what a row's own draw goes by
  int mode, skip;                      // mode < 0: none
  const float* q;
  double u;
};

// Most workgroups that count a row together: each hands over its counts, which the last one joins (15 rows of 151936: 36.7
// us by one workgroup a row, 25.1 by 4, 23.8 by 8, 24.8 by 16; one row 22.4 by 4, 20.5 by 8 and by 16).
constexpr int kGroup = 8;
constexpr int kGroupBins = 2 * kBins;  // values that they count: 16-bit counts
constexpr int kOwn = 2;                // segments of a wave whose loads are out together
struct Group {                         // a row counted by several workgroups, each over its own run of segments
  uint64_t* counts;                    // of each workgroup, 4 bins of 16 bits a word; null: one workgroup a row
  int* arrived;                        // workgroups of this row that are done
  int g, n;
};

// Starts on a row: the keys of its segments' maxima (sm: of this thread's), the row's maximum; what is counted later, 0.
template <bool HALF>
__device__ __forceinline__ float row_start(const SampleArgs& a, float sm, RowState& sh) {
  const int t = threadIdx.x;
  float mx = wave_max(sm);
  if ((t & 63) == 0) sh.red_f[t >> 6] = mx;
  if (t < a.nseg) sh.skey[t] = key_of_float<HALF>(sm);
  if (t == 0) sh.ncand = sh.nlist = 0;
  if (t < 512) sh.cnt[t] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowWaves; ++i) mx = fmaxf(mx, sh.red_f[i]);
  return mx;
}

// Of a row without any logit over -inf: nothing to draw from.
__device__ __forceinline__ RowInfo empty_row(float mx) { return RowInfo{0.0, 0.0, mx, 1 << 16, kNoTies, 0}; }

// A key that the top_k largest logits of a row reach (top: the largest): the k-th largest maximum of its segments, or
// of their parts.
template <bool HALF>
__device__ __forceinline__ int top_k_bound(const SampleArgs& a, const u16* x, int off, float sm, int top, RowState& sh) {
  const int t = threadIdx.x, lane = t & 63;
  if (a.parts) {
    for (int s = uniform(t >> 6); s < a.nseg; s += kRowWaves) {
      const u32x4_t v = load8<HALF>(x, s * kSegVals + 8 * lane - off, a.V);
      int ks[8], k = kLowKey<HALF>;
      keys8(v, ks);
#pragma unroll
      for (int j = 0; j < 8; ++j) k = max(k, ks[j] <= top ? ks[j] : k);
      k = max(k, dpp_i<0xB1, 0xF>(k));   // the exchanges of sum8_lanes
      k = max(k, dpp_i<0x4E, 0xF>(k));
      k = max(k, dpp_i<0x141, 0xF>(k));
      if (a.parts == 4) k = max(k, dpp_i<0x140, 0xF>(k));
      const int each = 64 / a.parts;
      if ((lane & (each - 1)) == 0) sh.list[a.parts * s + lane / each] = k;
    }
    __syncthreads();
    const int k = kth_key(t < a.parts * a.nseg, sh.list[t], a.top_k, sh.cnt);
    __syncthreads();
    return k;
  }
  return a.nseg >= a.top_k ? kth_key(t < a.nseg, key_of_float<HALF>(sm), a.top_k, sh.cnt) : kLowKey<HALF>;
}

// Logits that `take` (of a lane's keys: which of the 8) picks from the listed segments, into fw.cand as far as there is
// room; how many (sh.ncand, 0 on entry).
template <bool HALF, typename F>
__device__ __forceinline__ int gather(const SampleArgs& a, const u16* x, int off, int nlist, RowState& sh, Few& fw, F&& take) {
  const int lane = threadIdx.x & 63;
  each_listed<HALF>(a, x, off, sh.list, nlist, [&](int s, const u32x4_t& v) {
    const int v0 = s * kSegVals + 8 * lane - off;
    int ks[8];
    keys8(v, ks);
    const u32 on = take(s, ks);
    const int n = __popc(on), upto = wave_scan(n);
    int base = 0;
    if (lane == 63) base = atomicAdd(&sh.ncand, upto);
    int at = __builtin_amdgcn_readlane(base, 63) + upto - n;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (on >> j & 1) {
        if (at < kListed) fw.cand[at] = (uint64_t)(u32)(ks[j] + (1 << 15)) << 32 | (u32)~(v0 + j);
        ++at;
      }
    }
  });
  __syncthreads();
  return sh.ncand;
}

// More candidates than are sorted: the top_k themselves. Their least key by counts of its bytes over the candidates, what
// is above it, and the first by index of what equals it.
template <bool HALF>
__device__ __forceinline__ int gather_top(const SampleArgs& a, const u16* x, int off, int nlist, int kb, int top, RowState& sh,
                                          Few& fw) {
  const int t = threadIdx.x, lane = t & 63;
  int k = a.top_k, high = 0, low = 0;
  __syncthreads();
  if (t < 512) sh.cnt[t] = 0;
  if (t == 0) sh.ncand = 0;
  __syncthreads();
  for (int round = 0; round < 2; ++round) {
    each_listed<HALF>(a, x, off, sh.list, nlist, [&](int, const u32x4_t& v) {
      int ks[8];
      keys8(v, ks);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int u = ks[j] + (1 << 15);
        if (ks[j] >= kb && ks[j] <= top && (!round || u >> 8 == high))
          atomicAdd(&sh.cnt[256 * round + 255 - (round ? u & 255 : u >> 8)], 1);
      }
    });
    __syncthreads();
    const int got = 255 - nth_bin(sh.cnt + 256 * round, k);
    if (round == 0) high = got;
    else low = got;
  }
  const int thr = (high << 8 | low) - (1 << 15);       // k of the logits that equal it
  __syncthreads();
  if (t < a.nseg) sh.cnt[t] = 0;
  __syncthreads();
  each_listed<HALF>(a, x, off, sh.list, nlist, [&](int s, const u32x4_t& v) {
    int n = 0, ks[8];
    keys8(v, ks);
#pragma unroll
    for (int j = 0; j < 8; ++j) n += __popcll(__ballot(ks[j] == thr));
    if (lane == 0) sh.cnt[s] = n;
  });
  __syncthreads();
  int upto, all;
  const int before = block_scan(t < a.nseg ? sh.cnt[t] : 0, sh.red_i, upto, all);
  if (t < a.nseg) sh.cnt[t] = before;
  __syncthreads();
  return gather<HALF>(a, x, off, nlist, sh, fw, [&](int s, const int (&ks)[8]) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) n += ks[j] == thr;
    int rank = sh.cnt[s] + wave_scan(n) - n;
    u32 on = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if ((ks[j] > thr && ks[j] <= top) || (ks[j] == thr && rank < k)) on |= 1u << j;
      rank += ks[j] == thr;
    }
    return on;
  });
}

// What is kept of the n candidates of fw.cand (total: the mass of the whole row, where there is no top_k), px of token
// `draft`, and the token drawn (d.mode >= 0; else -1).
template <bool HALF>
__device__ __forceinline__ void sorted_row(const SampleArgs& a, int n, float mx, double total, int draft, float xd,
                                           const DrawIn& d, RowState& sh, Few& fw, RowInfo& out, int& token) {
  const int t = threadIdx.x;
  const double mc = -(double)mx * a.c;
  out.m = mx;
  out.pad = 0;
  if (t < n) {
    const uint64_t me = fw.cand[t];
    int r = 0;
    for (int i = 0; i < n; ++i) r += fw.cand[i] > me;
    fw.sorted[r] = me;
  }
  __syncthreads();
  const int idx = t < n ? (int)~(u32)fw.sorted[t] : 0;
  const float qv = d.mode == kDrawRest && t < n ? d.q[idx] : 0.f;      // on its way over the next step
  if (t < 64) {                     // the first wave, four a lane: what of the top_k lies before the mass
    double w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = 4 * t + i;
      w[i] = j < n && !(a.top_k && j >= a.top_k)
                 ? weight(val_of_key<HALF>((int)(fw.sorted[j] >> 32) - (1 << 15)), mx, a.c, mc) : 0.0;
      if (j < n) fw.w[j] = w[i];
    }
    double zk;
    double run = scan4(w, zk);
    const double goal = a.top_p * (a.top_k ? zk : total);
    const int nk = a.top_k ? min(a.top_k, n) : n;
    int kept = nk;                  // tokens of this lane or before it that are kept, if the cut is here
    double z = zk;
#pragma unroll
    for (int i = 3; i >= 0; --i) {  // the first at which the goal is reached, from the lane's last
      const double before = i == 0 ? run : i == 1 ? run + w[0] : i == 2 ? run + w[0] + w[1] : run + w[0] + w[1] + w[2];
      if (4 * t + i < nk && before >= goal && a.top_p < 1.0) {
        kept = 4 * t + i;
        z = before;
      }
    }
    const unsigned long long hit = __ballot(kept < nk);
    if (hit) {
      const int at = __ffsll(hit) - 1;
      kept = __builtin_amdgcn_readlane(kept, at);
      z = lane_value(z, at);
    }
    if (t == 0) {
      sh.keep = kept;               // at least 1: before is 0 at the first, the goal is not
      sh.z = z;
      sh.key = (int)(fw.sorted[kept - 1] >> 32) - (1 << 15);
      sh.cut = (int)~(u32)fw.sorted[kept - 1];
    }
  }
  __syncthreads();
  const int kept = sh.keep;
  out.z = sh.z;
  out.thr = sh.key;
  out.cut = sh.cut;
  out.px = px_of<HALF>(a, out, draft, xd);
  token = -1;
  if (d.mode < 0) return;
  // the draw: r by index, then the first wave, four a lane
  if (t < kept) {
    int at = 0;
    for (int i = 0; i < kept; ++i) at += (int)~(u32)fw.sorted[i] < idx;
    double r = fw.w[t];
    if (d.mode == kDrawRest) r = __builtin_fmax(r / out.z - (double)qv, 0.0);
    else if (d.mode == kDrawOther && idx == d.skip) r = 0;
    fw.r[at] = r;
    fw.order[at] = t;
  }
  __syncthreads();
  if (t < 64) {
    double r[4], all = 0, run = 0;
    for (int tries = 0; tries < 2; ++tries) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 4 * t + i;
        r[i] = j < kept ? (tries ? fw.w[fw.order[j]] : fw.r[j]) : 0.0;      // r zero throughout: p
      }
      run = scan4(r, all);
      if (all > 0) break;
    }
    const double goal = d.u * all;
    int pick = kListed, last = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      run += r[i];
      if (r[i] > 0) {
        last = 4 * t + i;
        if (run > goal && pick == kListed) pick = last;
      }
    }
    const unsigned long long hit = __ballot(pick < kListed), any = __ballot(last >= 0);
    // the last one with any mass where none passes the goal by a rounding
    const int j = hit ? __builtin_amdgcn_readlane(pick, __ffsll(hit) - 1)
                      : any ? __builtin_amdgcn_readlane(last, 63 - __clzll(any)) : -1;
    if (t == 0) sh.token = j >= 0 ? (int)~(u32)fw.sorted[fw.order[j]] : 0;
  }
  __syncthreads();
  token = sh.token;
}

// A row of a small top_k: what is kept of it, px of token `draft`, and the token drawn from it. WHOLE: there was no launch
// before this one, the segments' maxima are formed here.
template <bool HALF, bool WHOLE>
__device__ __forceinline__ void cut_row(const SampleArgs& a, int seq, int ri, int draft, const DrawIn& d, RowState& sh, Few& fw,
                                        RowInfo& out, int& token) {
  const int t = threadIdx.x;
  const u16* x = row_ptr(a, seq, ri);
  const int off = row_off(x);
  float sm = -INFINITY;                 // kMaxSegs <= kRowThreads
  if constexpr (WHOLE) {
    for (int s0 = uniform(t >> 6); s0 < a.nseg; s0 += kAhead * kRowWaves) {
      u32x4_t v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (s0 + u * kRowWaves < a.nseg) v[u] = load8<HALF>(x, (s0 + u * kRowWaves) * kSegVals + 8 * (t & 63) - off, a.V);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s0 + u * kRowWaves >= a.nseg) break;
        const float m = max8_wave<HALF>(v[u]);
        if ((t & 63) == 0) fw.segm[s0 + u * kRowWaves] = m;
      }
    }
    __syncthreads();
    if (t < a.nseg) sm = fw.segm[t];
  } else {
    if (t < a.nseg) sm = a.segm[((long)seq * a.per + ri) * a.nseg + t];
  }
  const float xd = draft >= 0 && draft < a.V ? val<HALF>(x[draft]) : -INFINITY;
  const float mx = row_start<HALF>(a, sm, sh);
  if (!(mx > -INFINITY)) {
    out = empty_row(mx);
    token = 0;
    return;
  }
  const int top = key_of_float<HALF>(mx);
  const int kb = min(max(top_k_bound<HALF>(a, x, off, sm, top, sh), kLowKey<HALF> + 1), top);
  const int nlist = list_segments(sh, 0, a.nseg, kb);
  int n = gather<HALF>(a, x, off, nlist, sh, fw, [&](int, const int (&ks)[8]) {
    u32 on = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) on |= (u32)(ks[j] >= kb && ks[j] <= top) << j;
    return on;
  });
  if (n > kListed) n = gather_top<HALF>(a, x, off, nlist, kb, top, sh, fw);
  sorted_row<HALF>(a, n, mx, 0.0, draft, xd, d, sh, fw, out, token);
}

// The part of one row that is sampled from: its threshold and normaliser (RowInfo), and px of token `draft`. False in
// the workgroups of a group that leave the row to another.
template <bool HALF>
__device__ __forceinline__ bool select_row(const SampleArgs& a, int seq, int ri, int draft, const Group& gr, RowShared& sh,
                                           RowInfo& out) {
  const int t = threadIdx.x, lane = t & 63;
  const u16* x = row_ptr(a, seq, ri);
  const int off = row_off(x);
  const long row = (long)seq * a.per + ri;
  const float sm = t < a.nseg ? a.segm[row * a.nseg + t] : -INFINITY;      // kMaxSegs <= kRowThreads
  const double ss = !a.top_k && t < a.nseg ? a.segs[row * a.nseg + t] : 0;
  // of a group: this workgroup's run of segments, those of a wave kRowWaves apart, its first ones on their way
  const int wave = uniform(t >> 6), spg = (a.nseg + gr.n - 1) / gr.n, s_end = min((gr.g + 1) * spg, a.nseg);
  u32x4_t own[kOwn];
  const auto load_own = [&](int s) {
#pragma unroll
    for (int u = 0; u < kOwn; ++u)
      if (s + u * kRowWaves < s_end) own[u] = load8<HALF>(x, (s + u * kRowWaves) * kSegVals + 8 * lane - off, a.V);
  };
  if (gr.counts) load_own(gr.g * spg + wave);
  const float mx = row_start<HALF>(a, sm, sh);
  if (!(mx > -INFINITY)) {
    out = empty_row(mx);
    return gr.g == 0;
  }
  out.m = mx;
  out.pad = 0;
  const double mc = -(double)mx * a.c;
  double total = 0;                     // of the whole row; needed where the mass itself is cut
  if (!a.top_k) {
    const double part = wave_total(ss * weight(sm, mx, a.c, mc));
    if (lane == 0) sh.red_d[t >> 6] = part;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRowWaves; ++i) total += sh.red_d[i];
  }
  const int top = key_of_float<HALF>(mx);
  const float xd = draft >= 0 && draft < a.V ? val<HALF>(x[draft]) : -INFINITY;

  // a key that every kept token reaches
  int kb = kLowKey<HALF>;
  if (!a.top_k) {
    // tokens of weight (1 - top_p) S / V or less: all together less than (1 - top_p) S. Room for an fp32 logarithm,
    // and one key for the rounding to 16 bits.
    const float w = (float)((1.0 - a.top_p) * total) / (float)a.V;
    kb = key_of_float<HALF>(mx + (__builtin_amdgcn_logf(w) - 1e-4f) / (float)a.c) - 1;
  } else {
    kb = top_k_bound<HALF>(a, x, off, sm, top, sh);
  }
  kb = min(max(kb, kLowKey<HALF> + 1), top);
  int nlist;
  if (gr.counts) {                      // their number alone
    const unsigned long long on = __ballot(t < a.nseg && sh.skey[t] >= kb);
    if (lane == 0 && on) atomicAdd(&sh.nlist, __popcll(on));
    __syncthreads();
    nlist = sh.nlist;
  } else {
    nlist = list_segments(sh, 0, a.nseg, kb);
  }

  // Few candidates are sorted. A top_k leaves little more than that many; a mass alone may leave most of a segment,
  // so that only rows where few segments reach are tried.
  const bool few = nlist <= (a.top_k ? kAhead * kRowWaves : kRowWaves / 2);
  const bool grouped = gr.counts && !few;
  const auto list_all = [&]() {
    __syncthreads();
    if (t == 0) sh.nlist = 0;
    __syncthreads();
    nlist = list_segments(sh, 0, a.nseg, kb);
  };
  if (few) {
    if (gr.g) return false;             // the first workgroup's alone
    if (gr.counts) list_all();
    const int n = gather<HALF>(a, x, off, nlist, sh, sh.few, [&](int, const int (&ks)[8]) {
      u32 on = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) on |= (u32)(ks[j] >= kb && ks[j] <= top) << j;
      return on;
    });
    if (n <= kListed) {
      int token;
      sorted_row<HALF>(a, n, mx, total, draft, xd, DrawIn{-1, -1, nullptr, 0.0}, sh, sh.few, out, token);
      return true;
    }
    __syncthreads();
  }

  int thr = kb - 1, keep = 0, ties = 0;  // thr = kb - 1: every listed token
  int range_hi = -(1 << 17), range_lo = 0;             // the keys now in the bins, bin range_hi - key
  int merged_hi = -(1 << 17), merged_lo = 0;           // of a group's counts: joined in the bins, bin merged_hi - key
  const int group_lo = max(kb, top - kGroupBins + 1);  // a group counts this far; what is below, its last workgroup alone
  const int words = (top - group_lo + 4) >> 2;
  if (grouped) {
    // a value at most as often as spg segments have logits: below 2^16
    for (int i = t; i < 2 * words; i += kRowThreads) sh.bins[i] = 0;
    __syncthreads();
    for (int s = gr.g * spg + wave; s < s_end; s += kOwn * kRowWaves) {
      if (s >= gr.g * spg + kOwn * kRowWaves) load_own(s);
#pragma unroll
      for (int u = 0; u < kOwn; ++u) {
        const int at = s + u * kRowWaves;
        if (at < s_end && uniform(sh.skey[at]) >= kb) count_seg<HALF, true>(own[u], sh.bins, top, group_lo);
      }
    }
    __syncthreads();
    uint64_t* out_c = gr.counts + (long)gr.g * (kGroupBins / 4);
    for (int i = t; i < words; i += kRowThreads) put_far(out_c + i, (uint64_t)(u32)sh.bins[2 * i] | (uint64_t)(u32)sh.bins[2 * i + 1] << 32);
    if (!arrives_last(gr.arrived, gr.n, &sh.last)) return false;
  }
  bool exchanged = grouped;              // the counts are a group's
  double z = 0;
  bool found = false;
  // two passes over the values in falling order: the top_k-th token, then the mass top_p
  for (int pass = a.top_k ? 0 : 1; pass < 2; ++pass) {
    const int lowest = pass == 1 && found ? thr : kb;    // top_p goes by the tokens of top_k
    const int thr_k = thr, keep_k = keep, ties_k = ties;
    const bool after_k = pass == 1 && found;
    if (pass == 1) {
      if (!(a.top_p < 1.0)) break;
      if (a.top_k) total = z;
    }
    const double goal = a.top_p * total;
    int seen = 0;
    double mass = 0;
    found = false;
    for (int hi = top, lo, span = kChunk<HALF>; hi >= lowest && !found; hi = lo - 1, span = min(4 * span, kBins - 4)) {
      lo = max(lowest, hi - span + 1);
      if (exchanged && hi < group_lo) {
        list_all();
        exchanged = false;
      }
      int base;                          // the bin of hi
      if (exchanged) {
        lo = max(lo, group_lo);
        if (merged_hi != hi || merged_lo > lo) {
          const int w0 = (top - hi) >> 2;
          for (int i = w0 + t; i <= (top - lo) >> 2; i += kRowThreads) {
            int c[4] = {};
            uint64_t w[kGroup];          // every workgroup's word at once
#pragma unroll
            for (int g = 0; g < kGroup; ++g) w[g] = g < gr.n ? get_far(gr.counts + (long)g * (kGroupBins / 4) + i) : 0;
#pragma unroll
            for (int g = 0; g < kGroup; ++g)
#pragma unroll
              for (int j = 0; j < 4; ++j) c[j] += (int)(w[g] >> (16 * j) & 0xFFFF);
#pragma unroll
            for (int j = 0; j < 4; ++j) sh.bins[4 * (i - w0) + j] = c[j];
          }
          merged_hi = hi;
          merged_lo = lo;
          __syncthreads();
        }
        base = (top - hi) & 3;
      } else {
        if (hi > range_hi || hi < range_lo) {
          range_hi = hi;
          range_lo = max(kb, hi - kBins + 1);
          count_keys<HALF>(a, x, off, sh, nlist, range_hi, range_lo);
        }
        lo = max(lo, range_lo);
        base = range_hi - hi;
      }
      // a run of bins a thread, an odd number of them: neighbours read other banks
      const int nb = hi - lo + 1, each = ((nb + kRowThreads - 1) / kRowThreads) | 1;
      static_assert(kBins / kRowThreads < 64, "a lane for every bin of a run");
      const int b0 = min(t * each, nb), b1 = min(b0 + each, nb);
      int cn = 0;
      double cm = 0;
      int some = 0;                      // values near zero are many, and mostly nobody's
      for (int b = b0; b < b1; ++b) some |= sh.bins[base + b];
      if (some) {
        FallingWeights<HALF> f;
        f.start(hi - b0, mx, a.c, mc);
        for (int b = b0; b < b1; ++b) {
          int n = sh.bins[base + b];
          if (after_k && hi - b == thr_k) n = keep_k;
          cn += n;
          cm += (double)n * f.w;
          if (b + 1 < b1) f.next(mx, a.c, mc);
        }
      }
      // running sums over the waves, a wave a lane, and the first wave with tokens in which the goal is reached
      const double m_in = wave_scan(cm);
      const int c_in = wave_scan(cn);
      if (lane == 63) {
        sh.red_d[wave] = m_in;
        sh.red_i[wave] = c_in;
      }
      __syncthreads();
      const double m_w = lane < kRowWaves ? sh.red_d[lane] : 0.0, m_to = wave_scan(m_w);
      const int c_w = lane < kRowWaves ? sh.red_i[lane] : 0, c_to = wave_scan(c_w);
      const unsigned long long there = __ballot(c_w && (pass == 0 ? seen + c_to >= a.top_k : mass + m_to >= goal));
      const int owner = there ? __ffsll(there) - 1 : kRowWaves;
      const double mass_before = mass + lane_value(lane_before(m_to), wave);
      const int cnt_before = seen + __builtin_amdgcn_readlane(c_to - c_w, wave);
      mass += lane_value(m_to, 63);
      seen += __builtin_amdgcn_readlane(c_to, 63);
      if (wave == owner) {              // its lane's bins, a bin a lane
        const unsigned long long reached = __ballot(cn && (pass == 0 ? cnt_before + c_in >= a.top_k : mass_before + m_in >= goal));
        const unsigned long long some = __ballot(cn > 0);
        const int from = reached ? __ffsll(reached) - 1 : 63 - __clzll(some);
        const int run_c = __builtin_amdgcn_readlane(cnt_before + lane_before(c_in), from);
        const double run_m = lane_value(mass_before + lane_before(m_in), from);
        const int b = (64 * wave + from) * each + lane;
        const bool in = lane < each && b < nb;
        const int n_all = in ? sh.bins[base + b] : 0;
        const int n = after_k && hi - b == thr_k && in ? keep_k : n_all;
        const double w = in ? weight(val_of_key<HALF>(hi - b), mx, a.c, mc) : 0.0;
        const int c_end = run_c + wave_scan(n), c0 = c_end - n;
        const double mb = wave_scan((double)n * w), m0 = run_m + lane_before(mb), m_end = run_m + mb;
        const bool reach = n && (pass == 0 ? c_end >= a.top_k : m_end >= goal);
        const unsigned long long hit = __ballot(reach), any = __ballot(n > 0);
        const int at = hit ? __ffsll(hit) - 1 : 63 - __clzll(any);       // the last of the run but for a rounding
        if (lane == at) {
          int r = n;
          if (hit && pass == 0) r = a.top_k - c0;
          if (hit && pass == 1) {       // tokens of this value before which less than the goal lies
            r = (int)fmin(fmax(__builtin_ceil((goal - m0) / w), 1.0), (double)n);
            while (r > 1 && m0 + (double)(r - 1) * w >= goal) --r;
            while (r < n && m0 + (double)r * w < goal) ++r;
          }
          sh.key = hi - b;
          sh.keep = r;
          sh.ties = n_all;
          sh.z = m0 + (double)r * w;
        }
      }
      __syncthreads();
      found = owner < kRowWaves;
      if (found) {
        thr = sh.key;
        keep = sh.keep;
        ties = sh.ties;
        z = sh.z;
      }
      __syncthreads();
    }
    if (!found) {                       // fewer tokens than top_k, or the goal is the whole mass but for a rounding
      z = mass;
      thr = after_k ? thr_k : kb - 1;
      keep = after_k ? keep_k : 0;
      ties = after_k ? ties_k : 0;
    }
  }
  out.thr = thr;
  out.z = z;
  out.cut = ties ? a.V : kNoTies;       // without a threshold value (thr = kb - 1) no token has that key
  if (keep < ties) {                    // the index of the last kept token of the threshold's value
    // the keep-th logit of the threshold's value among a lane's 8 from index v0, by one wave
    const auto place = [&](const u32x4_t& v, int v0, int want) {
      int n = 0, ks[8];
      keys8(v, ks);
#pragma unroll
      for (int j = 0; j < 8; ++j) n += ks[j] == thr;
      int run = wave_scan(n) - n;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (ks[j] == thr && ++run == want) sh.cut = v0 + j;
    };
    const auto count = [&](const u32x4_t& v) {
      int n = 0, ks[8];
      keys8(v, ks);
#pragma unroll
      for (int j = 0; j < 8; ++j) n += __popcll(__ballot(ks[j] == thr));
      return n;
    };
    if (grouped && thr >= group_lo) {   // the run of segments it lies in, by the groups' own counts
      const int b = top - thr;
      const int c = lane < gr.n ? (int)(get_far(gr.counts + (long)lane * (kGroupBins / 4) + (b >> 2)) >> (16 * (b & 3)) & 0xFFFF) : 0;
      const int upto = wave_scan(c), at = __ffsll(__ballot(upto >= keep)) - 1;
      keep -= __builtin_amdgcn_readlane(upto - c, at);
      const int s0 = at * spg, s1 = min(s0 + spg, a.nseg);
      for (int s = s0 + wave; s < s1; s += kOwn * kRowWaves) {
#pragma unroll
        for (int u = 0; u < kOwn; ++u)
          if (s + u * kRowWaves < s1) own[u] = load8<HALF>(x, (s + u * kRowWaves) * kSegVals + 8 * lane - off, a.V);
#pragma unroll
        for (int u = 0; u < kOwn; ++u) {
          if (s + u * kRowWaves >= s1) break;
          const int n = count(own[u]);
          if (lane == 0) sh.cnt[s + u * kRowWaves - s0] = n;
        }
      }
      __syncthreads();
      int first = 0;                    // the segment, by every wave for itself
      for (int i = 0; i < s1 - s0; i += 64) {
        const int n = i + lane < s1 - s0 ? sh.cnt[i + lane] : 0, end = wave_scan(n);
        const unsigned long long hit = __ballot(end >= keep);
        if (hit) {
          const int l = __ffsll(hit) - 1;
          first = i + l;
          keep -= __builtin_amdgcn_readlane(end - n, l);
          break;
        }
        keep -= __builtin_amdgcn_readlane(end, 63);
      }
      if ((first & (kRowWaves - 1)) == wave) {
        const int v0 = (s0 + first) * kSegVals + 8 * lane - off;
        static_assert(kOwn == 2, "own[0], own[1]");
        u32x4_t v = own[0];
        if (s1 - s0 > kOwn * kRowWaves) v = load8<HALF>(x, v0, a.V);
        else if (first >= kRowWaves) v = own[1];
        place(v, v0, keep);
      }
      __syncthreads();
    } else {
      if (t == 0) sh.nlist = 0;
      if (t < a.nseg) sh.cnt[t] = 0;
      __syncthreads();
      nlist = list_segments(sh, 0, a.nseg, thr);
      each_listed<HALF>(a, x, off, sh.list, nlist, [&](int s, const u32x4_t& v) {
        const int n = count(v);
        if (lane == 0) sh.cnt[s] = n;
      });
      __syncthreads();
      const int c = t < a.nseg ? sh.cnt[t] : 0;
      int upto, all;
      const int before = block_scan(c, sh.red_i, upto, all);
      if (before < keep && keep <= upto) {
        sh.owner = t;
        sh.keep = keep - before;
      }
      __syncthreads();
      if (t < 64) {
        const int v0 = sh.owner * kSegVals + 8 * lane - off;
        place(load8<HALF>(x, v0, a.V), v0, sh.keep);
      }
      __syncthreads();
    }
    out.cut = sh.cut;
  }
  out.px = px_of<HALF>(a, out, draft, xd);
  return true;
}

// ---------------------------------------------------------------- the accept rule

__device__ __forceinline__ double uniform_at(const VerifyIn& in, long at) {
  return in.u64 ? static_cast<const double*>(in.u)[at] : (double)static_cast<const float*>(in.u)[at];
}
__device__ __forceinline__ int drafts_of(const SampleArgs& a, const VerifyIn& in, int seq) {
  return in.lens ? min(max(in.lens[seq], 0), a.per - 1) : a.per - 1;
}

// How the token of row i is drawn if its draft is the first refused, or it is the row after the last draft.
__device__ __forceinline__ DrawIn draw_in(const SampleArgs& a, const VerifyIn& in, int seq, int i, int len) {
  DrawIn d;
  d.mode = i == len ? kDrawRow : in.q ? kDrawRest : kDrawOther;
  d.q = d.mode == kDrawRest ? in.q + seq * in.qb + i * in.qr : nullptr;
  d.skip = i < len ? in.draft[(long)seq * (a.per - 1) + i] : -1;
  d.u = uniform_at(in, (long)seq * a.per + a.per - 1);
  return d;
}

// q of a lane's 8 tokens from index v0, 0 outside the row.
__device__ __forceinline__ void load_q8(const float* q, int v0, int V, float (&out)[8]) {
  if (v0 >= 0 && v0 + 8 <= V && (reinterpret_cast<uintptr_t>(q + v0) & 15) == 0) {
    const f32x4_t a = *reinterpret_cast<const f32x4_t*>(q + v0), b = *reinterpret_cast<const f32x4_t*>(q + v0 + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      out[j] = a[j];
      out[4 + j] = b[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = v0 + j >= 0 && v0 + j < V ? q[v0 + j] : 0.f;
  }
}

// r of 8 logits from index v0 (q: of the same tokens, where the mode asks for it). Without a cut every
// logit's weight is formed; with one, those of which some lane keeps its own.
template <bool HALF, bool CUT>
__device__ __forceinline__ void rest8(const SampleArgs& a, const RowInfo& r, double inv, const u32x4_t& x, int v0, int mode,
                                      const float (&q)[8], int skip, double (&out)[8]) {
  const double mc = -(double)r.m * a.c;
  int ks[8];
  if constexpr (CUT) keys8(x, ks);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int v = v0 + j;
    const bool kept = !CUT || ks[j] > r.thr || (ks[j] == r.thr && v <= r.cut);       // a NaN's weight is 0
    double w = 0;
    if (!CUT || __any(kept)) {
      w = weight(val<HALF>(bits_of(x, j)), r.m, a.c, mc);
      if (mode == kDrawRest) w = __builtin_fmax(w * inv - (double)q[j], 0.0);
      else if (mode == kDrawOther && v == skip) w = 0;
      w = kept ? w : 0.0;
    }
    out[j] = w;
  }
}

struct DrawShared {
  double sums[kMaxSegs];
  double red[kRowWaves];
  double before;
  int list[kMaxSegs];                  // segments with a kept token
  int nlist, seg, last, token, first;
};

// The token drawn from row ri of a sequence: the first whose running sum of r passes u times the whole.
// `rest`: segment sums of r, by every workgroup of the launch (without a cut, only where r is max(p - q, 0): else they
// follow from the segments' own).
template <bool HALF, bool CUT>
__device__ __forceinline__ int draw_token(const SampleArgs& a, const RowInfo& r, int seq, int ri, const DrawIn& d,
                                          const double* rest, DrawShared& sh) {
  const int t = threadIdx.x, lane = t & 63;
  const u16* x = row_ptr(a, seq, ri);
  const int off = row_off(x);
  const long row = (long)seq * a.per + ri;
  const double inv = r.z > 0 ? 1.0 / r.z : 0.0;
  int mode = d.mode;
  if (t == 0) {
    sh.token = 0;
    sh.seg = kMaxSegs;
    sh.last = -1;
    sh.nlist = 0;
  }
  // sums of r over the segments; where r is zero throughout, of p
  const float sm = t < a.nseg ? a.segm[row * a.nseg + t] : -INFINITY;
  double all = 0, before = 0, upto = 0, mine = 0;
  if constexpr (CUT) {
    __syncthreads();
    const bool f = r.z > 0 && t < a.nseg && key_of_float<HALF>(sm) >= r.thr;
    if (f) sh.list[atomicAdd(&sh.nlist, 1)] = t;
    sh.sums[t] = t < a.nseg ? __builtin_bit_cast(double, get_far(reinterpret_cast<const uint64_t*>(rest) + t)) : 0;
    static_assert(kMaxSegs == kRowThreads, "a slot a thread");
    __syncthreads();
  }
  for (int tries = 0; tries < 2; ++tries) {
    if constexpr (CUT) {
      if (tries) each_listed<HALF>(a, x, off, sh.list, sh.nlist, [&](int s, const u32x4_t& v) {      // p
        double w[8], sum = 0;
        const float q[8] = {};
        rest8<HALF, true>(a, r, inv, v, s * kSegVals + 8 * lane - off, kDrawRow, q, -1, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += w[j];
        sum = wave_total(sum);
        if (lane == 0) sh.sums[s] = sum;
      });
    } else {
      if (t < a.nseg) {
        if (mode == kDrawRest) sh.sums[t] = __builtin_bit_cast(double, get_far(reinterpret_cast<const uint64_t*>(rest) + t));
        else sh.sums[t] = r.z > 0 ? a.segs[row * a.nseg + t] * weight(sm, r.m, a.c) : 0.0;
      }
      __syncthreads();
      if (mode == kDrawOther && r.z > 0 && d.skip >= 0 && d.skip < a.V && t < 64) {   // the token's own segment again, without it
        const int s = (d.skip + off) / kSegVals, v0 = s * kSegVals + 8 * lane - off;
        double w[8], sum = 0;
        const float q[8] = {};
        rest8<HALF, false>(a, r, inv, load8<HALF>(x, v0, a.V), v0, mode, q, d.skip, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += w[j];
        sum = wave_total(sum);
        if (lane == 0) sh.sums[s] = sum;
      }
    }
    __syncthreads();
    mine = t < a.nseg ? sh.sums[t] : 0.0;
    before = block_scan(mine, sh.red, upto, all);
    if (all > 0 || mode == kDrawRow) break;
    mode = kDrawRow;
  }
  // the first segment whose running sum passes the goal (the last one with any mass if none does by a rounding)
  const double goal = d.u * all;
  const unsigned long long any_mass = __ballot(mine > 0), passes = __ballot(mine > 0 && upto > goal);
  if (lane == 0 && any_mass) {          // t: the wave's first thread
    atomicMax(&sh.last, t + 63 - __clzll(any_mass));
    if (passes) atomicMin(&sh.seg, t + __ffsll(passes) - 1);
  }
  __syncthreads();
  const int s = sh.seg < kMaxSegs ? sh.seg : sh.last;
  if (s >= 0) {
    if (t == s) sh.before = before;
    __syncthreads();
    if (t < 64) {
      const int v0 = s * kSegVals + 8 * lane - off;
      double w[8], sum = 0;
      float q[8] = {};
      if (mode == kDrawRest) load_q8(d.q, v0, a.V, q);
      rest8<HALF, CUT>(a, r, inv, load8<HALF>(x, v0, a.V), v0, mode, q, d.skip, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += w[j];
      const double to = sh.before + wave_scan(sum);
      unsigned long long hit = __ballot(sum > 0 && to > goal);
      const unsigned long long any = __ballot(sum > 0);
      if (!hit) hit = any ? 1ull << (63 - __clzll(any)) : 0;
      if (hit && lane == __ffsll(hit) - 1) {
        double run = to - sum;
        int pick = 0;
        bool done = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          run += w[j];
          if (w[j] > 0 && !done) {
            pick = v0 + j;
            done = run > goal;
          }
        }
        sh.token = pick;
      }
    }
    __syncthreads();
  }
  return sh.token;
}

__device__ __forceinline__ void write_tokens(const SampleArgs& a, const VerifyIn& in, int seq, int n, int token) {
  for (int i = threadIdx.x; i < a.per; i += kRowThreads)
    in.tokens[(long)seq * a.per + i] = i < n ? in.draft[(long)seq * (a.per - 1) + i] : i == n ? token : -1;
  if (threadIdx.x == 0) in.n[seq] = n;
}

struct CutShared : RowState {
  Few few;
  int first;
};

// Rows of a small top_k: one row a workgroup. It draws its token too, in case its draft is the first refused (the random
// number of the draw is there from the start); the last workgroup of a sequence accepts.
template <bool HALF, bool WHOLE>
__global__ __launch_bounds__(kRowThreads) void sample_cut_kernel(const SampleArgs a, const VerifyIn in, uint64_t* drawn) {
  __shared__ CutShared sh;
  const int ri = blockIdx.x, seq = blockIdx.y, m = a.per - 1, t = threadIdx.x;
  const long row = (long)seq * a.per + ri;
  DrawIn d = {-1, -1, nullptr, 0.0};
  const int len = drafts_of(a, in, seq), draft = ri < m ? in.draft[(long)seq * m + ri] : -1;
  if (ri <= len) d = draw_in(a, in, seq, ri, len);
  const bool inside = draft >= 0 && draft < a.V;
  double uq = 0;
  if (ri < len) uq = inside ? uniform_at(in, row) * (in.q ? (double)d.q[draft] : 1.0) : INFINITY;
  int token;
  RowInfo mine;
  cut_row<HALF, WHOLE>(a, seq, ri, draft, d, sh, sh.few, mine, token);
  if constexpr (WHOLE) {                // rows without drafts
    write_tokens(a, in, seq, 0, token);
    return;
  }
  if (t == 0) {
    if (ri < m) in.px[(long)seq * m + ri] = (float)mine.px;
    put_far(drawn + row, (uint64_t)(ri >= len || !(uq < mine.px)) << 32 | (u32)token);
  }
  if (!arrives_last(a.arrived + seq, a.per, &sh.last)) return;
  if (t == 0) sh.first = len;
  __syncthreads();
  uint64_t res = 0;
  if (t <= len) {                       // kMaxDraft < kRowThreads
    res = get_far(drawn + (long)seq * a.per + t);
    if (res >> 32) atomicMin(&sh.first, t);
  }
  __syncthreads();
  const int n = sh.first;
  if (t == n) sh.token = (int)(u32)res;
  __syncthreads();
  write_tokens(a, in, seq, n, sh.token);
}

__device__ __forceinline__ void write_info(uint64_t* info, long row, const RowInfo& r) {
  static_assert(sizeof(RowInfo) == 32, "four words");
  const int t = threadIdx.x;
  if (t >= 4) return;
  uint64_t w[4];
  __builtin_memcpy(w, &r, 32);
  info[4 * row + t] = t == 0 ? w[0] : t == 1 ? w[1] : t == 2 ? w[2] : w[3];
}

// What is kept of a row of a small top_k, for the launch that writes probabilities.
template <bool HALF>
__global__ __launch_bounds__(kRowThreads) void sample_few_kernel(const SampleArgs a, uint64_t* info) {
  __shared__ CutShared sh;
  int token;
  RowInfo mine;
  cut_row<HALF, false>(a, blockIdx.x, 0, -1, DrawIn{-1, -1, nullptr, 0.0}, sh, sh.few, mine, token);
  write_info(info, blockIdx.x, mine);
}

// The probabilities of a row of a small top_k, by a workgroup that takes it whole: zeros while its logits are on their
// way, then the few that are not.
template <bool HALF>
__global__ __launch_bounds__(kRowThreads) void sample_whole_kernel(const SampleArgs a, float* __restrict__ out, long ldo) {
  __shared__ CutShared sh;
  const int t = threadIdx.x;
  float* y = out + (long)blockIdx.x * ldo;
  const int head = min((int)(-(reinterpret_cast<uintptr_t>(y) >> 2) & 3), a.V), quads = (a.V - head) / 4;
  if (t < head) y[t] = 0.f;
  for (int i = t; i < quads; i += kRowThreads) *reinterpret_cast<f32x4_t*>(y + head + 4 * i) = f32x4_t{};
  if (t < a.V - head - 4 * quads) y[head + 4 * quads + t] = 0.f;
  int token;
  RowInfo mine;
  cut_row<HALF, true>(a, blockIdx.x, 0, -1, DrawIn{-1, -1, nullptr, 0.0}, sh, sh.few, mine, token);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // the zeros are there, every thread's
  __syncthreads();
  if (mine.z > 0 && t < sh.keep) y[(int)~(u32)sh.few.sorted[t]] = (float)(sh.few.w[t] * (1.0 / mine.z));
}

// The same by counts, for either launch behind this one: by a group of workgroups where the rows are few (gridDim.x).
template <bool HALF>
__global__ __launch_bounds__(kRowThreads) void sample_select_kernel(const SampleArgs a, const VerifyIn in, uint64_t* info,
                                                                   uint64_t* counts, int* arrived) {
  __shared__ RowShared sh;
  const int ri = blockIdx.y, seq = blockIdx.z, m = a.per - 1;
  const long row = (long)seq * a.per + ri;
  const int draft = in.draft && ri < m ? in.draft[(long)seq * m + ri] : -1;
  const Group gr = {gridDim.x > 1 ? counts + row * gridDim.x * (kGroupBins / 4) : nullptr, arrived + row, (int)blockIdx.x,
                    (int)gridDim.x};
  RowInfo mine;
  if (!select_row<HALF>(a, seq, ri, draft, gr, sh, mine)) return;
  write_info(info, row, mine);
  if (threadIdx.x == 0 && draft != -1) in.px[(long)seq * m + ri] = (float)mine.px;
  else if (threadIdx.x == 0 && in.draft && ri < m) in.px[(long)seq * m + ri] = 0.f;
}

struct SpreadShared {
  double z[kMaxDraft + 1];             // of the rows: RowInfo, without px
  float m[kMaxDraft + 1];
  int thr[kMaxDraft + 1], cut[kMaxDraft + 1], draft[kMaxDraft + 1];
  DrawShared draw;
  int last;
};

// Workgroups over the segments of a sequence. Each accepts (without a cut it joins the rows first); where r is not
// known from the segment sums (a cut, or draft probabilities and a refused draft), each sums r over its segments of
// the row to draw from, and the last draws.
template <bool HALF, bool CUT>
__global__ __launch_bounds__(kRowThreads) void sample_spread_kernel(const SampleArgs a, const VerifyIn in,
                                                                    const uint64_t* __restrict__ info, double* rest) {
  __shared__ SpreadShared sh;
  const int seq = blockIdx.y, m = a.per - 1, t = threadIdx.x, lane = t & 63;
  const int len = drafts_of(a, in, seq);
  const double u_last = uniform_at(in, (long)seq * a.per + m);
  // the last threads, a row each: what its draft is accepted by, on its way while the rows are joined
  const int i = kRowThreads - 1 - t;
  double px = 0, uq = 0;
  float xd = -INFINITY;
  RowInfo mine = {0.0, 0.0, 0.f, kLowKey<HALF>, kNoTies, 0};
  if (i < a.per) {
    const long row = (long)seq * a.per + i;
    if constexpr (CUT) __builtin_memcpy(&mine, info + 4 * row, 32);
    const int draft = i < m ? in.draft[(long)seq * m + i] : -1;
    const bool inside = draft >= 0 && draft < a.V;
    sh.draft[i] = draft;
    uq = inside ? uniform_at(in, row) * (in.q ? (double)in.q[seq * in.qb + i * in.qr + draft] : 1.0) : INFINITY;
    if (!CUT && inside) xd = val<HALF>(row_ptr(a, seq, i)[draft]);
  }
  if constexpr (!CUT) {
    for (int r = uniform(t >> 6); r < a.per; r += kRowWaves) {
      const long row = (long)seq * a.per + r;
      float mx;
      const double z = join_wave(a.segm + row * a.nseg, a.segs + row * a.nseg, a.nseg, a.c, mx);
      if (lane == 0) {
        sh.z[r] = z;
        sh.m[r] = mx;
      }
    }
  }
  if (t == 0) sh.draw.first = len;
  __syncthreads();
  if (i < a.per) {
    if constexpr (CUT) {
      px = mine.px;
      sh.z[i] = mine.z;
      sh.m[i] = mine.m;
    } else {
      px = sh.z[i] > 0 && xd > -INFINITY ? weight(xd, sh.m[i], a.c) / sh.z[i] : 0.0;
      if (blockIdx.x == 0 && i < m) in.px[(long)seq * m + i] = (float)px;
    }
    sh.thr[i] = mine.thr;
    sh.cut[i] = mine.cut;
    if (i < len && !(uq < px)) atomicMin(&sh.draw.first, i);
  }
  __syncthreads();
  const int n = sh.draw.first;
  DrawIn d;
  d.mode = n == len ? kDrawRow : in.q ? kDrawRest : kDrawOther;
  d.q = d.mode == kDrawRest ? in.q + seq * in.qb + n * in.qr : nullptr;
  d.skip = n < len ? sh.draft[n] : -1;
  d.u = u_last;
  const RowInfo r = {sh.z[n], 0.0, sh.m[n], sh.thr[n], sh.cut[n], 0};
  double* sums = rest + (long)seq * a.nseg;
  if (CUT || d.mode == kDrawRest) {
    const u16* x = row_ptr(a, seq, n);
    const int off = row_off(x);
    const double inv = r.z > 0 ? 1.0 / r.z : 0.0;
    const int stride = gridDim.x * kRowWaves, s0 = blockIdx.x * kRowWaves + uniform(t >> 6);
    constexpr int kOut = 2;             // segments of a wave whose loads are out together
    for (int s1 = s0; s1 < a.nseg; s1 += kOut * stride) {
      u32x4_t v[kOut];
      float q[kOut][8] = {};
      float sm[kOut];
      bool on[kOut];
#pragma unroll
      for (int i = 0; i < kOut; ++i) {
        const int s = s1 + i * stride, v0 = s * kSegVals + 8 * lane - off;
        on[i] = s < a.nseg && r.z > 0;
        if (!on[i]) continue;
        if constexpr (CUT) sm[i] = a.segm[((long)seq * a.per + n) * a.nseg + s];
        v[i] = load8<HALF>(x, v0, a.V);
        if (d.mode == kDrawRest) load_q8(d.q, v0, a.V, q[i]);
      }
#pragma unroll
      for (int i = 0; i < kOut; ++i) {
        const int s = s1 + i * stride;
        if (s >= a.nseg) break;
        double sum = 0;
        if (on[i] && (!CUT || key_of_float<HALF>(sm[i]) >= r.thr)) {
          double w[8];
          rest8<HALF, CUT>(a, r, inv, v[i], s * kSegVals + 8 * lane - off, d.mode, q[i], d.skip, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) sum += w[j];
          sum = wave_total(sum);
        }
        if (lane == 0) put_far(reinterpret_cast<uint64_t*>(sums) + s, __builtin_bit_cast(uint64_t, sum));
      }
    }
    if (!arrives_last(a.arrived + seq, gridDim.x, &sh.last)) return;
  } else if (blockIdx.x) {
    return;
  }
  const int token = draw_token<HALF, CUT>(a, r, seq, n, d, sums, sh.draw);
  write_tokens(a, in, seq, n, token);
}

// ---------------------------------------------------------------- probabilities

template <bool HALF, bool CUT, int SPW>
__global__ __launch_bounds__(kStatThreads) void sample_probs_kernel(const SampleArgs a, const uint64_t* __restrict__ info,
                                                                    float* __restrict__ out, long ldo) {
  const int lane = threadIdx.x & 63, row = blockIdx.y;
  const int s0 = (blockIdx.x * (kStatThreads / 64) + uniform(threadIdx.x >> 6)) * SPW;
  const u16* x = row_ptr(a, row, 0);
  const int off = row_off(x);
  u32x4_t v[SPW];
  float sm[SPW];
#pragma unroll
  for (int i = 0; i < SPW; ++i) {
    v[i] = load8<HALF>(x, (s0 + i) * kSegVals + 8 * lane - off, a.V);
    sm[i] = CUT && s0 + i < a.nseg ? a.segm[(long)row * a.nseg + s0 + i] : 0;
  }
  RowInfo r;
  if constexpr (CUT) {
    __builtin_memcpy(&r, info + 4 * (long)row, 32);
  } else {
    r.z = join_wave(a.segm + (long)row * a.nseg, a.segs + (long)row * a.nseg, a.nseg, a.c, r.m);
    r.thr = kLowKey<HALF>;
    r.cut = kNoTies;
  }
  const double inv = r.z > 0 ? 1.0 / r.z : 0.0;
  float* y = out + (long)row * ldo;
#pragma unroll
  for (int i = 0; i < SPW; ++i) {
    const int s = s0 + i;
    if (s >= a.nseg) return;
    const int v0 = s * kSegVals + 8 * lane - off;
    float p[8] = {};
    if (!CUT || key_of_float<HALF>(sm[i]) >= r.thr) {
      double w[8];
      const float q[8] = {};
      rest8<HALF, CUT>(a, r, inv, v[i], v0, kDrawRow, q, -1, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = (float)(w[j] * inv);
    }
    if (v0 >= 0 && v0 + 8 <= a.V && (reinterpret_cast<uintptr_t>(y + v0) & 15) == 0) {
      *reinterpret_cast<f32x4_t*>(y + v0) = f32x4_t{p[0], p[1], p[2], p[3]};
      *reinterpret_cast<f32x4_t*>(y + v0 + 4) = f32x4_t{p[4], p[5], p[6], p[7]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v0 + j >= 0 && v0 + j < a.V) y[v0 + j] = p[j];
    }
  }
}

// ---------------------------------------------------------------- host

// Workgroups that count a row together: a CU each, at least a segment a wave, at most kGroup; 0 for one a row.
constexpr int kGroupSegs = 65535 / kSegVals;          // counts of 16 bits
int group_size(int64_t rows, int nseg) {
  const int64_t g = rows < 256 ? 256 / rows : 1, most = (nseg + kRowWaves - 1) / kRowWaves;
  const int64_t n = g < most ? g : most;
  const int size = (int)(n < kGroup ? n : kGroup);
  return size < 2 || (nseg + size - 1) / size > kGroupSegs ? 0 : size;
}

struct Layout {
  size_t segs, rest, info, drawn, segm, arrived, counts, bytes;
};

Layout layout(int64_t rows, int64_t V, int64_t sequences) {
  const size_t n = (size_t)((V + 7 + kSegVals - 1) / kSegVals);
  const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  Layout l;
  l.segs = 0;
  l.rest = up(l.segs + (size_t)rows * n * 8);
  l.info = up(l.rest + (size_t)sequences * n * 8);
  l.drawn = up(l.info + (size_t)rows * sizeof(RowInfo));
  l.segm = up(l.drawn + (size_t)rows * 8);
  l.arrived = up(l.segm + (size_t)rows * n * 4);
  l.counts = up(l.arrived + (size_t)(sequences + rows) * 4);
  l.bytes = l.counts + (size_t)rows * group_size(rows, (int)n) * kGroupBins * 2;
  return l;
}

constexpr int64_t kMaxVocab = (int64_t)kMaxSegs * kSegVals - 8;

// Whether what is kept may well be more than can be sorted: what the mass alone cuts, a large top_k. Its counting and its
// draw are then worth more workgroups than one, and a launch each.
bool many(int top_k) { return !top_k || top_k > kListed / 2; }
int top_k_of(int64_t top_k, int64_t V) { return top_k < V ? (int)top_k : 0; }
// Bytes of a layout that a sampler uses: all of it where it counts.
size_t needed(const Layout& l, int top_k, double top_p) { return (top_k || top_p < 1.0) && many(top_k) ? l.bytes : l.counts; }

bool shape_ok(int64_t rows, int64_t V) { return rows >= 1 && rows <= 65535 && V >= 1 && V <= kMaxVocab; }

// Parts a segment that a top_k's bound goes by, 0 for whole segments. The k-th largest of n maxima is reached by
// n ln(n / (n - k)) logits or so; where that is near what can be sorted, and where there are fewer segments than k, the
// maxima of parts, at another pass over the row (24 rows of 70000, top 128: 24.4 us, 46.9 by whole segments).
int bound_parts(int nseg, int top_k) {
  if (!top_k) return 0;
  const int parts = nseg <= kMaxSegs / 8 ? 8 : nseg <= kMaxSegs / 4 ? 4 : 0;
  if (nseg < top_k) return parts * nseg >= top_k ? parts : 0;
  return top_k <= kListed / 2 && nseg * std::log(nseg / (nseg - top_k + 0.5)) > 0.7 * kListed ? parts : 0;
}

int sample_args(const char* what, int64_t dtype, const void* logits, int64_t rows, int64_t V, double temperature, int64_t top_k,
                double top_p, void* ws, int64_t ws_bytes, const Layout& l, SampleArgs& a) {
  if (!logits || !ws) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  if (dtype != DSPARK_DTYPE_BF16 && dtype != DSPARK_DTYPE_F16) return fail(DSPARK_ERR_UNSUPPORTED, "%s: dtype %lld (bf16 or fp16 logits)", what, (long long)dtype);
  if (!(temperature >= 1e-30 && temperature <= 1e30)) return fail(DSPARK_ERR_ARG, "%s: temperature %g (greedy: argmax_accept)", what, temperature);
  if (!(top_p > 0.0 && top_p <= 1.0) || top_k < 0) return fail(DSPARK_ERR_ARG, "%s: top_k %lld, top_p %g", what, (long long)top_k, top_p);
  if (!aligned(logits, 2) || !aligned(ws, 256)) return fail(DSPARK_ERR_ALIGN, "%s: logits need 2-byte, the workspace 256-byte alignment", what);
  const size_t need = needed(l, top_k_of(top_k, V), top_p);
  if (ws_bytes < (int64_t)need) return fail(DSPARK_ERR_WORKSPACE, "%s: workspace %lld < %zu bytes", what, (long long)ws_bytes, need);
  char* w = static_cast<char*>(ws);
  a.x = static_cast<const u16*>(logits);
  a.rows = (int)rows;
  a.V = (int)V;
  a.nseg = (int)((V + 7 + kSegVals - 1) / kSegVals);
  a.c = 1.4426950408889634 / temperature;
  a.top_p = top_p;
  a.top_k = top_k_of(top_k, V);
  a.parts = bound_parts(a.nseg, a.top_k);
  a.segm = reinterpret_cast<float*>(w + l.segm);
  a.segs = reinterpret_cast<double*>(w + l.segs);
  return DSPARK_OK;
}

// Segments from which the table pays: 8 rows of 151936 9.9 us without it, 10.8 with; 24 rows 15.3, 15.1; 55 rows 27.2, 24.6;
// 256 rows verified 53.0, 37.9.
constexpr long kTabSegs = 8192;

unsigned groups(int nseg, int spw) { return (unsigned)((nseg + spw * (kStatThreads / 64) - 1) / (spw * (kStatThreads / 64))); }

template <bool HALF>
void launch_segments(const SampleArgs& a, hipStream_t s) {
  const long total = (long)a.rows * a.nseg;
  if (!HALF && !a.top_k && !(a.top_p < 1.0) && a.c <= kTabMaxC && total >= kTabSegs && total < (1l << 30)) {
    const int waves = 256 * (kTabThreads / 64), steps = (int)((total + waves - 1) / waves);
    const unsigned blocks = (unsigned)((total + (long)steps * (kTabThreads / 64) - 1) / ((long)steps * (kTabThreads / 64)));
    hipLaunchKernelGGL(sample_table_kernel, dim3(blocks), dim3(kTabThreads), 0, s, a, (int)total, steps);
    return;
  }
  const dim3 grid(groups(a.nseg, kSegWave), (unsigned)a.per, (unsigned)(a.rows / a.per)), block(kStatThreads);
  if (a.top_k) hipLaunchKernelGGL((sample_segments_kernel<HALF, kSegWave, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((sample_segments_kernel<HALF, kSegWave, true>), grid, block, 0, s, a);
}

template <bool HALF>
void launch_select(const SampleArgs& a, const VerifyIn& in, char* w, const Layout& l, hipStream_t s) {
  const int group = group_size(a.rows, a.nseg);
  hipLaunchKernelGGL((sample_select_kernel<HALF>), dim3(group ? group : 1, (unsigned)a.per, (unsigned)(a.rows / a.per)),
                     dim3(kRowThreads), 0, s, a, in, reinterpret_cast<uint64_t*>(w + l.info),
                     reinterpret_cast<uint64_t*>(w + l.counts), a.arrived + a.rows / a.per);
}

template <bool HALF>
void probs(const SampleArgs& a, char* w, const Layout& l, float* out, long ldo, hipStream_t s) {
  const uint64_t* info = reinterpret_cast<uint64_t*>(w + l.info);
  const dim3 block(kStatThreads);
  const dim3 grid((unsigned)a.rows), row(kRowThreads);
  const bool cut = a.top_k || a.top_p < 1.0;
  if (cut && !many(a.top_k) && a.nseg <= kWholeSegs) {
    hipLaunchKernelGGL((sample_whole_kernel<HALF>), grid, row, 0, s, a, out, ldo);
    return;
  }
  launch_segments<HALF>(a, s);
  if (cut) {
    if (many(a.top_k)) launch_select<HALF>(a, VerifyIn{}, w, l, s);
    else hipLaunchKernelGGL((sample_few_kernel<HALF>), grid, row, 0, s, a, reinterpret_cast<uint64_t*>(w + l.info));
    hipLaunchKernelGGL((sample_probs_kernel<HALF, true, kProbCutWave>), dim3(groups(a.nseg, kProbCutWave), (unsigned)a.rows),
                       block, 0, s, a, info, out, ldo);
  } else {
    hipLaunchKernelGGL((sample_probs_kernel<HALF, false, kProbWave>), dim3(groups(a.nseg, kProbWave), (unsigned)a.rows), block,
                       0, s, a, info, out, ldo);
  }
}

template <bool HALF>
void verify(const SampleArgs& a, const VerifyIn& in, char* w, const Layout& l, hipStream_t s) {
  const unsigned B = (unsigned)(a.rows / a.per);
  uint64_t* info = reinterpret_cast<uint64_t*>(w + l.info);
  double* rest = reinterpret_cast<double*>(w + l.rest);
  const bool cut = a.top_k || a.top_p < 1.0;
  // over the rows that are drawn from, a workgroup a CU, at most one a wave and segment
  const unsigned most = (unsigned)((a.nseg + kRowWaves - 1) / kRowWaves), fill = B < 256 ? 256 / B : 1;
  const unsigned spread = most < fill ? most : fill;
  if (cut && !many(a.top_k) && a.per == 1 && a.nseg <= kWholeSegs) {
    hipLaunchKernelGGL((sample_cut_kernel<HALF, true>), dim3(1, B), dim3(kRowThreads), 0, s, a, in,
                       reinterpret_cast<uint64_t*>(w + l.drawn));
    return;
  }
  launch_segments<HALF>(a, s);
  if (cut && many(a.top_k)) {
    launch_select<HALF>(a, in, w, l, s);
    hipLaunchKernelGGL((sample_spread_kernel<HALF, true>), dim3(spread, B), dim3(kRowThreads), 0, s, a, in, info, rest);
  } else if (cut) {
    hipLaunchKernelGGL((sample_cut_kernel<HALF, false>), dim3((unsigned)a.per, B), dim3(kRowThreads), 0, s, a, in,
                       reinterpret_cast<uint64_t*>(w + l.drawn));
  } else {
    hipLaunchKernelGGL((sample_spread_kernel<HALF, false>), dim3(in.q ? spread : 1, B), dim3(kRowThreads), 0, s, a, in, info,
                       rest);
  }
}

}  // namespace
}  // namespace dspark

using namespace dspark;

extern "C" size_t dspark_sampling_workspace(int64_t rows, int64_t V, int64_t sequences) {
  if (!shape_ok(rows, V) || sequences < 0 || sequences > rows) return 0;
  return layout(rows, V, sequences ? sequences : rows).bytes;
}

extern "C" size_t dspark_sampling_workspace_for(int64_t rows, int64_t V, int64_t sequences, int64_t top_k, double top_p) {
  if (!shape_ok(rows, V) || sequences < 0 || sequences > rows) return 0;
  return needed(layout(rows, V, sequences ? sequences : rows), top_k_of(top_k, V), top_p);
}

extern "C" int dspark_sampling_probs(const dspark_sampling_probs_args* p, dspark_stream stream) {
  const char* what = "sampling_probs";
  if (!p || !p->out) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  if (!shape_ok(p->rows, p->V) || (p->rows > 1 && (p->ld < p->V || p->ldo < p->V)))
    return fail(DSPARK_ERR_SHAPE, "%s: rows=%lld V=%lld ld=%lld", what, (long long)p->rows, (long long)p->V, (long long)p->ld);
  if (!aligned(p->out, 4)) return fail(DSPARK_ERR_ALIGN, "%s: out needs 4-byte alignment", what);
  const Layout l = layout(p->rows, p->V, p->rows);
  SampleArgs a;
  const int st = sample_args(what, p->dtype, p->logits, p->rows, p->V, p->temperature, p->top_k, p->top_p, p->workspace,
                             p->workspace_bytes, l, a);
  if (st) return st;
  a.ldb = p->ld;
  a.ldr = 0;
  a.per = 1;
  char* w = static_cast<char*>(p->workspace);
  a.arrived = reinterpret_cast<int*>(w + l.arrived);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == DSPARK_DTYPE_F16) probs<true>(a, w, l, p->out, p->ldo, s);
  else probs<false>(a, w, l, p->out, p->ldo, s);
  return check_launch(what);
}

extern "C" int dspark_speculative_verify(const dspark_speculative_verify_args* p, dspark_stream stream) {
  const char* what = "speculative_verify";
  if (!p || !p->uniforms || !p->n_accepted || !p->tokens || (p->drafts > 0 && (!p->draft || !p->draft_p)))
    return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  if (p->sequences < 1 || p->sequences > 65535 || p->drafts < 0 || p->drafts > kMaxDraft ||
      !shape_ok(p->sequences * (p->drafts + 1), p->V))
    return fail(DSPARK_ERR_SHAPE, "%s: sequences=%lld drafts=%lld V=%lld", what, (long long)p->sequences,
                (long long)p->drafts, (long long)p->V);
  if (p->ld_seq < 0 || p->ld_row < 0 || (p->draft_probs && (p->q_seq < 0 || p->q_row < 0)))
    return fail(DSPARK_ERR_SHAPE, "%s: negative strides", what);
  if (!aligned(p->uniforms, p->uniforms_f64 ? 8 : 4) || !aligned(p->draft, 4) || !aligned(p->draft_probs, 4) ||
      !aligned(p->draft_lens, 4) || !aligned(p->n_accepted, 4) || !aligned(p->tokens, 4) || !aligned(p->draft_p, 4))
    return fail(DSPARK_ERR_ALIGN, "%s: arrays need the alignment of their type", what);
  const int64_t rows = p->sequences * (p->drafts + 1);
  const Layout l = layout(rows, p->V, p->sequences);
  SampleArgs a;
  const int st = sample_args(what, p->dtype, p->logits, rows, p->V, p->temperature, p->top_k, p->top_p, p->workspace,
                             p->workspace_bytes, l, a);
  if (st) return st;
  a.ldb = p->ld_seq;
  a.ldr = p->ld_row;
  a.per = (int)p->drafts + 1;
  VerifyIn in;
  in.draft = p->draft;
  in.q = p->drafts > 0 ? p->draft_probs : nullptr;
  in.qb = p->q_seq;
  in.qr = p->q_row;
  in.lens = p->draft_lens;
  in.u = p->uniforms;
  in.u64 = p->uniforms_f64 != 0;
  in.n = p->n_accepted;
  in.tokens = p->tokens;
  in.px = p->draft_p;
  char* w = static_cast<char*>(p->workspace);
  a.arrived = reinterpret_cast<int*>(w + l.arrived);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == DSPARK_DTYPE_F16) verify<true>(a, in, w, l, s);
  else verify<false>(a, in, w, l, s);
  return check_launch(what);
}
