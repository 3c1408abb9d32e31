// The kernels and entry points of dspark_sampling.h: the truncated softmax of a row
// (dspark_sampling_probs) and the accept rule of a sampled round (dspark_speculative_verify).
#include "dspark_sampling.h"

namespace dspark {
namespace {

// ---------------------------------------------------------------- segments of every row

constexpr int kStatThreads = 256;

// Maximum and sum of weights of every segment: a wave takes SPW segments, their loads first.
template <bool HALF, int SPW, bool SUM>
__global__ __launch_bounds__(kStatThreads) void sample_segments_kernel(const SampleArgs a) {
  const int lane = threadIdx.x & 63, row = blockIdx.y;
  const int s0 = (blockIdx.x * (kStatThreads / 64) + uniform(threadIdx.x >> 6)) * SPW;
  const u16* x = row_ptr(a, row);
  const int off = row_off(x);
  u32x4_t v[SPW];
#pragma unroll
  for (int i = 0; i < SPW; ++i) v[i] = load8<HALF>(x, (s0 + i) * kSegVals + 8 * lane - off, a.V);
#pragma unroll
  for (int i = 0; i < SPW; ++i) {
    if (s0 + i >= a.nseg) return;
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, val<HALF>(bits_of(v[i], j)));
    m = wave_max(m);
    const long at = (long)row * a.nseg + s0 + i;
    if constexpr (SUM) {
      double s = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += weight(val<HALF>(bits_of(v[i], j)), m, a.c);
      s = wave_total(s);
      if (lane == 0) a.segs[at] = m > -INFINITY ? s : 0.0;
    }
    if (lane == 0) a.segm[at] = m;
  }
}

// ---------------------------------------------------------------- what is kept of a row

struct RowShared {
  int bins[kBins];
  int skey[kMaxSegs];                  // key of each segment's maximum
  int list[kMaxSegs];                  // the segments that may hold a kept token, in order
  int cnt[kMaxSegs];
  double red_d[kRowThreads / 64];
  float red_f[kRowThreads / 64];
  int red_i[kRowThreads / 64];
  int owner, key, keep, ties, kb, cut;
  double z, mass;
};

// Counts the logits of the listed segments by key, bin hi - key for lo <= key <= hi.
template <bool HALF>
__device__ __forceinline__ void count_keys(const SampleArgs& a, const u16* x, int off, RowShared& sh, int nlist, int hi,
                                           int lo) {
  for (int i = threadIdx.x; i <= hi - lo; i += kRowThreads) sh.bins[i] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  constexpr int kWaves = kRowThreads / 64, kAhead = 4;    // segments of a wave whose loads are out together
  for (int i0 = uniform(threadIdx.x >> 6); i0 < nlist; i0 += kAhead * kWaves) {
    u32x4_t v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * kWaves;
      if (i < nlist) v[u] = load8<HALF>(x, sh.list[i] * kSegVals + 8 * lane - off, a.V);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i0 + u * kWaves >= nlist) break;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = key_of<HALF>(bits_of(v[u], j));
        if (k >= lo && k <= hi) atomicAdd(&sh.bins[hi - k], 1);
      }
    }
  }
  __syncthreads();
}

// The part of one row that is sampled from: its threshold and normaliser (RowInfo without px).
template <bool HALF>
__device__ __forceinline__ RowInfo select_row(const SampleArgs& a, int row, RowShared& sh) {
  const int t = threadIdx.x;
  const u16* x = row_ptr(a, row);
  const int off = row_off(x);
  const float* segm = a.segm + (long)row * a.nseg;
  RowInfo out;
  double total = 0;                     // of the whole row; needed where the mass itself is cut
  if (a.top_k) {
    float mx = -INFINITY;
    for (int s = t; s < a.nseg; s += kRowThreads) mx = fmaxf(mx, segm[s]);
    mx = wave_max(mx);
    if ((t & 63) == 0) sh.red_f[t >> 6] = mx;
    __syncthreads();
    for (int i = 0; i < kRowThreads / 64; ++i) mx = fmaxf(mx, sh.red_f[i]);
    out.m = mx;
  } else {
    total = join_segments(segm, a.segs + (long)row * a.nseg, a.nseg, a.c, sh.red_f, sh.red_d, out.m);
  }
  out.px = 0;
  out.pad = 0;
  if (!(out.m > -INFINITY)) {           // nothing to draw from
    out.z = 0;
    out.thr = 1 << 16;
    out.cut = kNoTies;
    return out;
  }
  const int top = key_of_float<HALF>(out.m);
  for (int s = t; s < a.nseg; s += kRowThreads) sh.skey[s] = key_of_float<HALF>(segm[s]);
  __syncthreads();

  // a key that every kept token reaches
  if (t < 64) {
    int kb = kLowKey<HALF> + 1;
    if (a.top_k) {
      if (a.nseg >= a.top_k) {          // the top_k-th largest segment maximum, bit by bit
        int k = 0;
        for (int bit = 15; bit >= 0; --bit) {
          const int tryk = k | (1 << bit);
          int n = 0;
          for (int s = t; s < kMaxSegs && s - t < a.nseg; s += 64)
            n += __popcll(__ballot(s < a.nseg && sh.skey[s < a.nseg ? s : 0] >= tryk));
          if (n >= a.top_k) k = tryk;
        }
        kb = max(kb, k);
      }
    } else {
      // tokens of weight (1 - top_p) S / V or less: all together less than (1 - top_p) S. One key of room
      // for the rounding to 16 bits.
      const double w = (1.0 - a.top_p) * total / (double)a.V;
      kb = max(kb, key_of_float<HALF>((float)((double)out.m + log2(w) / a.c)) - 1);
    }
    if (t == 0) sh.kb = min(kb, top);
  }
  __syncthreads();
  const int kb = sh.kb;
  int nlist;
  {
    const int s0 = 2 * t;
    const int f0 = s0 < a.nseg && sh.skey[s0] >= kb, f1 = s0 + 1 < a.nseg && sh.skey[s0 + 1] >= kb;
    const int end = block_scan(f0 + f1, sh.red_i, nlist);
    if (f0) sh.list[end - f0 - f1] = s0;
    if (f1) sh.list[end - f1] = s0 + 1;
  }
  __syncthreads();

  int thr = kb - 1, keep = 0, ties = 0;  // thr = kb - 1: every listed token
  int loaded = 1 << 17;                  // the range of keys now in the bins starts here
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
    for (int hi = top; hi >= lowest && !found; hi -= kBins) {
      const int lo = max(lowest, hi - kBins + 1);
      if (!(hi == top && loaded <= lo && top - loaded < kBins)) {
        count_keys<HALF>(a, x, off, sh, nlist, hi, lo);
        loaded = hi == top ? lo : 1 << 17;
      }
      const int nb = hi - lo + 1, each = (nb + kRowThreads - 1) / kRowThreads;
      const int b0 = min(t * each, nb), b1 = min(b0 + each, nb);
      int cn = 0;
      double cm = 0;
      for (int b = b0; b < b1; ++b) {
        int n = sh.bins[b];
        if (!n) continue;
        if (after_k && hi - b == thr_k) n = keep_k;
        cn += n;
        cm += (double)n * weight(val_of_key<HALF>(hi - b), out.m, a.c);
      }
      if (t == 0) sh.owner = kRowThreads;
      int cnt_all;
      double mass_all;
      const int cnt_end = block_scan(cn, sh.red_i, cnt_all);
      const double mass_end = block_scan(cm, sh.red_d, mass_all);
      // the thread whose bins the goal falls into (the first: running sums may step back by a rounding)
      const bool mine = pass == 0 ? seen + cnt_end >= a.top_k && cn : mass + mass_end >= goal && cn;
      if (mine) atomicMin(&sh.owner, t);
      __syncthreads();
      if (sh.owner == t) {
        int run = seen + cnt_end - cn, r = 0;
        double m0 = mass + (mass_end - cm);
        bool hit = false;
        for (int b = b0; b < b1 && !hit; ++b) {
          int n = sh.bins[b];
          if (!n) continue;
          const int all = n;
          if (after_k && hi - b == thr_k) n = keep_k;
          const double w = weight(val_of_key<HALF>(hi - b), out.m, a.c);
          if (pass == 0) {
            hit = run + n >= a.top_k;
            r = hit ? a.top_k - run : n;
          } else {
            hit = m0 + (double)n * w >= goal;
            r = n;
            if (hit) {                  // tokens of this value before which less than the goal lies
              r = (int)fmin(fmax(__builtin_ceil((goal - m0) / w), 1.0), (double)n);
              while (r > 1 && m0 + (double)(r - 1) * w >= goal) --r;
              while (r < n && m0 + (double)r * w < goal) ++r;
            }
          }
          run += n;
          m0 += (double)r * w;
          sh.key = hi - b;
          sh.keep = r;
          sh.ties = all;
          sh.z = m0;
        }
      }
      __syncthreads();
      seen += cnt_all;
      mass += mass_all;
      found = sh.owner < kRowThreads;
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
  out.cut = ties ? a.V : kNoTies;            // without a threshold value (thr = kb - 1) no token has that key
  if (keep < ties) {                    // the index of the last kept token of the threshold's value
    const int lane = t & 63;
    for (int i = uniform(t >> 6); i < nlist; i += kRowThreads / 64) {
      const int s = sh.list[i];
      int n = 0;
      if (sh.skey[s] >= thr) {
        const u32x4_t v = load8<HALF>(x, s * kSegVals + 8 * lane - off, a.V);
#pragma unroll
        for (int j = 0; j < 8; ++j) n += __popcll(__ballot(key_of<HALF>(bits_of(v, j)) == thr));
      }
      if (lane == 0) sh.cnt[i] = n;
    }
    __syncthreads();
    const int i0 = 2 * t;
    const int c0 = i0 < nlist ? sh.cnt[i0] : 0, c1 = i0 + 1 < nlist ? sh.cnt[i0 + 1] : 0;
    int all;
    const int end = block_scan(c0 + c1, sh.red_i, all);
    const int before = end - c0 - c1;
    if (before < keep && keep <= end) {
      const bool second = keep > before + c0;
      sh.owner = sh.list[second ? i0 + 1 : i0];
      sh.keep = keep - before - (second ? c0 : 0);
    }
    __syncthreads();
    if (t < 64) {
      const int v0 = sh.owner * kSegVals + 8 * lane - off, want = sh.keep;
      const u32x4_t v = load8<HALF>(x, v0, a.V);
      int n = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) n += key_of<HALF>(bits_of(v, j)) == thr;
      int run = wave_scan(n) - n;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (key_of<HALF>(bits_of(v, j)) == thr && ++run == want) sh.cut = v0 + j;
    }
    __syncthreads();
    out.cut = sh.cut;
  }
  return out;
}

// p of one token
template <bool HALF>
__device__ __forceinline__ double prob_of(const SampleArgs& a, const RowInfo& r, int row, int v) {
  if (v < 0 || v >= a.V || !(r.z > 0)) return 0;
  const u32 b = row_ptr(a, row)[v];
  const int k = key_of<HALF>(b);
  if (k < r.thr || (k == r.thr && v > r.cut)) return 0;
  return weight(val<HALF>(b), r.m, a.c) / r.z;
}

// One row a workgroup: its threshold (CUT) or its normaliser, and the drafted token's probability.
template <bool HALF, bool CUT>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(const SampleArgs a, RowInfo* __restrict__ info,
                                                                 const int32_t* __restrict__ draft, float* __restrict__ px) {
  const int row = blockIdx.x;
  RowInfo r;
  if constexpr (CUT) {
    __shared__ RowShared sh;
    r = select_row<HALF>(a, row, sh);
  } else {
    __shared__ float red_f[kRowThreads / 64];
    __shared__ double red_d[kRowThreads / 64];
    r.z = join_segments(a.segm + (long)row * a.nseg, a.segs + (long)row * a.nseg, a.nseg, a.c, red_f, red_d, r.m);
    r.thr = kLowKey<HALF>;
    r.cut = kNoTies;
    r.pad = 0;
  }
  if (threadIdx.x == 0) {
    r.px = 0;
    const int i = row % a.per, b = row / a.per;
    if (draft && i < a.per - 1) {
      const long at = (long)b * (a.per - 1) + i;
      r.px = prob_of<HALF>(a, r, row, draft[at]);
      px[at] = (float)r.px;
    }
    info[row] = r;
  }
}

// ---------------------------------------------------------------- the accept rule

// The first refused draft of sequence b (its number of drafts if none is); `first` in LDS.
__device__ __forceinline__ int first_refused(const SampleArgs& a, const VerifyIn& in, const RowInfo* info, int b, int* first,
                                             int& len) {
  const int m = a.per - 1;
  len = in.lens ? min(max(in.lens[b], 0), m) : m;
  if (threadIdx.x == 0) *first = len;
  __syncthreads();
  for (int i = threadIdx.x; i < len; i += blockDim.x) {
    const int v = in.draft[(long)b * m + i];
    const long at = (long)b * a.per + i;
    const double u = in.u64 ? static_cast<const double*>(in.u)[at] : (double)static_cast<const float*>(in.u)[at];
    const bool inside = v >= 0 && v < a.V;
    const double q = in.q ? (inside ? (double)in.q[(long)b * in.qb + (long)i * in.qr + v] : 0.0) : 1.0;
    if (!(inside && u * q < info[at].px)) atomicMin(first, i);
  }
  __syncthreads();
  return *first;
}

enum { kDrawRow = 0, kDrawRest = 1, kDrawOther = 2 };   // r = p, max(p - q, 0), p without one token

// r of 8 logits from index v0 (logits outside the row are -inf, their weight 0 and their q not read)
template <bool HALF>
__device__ __forceinline__ void rest8(const SampleArgs& a, const RowInfo& r, const u32x4_t& x, int v0, int mode,
                                      const float* q, int skip, double (&out)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const u32 b = bits_of(x, j);
    const int k = key_of<HALF>(b), v = v0 + j;
    double w = 0;
    if (k > r.thr || (k == r.thr && v <= r.cut)) {
      w = weight(val<HALF>(b), r.m, a.c);
      if (mode == kDrawRest) w = __builtin_fmax(w / r.z - ((v >= 0 && v < a.V) ? (double)q[v] : 0.0), 0.0);
      else if (mode == kDrawOther && v == skip) w = 0;
    }
    out[j] = w;
  }
}

// Segment sums of max(p - q, 0) of each sequence's refused row, nothing cut: over the whole chip.
template <bool HALF, int SPW>
__global__ __launch_bounds__(kStatThreads) void sample_rest_kernel(const SampleArgs a, const VerifyIn in,
                                                                   const RowInfo* __restrict__ info, double* __restrict__ rest) {
  __shared__ int first;
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  int len;
  const int n = first_refused(a, in, info, b, &first, len);
  if (n >= len) return;
  const int row = b * a.per + n;
  const RowInfo r = info[row];
  const u16* x = row_ptr(a, row);
  const float* q = in.q + (long)b * in.qb + (long)n * in.qr;
  const int off = row_off(x);
  const int s0 = (blockIdx.x * (kStatThreads / 64) + uniform(threadIdx.x >> 6)) * SPW;
#pragma unroll
  for (int i = 0; i < SPW; ++i) {
    const int s = s0 + i;
    if (s >= a.nseg) return;
    const int v0 = s * kSegVals + 8 * lane - off;
    double w[8];
    rest8<HALF>(a, r, load8<HALF>(x, v0, a.V), v0, kDrawRest, q, -1, w);
    double t = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) t += w[j];
    t = wave_total(t);
    if (lane == 0) rest[(long)b * a.nseg + s] = t;
  }
}

// The accepted drafts of one sequence and the token after them.
template <bool HALF, bool CUT>
__global__ __launch_bounds__(kRowThreads) void sample_draw_kernel(const SampleArgs a, const VerifyIn in,
                                                                  const RowInfo* __restrict__ info,
                                                                  const double* __restrict__ rest) {
  __shared__ double sums[kMaxSegs];
  __shared__ int skey[kMaxSegs];
  __shared__ double red[kRowThreads / 64];
  __shared__ double before_s;
  __shared__ int first, seg, last, token;
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, m = a.per - 1;
  int len;
  const int n = first_refused(a, in, info, b, &first, len);
  const int row = b * a.per + n;
  const RowInfo r = info[row];
  const u16* x = row_ptr(a, row);
  const int off = row_off(x);
  const float* segm = a.segm + (long)row * a.nseg;
  const float* q = in.q && n < len ? in.q + (long)b * in.qb + (long)n * in.qr : nullptr;
  const int skip = n < len ? in.draft[(long)b * m + n] : -1;
  const long at = (long)b * a.per + m;
  const double u = in.u64 ? static_cast<const double*>(in.u)[at] : (double)static_cast<const float*>(in.u)[at];
  int mode = n == len ? kDrawRow : q ? kDrawRest : kDrawOther;
  if (t == 0) token = 0;
  if constexpr (CUT) {
    for (int s = t; s < a.nseg; s += kRowThreads) skey[s] = key_of_float<HALF>(segm[s]);
    __syncthreads();
  }

  // sums of r over the segments; where r is zero throughout, of p
  double all = 0, end = 0, s0 = 0, s1 = 0;
  for (int tries = 0; tries < 2; ++tries) {
    if constexpr (CUT) {
      constexpr int kWaves = kRowThreads / 64, kAhead = 4;
      for (int i0 = uniform(t >> 6); i0 < a.nseg; i0 += kAhead * kWaves) {
        u32x4_t v[kAhead];
        bool on[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int s = i0 + k * kWaves;
          on[k] = s < a.nseg && r.z > 0 && skey[s] >= r.thr;
          if (on[k]) v[k] = load8<HALF>(x, s * kSegVals + 8 * lane - off, a.V);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int s = i0 + k * kWaves;
          if (s >= a.nseg) break;
          double w[8], sum = 0;
          if (on[k]) {
            rest8<HALF>(a, r, v[k], s * kSegVals + 8 * lane - off, mode, q, skip, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += w[j];
            sum = wave_total(sum);
          }
          if (lane == 0) sums[s] = sum;
        }
      }
    } else {
      for (int s = t; s < a.nseg; s += kRowThreads)
        sums[s] = mode == kDrawRest ? rest[(long)b * a.nseg + s]
                                    : a.segs[(long)row * a.nseg + s] * weight(segm[s], r.m, a.c);
      __syncthreads();
      if (mode == kDrawOther && skip >= 0 && skip < a.V && t < 64) {   // the token's own segment again, without it
        const int s = (skip + off) / kSegVals, v0 = s * kSegVals + 8 * lane - off;
        double w[8], sum = 0;
        rest8<HALF>(a, r, load8<HALF>(x, v0, a.V), v0, mode, nullptr, skip, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += w[j];
        sum = wave_total(sum);
        if (lane == 0) sums[s] = sum;
      }
    }
    __syncthreads();
    s0 = 2 * t < a.nseg ? sums[2 * t] : 0;
    s1 = 2 * t + 1 < a.nseg ? sums[2 * t + 1] : 0;
    end = block_scan(s0 + s1, red, all);
    if (all > 0 || mode == kDrawRow) break;
    mode = kDrawRow;
  }
  // the first segment whose running sum passes the goal (the last one with any mass if none does by a rounding)
  const double goal = u * all;
  if (t == 0) {
    seg = kMaxSegs;
    last = -1;
  }
  __syncthreads();
  const double b0 = end - (s0 + s1), b1 = b0 + s0;
  if (s0 > 0 && b1 > goal) atomicMin(&seg, 2 * t);
  else if (s1 > 0 && end > goal) atomicMin(&seg, 2 * t + 1);
  if (s1 > 0) atomicMax(&last, 2 * t + 1);
  else if (s0 > 0) atomicMax(&last, 2 * t);
  __syncthreads();
  const int s = seg < kMaxSegs ? seg : last;
  if (s >= 0) {
    if (t == s >> 1) before_s = (s & 1) ? b1 : b0;
    __syncthreads();
    if (t < 64) {
      const int v0 = s * kSegVals + 8 * lane - off;
      double w[8], sum = 0;
      rest8<HALF>(a, r, load8<HALF>(x, v0, a.V), v0, mode, q, skip, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += w[j];
      const double to = before_s + wave_scan(sum);
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
        token = pick;
      }
    }
  }
  __syncthreads();
  for (int i = t; i < a.per; i += kRowThreads)
    in.tokens[(long)b * a.per + i] = i < n ? in.draft[(long)b * m + i] : i == n ? token : -1;
  if (t == 0) in.n[b] = n;
}

// ---------------------------------------------------------------- probabilities

template <bool HALF, bool CUT, int SPW>
__global__ __launch_bounds__(kStatThreads) void sample_probs_kernel(const SampleArgs a, const RowInfo* __restrict__ info,
                                                                    float* __restrict__ out, long ldo) {
  const int lane = threadIdx.x & 63, row = blockIdx.y;
  const int s0 = (blockIdx.x * (kStatThreads / 64) + uniform(threadIdx.x >> 6)) * SPW;
  const u16* x = row_ptr(a, row);
  const int off = row_off(x);
  const RowInfo r = info[row];
  const double inv = r.z > 0 ? 1.0 / r.z : 0.0;
  float* y = out + (long)row * ldo;
#pragma unroll
  for (int i = 0; i < SPW; ++i) {
    const int s = s0 + i;
    if (s >= a.nseg) return;
    const int v0 = s * kSegVals + 8 * lane - off;
    float p[8] = {};
    if (!CUT || key_of_float<HALF>(a.segm[(long)row * a.nseg + s]) >= r.thr) {
      const u32x4_t v = load8<HALF>(x, v0, a.V);
      double w[8];
      rest8<HALF>(a, r, v, v0, kDrawRow, nullptr, -1, w);
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

struct Layout {
  size_t segm, segs, info, rest, bytes;
};

Layout layout(int64_t rows, int64_t V, int64_t sequences) {
  const size_t n = (size_t)((V + 7 + kSegVals - 1) / kSegVals);
  const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  Layout l;
  l.segs = 0;
  l.rest = up(l.segs + (size_t)rows * n * 8);
  l.info = up(l.rest + (size_t)sequences * n * 8);
  l.segm = up(l.info + (size_t)rows * sizeof(RowInfo));
  l.bytes = up(l.segm + (size_t)rows * n * 4);
  return l;
}

constexpr int64_t kMaxVocab = (int64_t)kMaxSegs * kSegVals - 8;

bool shape_ok(int64_t rows, int64_t V) { return rows >= 1 && rows <= 65535 && V >= 1 && V <= kMaxVocab; }

int sample_args(const char* what, int64_t dtype, const void* logits, int64_t rows, int64_t V, double temperature, int64_t top_k,
                double top_p, void* ws, int64_t ws_bytes, const Layout& l, SampleArgs& a) {
  if (!logits || !ws) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  if (dtype != DSPARK_DTYPE_BF16 && dtype != DSPARK_DTYPE_F16) return fail(DSPARK_ERR_UNSUPPORTED, "%s: dtype %lld (bf16 or fp16 logits)", what, (long long)dtype);
  if (!(temperature >= 1e-30 && temperature <= 1e30)) return fail(DSPARK_ERR_ARG, "%s: temperature %g (greedy: argmax_accept)", what, temperature);
  if (!(top_p > 0.0 && top_p <= 1.0) || top_k < 0) return fail(DSPARK_ERR_ARG, "%s: top_k %lld, top_p %g", what, (long long)top_k, top_p);
  if (!aligned(logits, 2) || !aligned(ws, 256)) return fail(DSPARK_ERR_ALIGN, "%s: logits need 2-byte, the workspace 256-byte alignment", what);
  if (ws_bytes < (int64_t)l.bytes) return fail(DSPARK_ERR_WORKSPACE, "%s: workspace %lld < %zu bytes", what, (long long)ws_bytes, l.bytes);
  char* w = static_cast<char*>(ws);
  a.x = static_cast<const u16*>(logits);
  a.rows = (int)rows;
  a.V = (int)V;
  a.nseg = (int)((V + 7 + kSegVals - 1) / kSegVals);
  a.c = 1.4426950408889634 / temperature;
  a.top_p = top_p;
  a.top_k = top_k < V ? (int)top_k : 0;
  a.segm = reinterpret_cast<float*>(w + l.segm);
  a.segs = reinterpret_cast<double*>(w + l.segs);
  return DSPARK_OK;
}

unsigned groups(int nseg, int spw) { return (unsigned)((nseg + spw * (kStatThreads / 64) - 1) / (spw * (kStatThreads / 64))); }

template <bool HALF>
void launch_segments(const SampleArgs& a, hipStream_t s) {
  const dim3 grid(groups(a.nseg, 4), (unsigned)a.rows), block(kStatThreads);
  if (a.top_k) hipLaunchKernelGGL((sample_segments_kernel<HALF, 4, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((sample_segments_kernel<HALF, 4, true>), grid, block, 0, s, a);
}

template <bool HALF, bool CUT>
void launch_rows(const SampleArgs& a, RowInfo* info, const int32_t* draft, float* px, hipStream_t s) {
  hipLaunchKernelGGL((sample_row_kernel<HALF, CUT>), dim3((unsigned)a.rows), dim3(kRowThreads), 0, s, a, info, draft, px);
}

template <bool HALF, bool CUT>
void probs(const SampleArgs& a, RowInfo* info, float* out, long ldo, hipStream_t s) {
  launch_segments<HALF>(a, s);
  launch_rows<HALF, CUT>(a, info, nullptr, nullptr, s);
  hipLaunchKernelGGL((sample_probs_kernel<HALF, CUT, 4>), dim3(groups(a.nseg, 4), (unsigned)a.rows), dim3(kStatThreads), 0, s,
                     a, info, out, ldo);
}

template <bool HALF, bool CUT>
void verify(const SampleArgs& a, const VerifyIn& in, RowInfo* info, double* rest, hipStream_t s) {
  const unsigned B = (unsigned)(a.rows / a.per);
  launch_segments<HALF>(a, s);
  launch_rows<HALF, CUT>(a, info, in.draft, in.px, s);
  if (!CUT && in.q)
    hipLaunchKernelGGL((sample_rest_kernel<HALF, 4>), dim3(groups(a.nseg, 4), B), dim3(kStatThreads), 0, s, a, in, info, rest);
  hipLaunchKernelGGL((sample_draw_kernel<HALF, CUT>), dim3(B), dim3(kRowThreads), 0, s, a, in, info, rest);
}

}  // namespace
}  // namespace dspark

using namespace dspark;

extern "C" size_t dspark_sampling_workspace(int64_t rows, int64_t V, int64_t sequences) {
  if (!shape_ok(rows, V) || sequences < 0 || sequences > rows) return 0;
  return layout(rows, V, sequences).bytes;
}

extern "C" int dspark_sampling_probs(const dspark_sampling_probs_args* p, dspark_stream stream) {
  const char* what = "sampling_probs";
  if (!p || !p->out) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  if (!shape_ok(p->rows, p->V) || (p->rows > 1 && (p->ld < p->V || p->ldo < p->V)))
    return fail(DSPARK_ERR_SHAPE, "%s: rows=%lld V=%lld ld=%lld", what, (long long)p->rows, (long long)p->V, (long long)p->ld);
  if (!aligned(p->out, 4)) return fail(DSPARK_ERR_ALIGN, "%s: out needs 4-byte alignment", what);
  const Layout l = layout(p->rows, p->V, 0);
  SampleArgs a;
  const int st = sample_args(what, p->dtype, p->logits, p->rows, p->V, p->temperature, p->top_k, p->top_p, p->workspace,
                             p->workspace_bytes, l, a);
  if (st) return st;
  a.ldb = p->ld;
  a.ldr = 0;
  a.per = 1;
  RowInfo* info = reinterpret_cast<RowInfo*>(static_cast<char*>(p->workspace) + l.info);
  const bool cut = a.top_k || a.top_p < 1.0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == DSPARK_DTYPE_F16) cut ? probs<true, true>(a, info, p->out, p->ldo, s) : probs<true, false>(a, info, p->out, p->ldo, s);
  else cut ? probs<false, true>(a, info, p->out, p->ldo, s) : probs<false, false>(a, info, p->out, p->ldo, s);
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
  if (!aligned(p->uniforms, p->uniforms_f64 ? 8 : 4)) return fail(DSPARK_ERR_ALIGN, "%s: uniforms alignment", what);
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
  RowInfo* info = reinterpret_cast<RowInfo*>(w + l.info);
  double* rest = reinterpret_cast<double*>(w + l.rest);
  const bool cut = a.top_k || a.top_p < 1.0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == DSPARK_DTYPE_F16) cut ? verify<true, true>(a, in, info, rest, s) : verify<true, false>(a, in, info, rest, s);
  else cut ? verify<false, true>(a, in, info, rest, s) : verify<false, false>(a, in, info, rest, s);
  return check_launch(what);
}
