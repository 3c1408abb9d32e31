// The kernels and entry points of dspark_sampling.h: the truncated softmax of a row
// (dspark_sampling_probs) and the accept rule of a sampled round (dspark_speculative_verify).
//
// A call is two launches (probabilities: three where something is cut). The first leaves every segment's
// maximum and sum; in the second, with a cut, a workgroup a row finds what is kept of it, and the last one of
// a sequence to arrive accepts and draws; without a cut, workgroups over a sequence's segments join its rows,
// accept, sum max(p - q, 0) over their own segments of the refused row, and the last one draws.
#include "dspark_sampling.h"

namespace dspark {
namespace {

// ---------------------------------------------------------------- segments of every row

constexpr int kStatThreads = 256;

// Maximum and sum of weights of every segment: a wave takes SPW segments, their loads first.
template <bool HALF, int SPW, bool SUM>
__global__ __launch_bounds__(kStatThreads) void sample_segments_kernel(const SampleArgs a) {
  const int lane = threadIdx.x & 63, seq = blockIdx.z;
  if (a.arrived && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.arrived[seq] = 0;
  const int s0 = (blockIdx.x * (kStatThreads / 64) + uniform(threadIdx.x >> 6)) * SPW;
  const u16* x = row_ptr(a, seq, blockIdx.y);
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

// ---------------------------------------------------------------- what is kept of a row

constexpr int kAhead = 4;              // segments of a wave whose loads are out together

struct RowShared {
  union {
    int bins[kBins];
    struct {
      uint64_t cand[kListed];          // key << 32 | ~index: the larger the earlier in falling order
      uint64_t sorted[kListed];
    };
  };
  int skey[kMaxSegs];                  // key of each segment's maximum
  int list[kMaxSegs];                  // the segments that may hold a kept token, in order
  int cnt[kMaxSegs];
  double red_d[kRowWaves];
  float red_f[kRowWaves];
  int red_i[kRowWaves];
  int owner, key, keep, ties, kb, cut, ncand, last;
  double z, px;
};

// The largest key that at least k of the n (<= kMaxSegs) values reach, bit by bit: one wave, 16 values a lane.
__device__ __forceinline__ int kth_key(const int* v, int n, int k) {
  const int lane = threadIdx.x & 63;
  int mine[kMaxSegs / 64];
#pragma unroll
  for (int i = 0; i < kMaxSegs / 64; ++i) mine[i] = 64 * i + lane < n ? v[64 * i + lane] : -1;
  int key = 0;
  for (int bit = 1 << 15; bit; bit >>= 1) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kMaxSegs / 64; ++i)
      if (64 * i < n) c += __popcll(__ballot(mine[i] >= (key | bit)));
    if (c >= k) key |= bit;
  }
  return key;
}

// Calls f(segment's place in the list, its 8 logits of this lane) for every listed segment, a wave at a time.
template <bool HALF, typename F>
__device__ __forceinline__ void each_listed(const SampleArgs& a, const u16* x, int off, const int* list, int nlist, F&& f) {
  const int lane = threadIdx.x & 63;
  for (int i0 = uniform(threadIdx.x >> 6); i0 < nlist; i0 += kAhead * kRowWaves) {
    u32x4_t v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * kRowWaves;
      if (i < nlist) v[u] = load8<HALF>(x, list[i] * kSegVals + 8 * lane - off, a.V);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i0 + u * kRowWaves >= nlist) break;
      f(i0 + u * kRowWaves, v[u]);
    }
  }
}

// Counts the logits of the listed segments by key, bin hi - key for lo <= key <= hi.
template <bool HALF>
__device__ __forceinline__ void count_keys(const SampleArgs& a, const u16* x, int off, RowShared& sh, int nlist, int hi,
                                           int lo) {
  for (int i = threadIdx.x; i <= hi - lo; i += kRowThreads) sh.bins[i] = 0;
  __syncthreads();
  each_listed<HALF>(a, x, off, sh.list, nlist, [&](int, const u32x4_t& v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = key_of<HALF>(bits_of(v, j));
      if (k >= lo && k <= hi) atomicAdd(&sh.bins[hi - k], 1);
    }
  });
  __syncthreads();
}

// The part of one row that is sampled from: its threshold and normaliser (RowInfo), and px of token `draft`.
// Up to kListed of its tokens are written out as (index, weight) in falling order.
template <bool HALF>
__device__ __forceinline__ RowInfo select_row(const SampleArgs& a, int seq, int ri, int draft, RowShared& sh, int* out_idx,
                                              double* out_w) {
  const int t = threadIdx.x, lane = t & 63;
  const u16* x = row_ptr(a, seq, ri);
  const int off = row_off(x);
  const long row = (long)seq * a.per + ri;
  const float sm = t < a.nseg ? a.segm[row * a.nseg + t] : -INFINITY;      // kMaxSegs <= kRowThreads
  const double ss = !a.top_k && t < a.nseg ? a.segs[row * a.nseg + t] : 0;
  const u32 dbits = draft >= 0 && draft < a.V ? x[draft] : 0x8000u | kInfBits<HALF>;
  RowInfo out;
  float mx = wave_max(sm);
  if (lane == 0) sh.red_f[t >> 6] = mx;
  if (t < a.nseg) sh.skey[t] = key_of_float<HALF>(sm);
  if (t == 0) {
    sh.ncand = 0;
    sh.px = 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowWaves; ++i) mx = fmaxf(mx, sh.red_f[i]);
  out.m = mx;
  out.px = 0;
  out.listed = -1;
  if (!(mx > -INFINITY)) {              // nothing to draw from
    out.z = 0;
    out.thr = 1 << 16;
    out.cut = kNoTies;
    out.listed = 0;
    return out;
  }
  double total = 0;                     // of the whole row; needed where the mass itself is cut
  if (!a.top_k) {
    const double part = wave_total(ss * weight(sm, mx, a.c));
    if (lane == 0) sh.red_d[t >> 6] = part;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRowWaves; ++i) total += sh.red_d[i];
  }
  const int top = key_of_float<HALF>(mx);

  // a key that every kept token reaches
  if (a.top_k && a.nseg < a.top_k && a.nseg <= kMaxSegs / 8) {
    // few segments: the maxima of groups of 8 lanes instead
    for (int s = uniform(t >> 6); s < a.nseg; s += kRowWaves) {
      const u32x4_t v = load8<HALF>(x, s * kSegVals + 8 * lane - off, a.V);
      int k = key_of<HALF>(bits_of(v, 0));
#pragma unroll
      for (int j = 1; j < 8; ++j) k = max(k, key_of<HALF>(bits_of(v, j)));
      k = max(k, dpp_i<0xB1, 0xF>(k));   // the exchanges of sum8_lanes
      k = max(k, dpp_i<0x4E, 0xF>(k));
      k = max(k, dpp_i<0x141, 0xF>(k));
      if ((lane & 7) == 0) sh.cnt[8 * s + (lane >> 3)] = k;
    }
    __syncthreads();
    if (t < 64) {
      const int kb = 8 * a.nseg >= a.top_k ? kth_key(sh.cnt, 8 * a.nseg, a.top_k) : 0;
      if (t == 0) sh.kb = min(max(kb, kLowKey<HALF> + 1), top);
    }
  } else if (t < 64) {
    int kb = 0;
    if (a.top_k) {
      if (a.nseg >= a.top_k) kb = kth_key(sh.skey, a.nseg, a.top_k);
    } else {
      // tokens of weight (1 - top_p) S / V or less: all together less than (1 - top_p) S. One key of room
      // for the rounding to 16 bits.
      const double w = (1.0 - a.top_p) * total / (double)a.V;
      kb = key_of_float<HALF>((float)((double)mx + log2(w) / a.c)) - 1;
    }
    if (t == 0) sh.kb = min(max(kb, kLowKey<HALF> + 1), top);
  }
  __syncthreads();
  const int kb = sh.kb;
  int nlist;
  {
    const int f = t < a.nseg && sh.skey[t] >= kb;
    int upto;
    const int at = block_scan(f, sh.red_i, upto, nlist);
    if (f) sh.list[at] = t;
  }
  __syncthreads();

  // few candidates: sort them
  if (nlist <= kAhead * kRowWaves) {
    each_listed<HALF>(a, x, off, sh.list, nlist, [&](int i, const u32x4_t& v) {
      const int v0 = sh.list[i] * kSegVals + 8 * lane - off;
      int n = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) n += key_of<HALF>(bits_of(v, j)) >= kb;
      const int upto = wave_scan(n);
      int base = 0;
      if (lane == 63) base = atomicAdd(&sh.ncand, upto);
      int at = __builtin_amdgcn_readlane(base, 63) + upto - n;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = key_of<HALF>(bits_of(v, j));
        if (k >= kb) {
          if (at < kListed) sh.cand[at] = (uint64_t)(u32)k << 32 | (u32)~(v0 + j);
          ++at;
        }
      }
    });
    __syncthreads();
    const int n = sh.ncand;
    if (n <= kListed) {
      if (t < n) {
        const uint64_t me = sh.cand[t];
        int r = 0;
        for (int i = 0; i < n; ++i) r += sh.cand[i] > me;
        sh.sorted[r] = me;
      }
      __syncthreads();
      const uint64_t me = t < n ? sh.sorted[t] : 0;
      const int key = (int)(me >> 32), idx = (int)~(u32)me;
      const double w = t < n && !(a.top_k && t >= a.top_k) ? weight(val_of_key<HALF>(key), mx, a.c) : 0.0;
      double upto, zk;
      const double before = block_scan(w, sh.red_d, upto, zk);
      const double goal = a.top_p * (a.top_k ? zk : total);
      const int nk = a.top_k ? min(a.top_k, n) : n;
      if (t == 0) sh.keep = nk;
      __syncthreads();
      if (a.top_p < 1.0 && t < nk && before >= goal) atomicMin(&sh.keep, t);
      __syncthreads();
      const int kept = sh.keep;         // at least 1: before is 0 at the first, the goal is not
      if (t == kept - 1) {
        sh.z = upto;
        sh.key = key;
        sh.cut = idx;
      }
      __syncthreads();
      out.z = sh.z;
      out.thr = sh.key;
      out.cut = sh.cut;
      out.listed = kept;
      if (out_idx && t < kept) {
        put_far(out_idx + t, idx);
        put_far(reinterpret_cast<uint64_t*>(out_w) + t, __builtin_bit_cast(uint64_t, w));
      }
      const int dk = key_of<HALF>(dbits);
      if (draft >= 0 && draft < a.V && (dk > out.thr || (dk == out.thr && draft <= out.cut)))
        out.px = weight(val<HALF>(dbits), mx, a.c) / out.z;
      return out;
    }
    __syncthreads();
  }

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
        cm += (double)n * weight(val_of_key<HALF>(hi - b), mx, a.c);
      }
      if (t == 0) sh.owner = kRowThreads;
      int cnt_all, cnt_end;
      double mass_all, mass_end;
      const int cnt_before = block_scan(cn, sh.red_i, cnt_end, cnt_all);
      const double mass_before = block_scan(cm, sh.red_d, mass_end, mass_all);
      // the thread whose bins the goal falls into (the first: running sums may step back by a rounding)
      const bool mine = pass == 0 ? seen + cnt_end >= a.top_k && cn : mass + mass_end >= goal && cn;
      if (mine) atomicMin(&sh.owner, t);
      __syncthreads();
      if (sh.owner == t) {
        int run = seen + cnt_before, r = 0;
        double m0 = mass + mass_before;
        bool hit = false;
        for (int b = b0; b < b1 && !hit; ++b) {
          int n = sh.bins[b];
          if (!n) continue;
          const int all = n;
          if (after_k && hi - b == thr_k) n = keep_k;
          const double w = weight(val_of_key<HALF>(hi - b), mx, a.c);
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
  out.cut = ties ? a.V : kNoTies;       // without a threshold value (thr = kb - 1) no token has that key
  if (keep < ties) {                    // the index of the last kept token of the threshold's value
    each_listed<HALF>(a, x, off, sh.list, nlist, [&](int i, const u32x4_t& v) {
      int n = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) n += __popcll(__ballot(key_of<HALF>(bits_of(v, j)) == thr));
      if (lane == 0) sh.cnt[i] = n;
    });
    __syncthreads();
    const int c = t < nlist ? sh.cnt[t] : 0;
    int upto, all;
    const int before = block_scan(c, sh.red_i, upto, all);
    if (before < keep && keep <= upto) {
      sh.owner = sh.list[t];
      sh.keep = keep - before;
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
  const int dk = key_of<HALF>(dbits);
  if (draft >= 0 && draft < a.V && z > 0 && (dk > out.thr || (dk == out.thr && draft <= out.cut)))
    out.px = weight(val<HALF>(dbits), mx, a.c) / z;
  return out;
}

// ---------------------------------------------------------------- the accept rule

__device__ __forceinline__ double uniform_at(const VerifyIn& in, long at) {
  return in.u64 ? static_cast<const double*>(in.u)[at] : (double)static_cast<const float*>(in.u)[at];
}
__device__ __forceinline__ int drafts_of(const SampleArgs& a, const VerifyIn& in, int seq) {
  return in.lens ? min(max(in.lens[seq], 0), a.per - 1) : a.per - 1;
}

// Whether draft i of sequence seq, with probability px, is refused.
__device__ __forceinline__ bool refused(const SampleArgs& a, const VerifyIn& in, int seq, int i, double px) {
  const int v = in.draft[(long)seq * (a.per - 1) + i];
  const bool inside = v >= 0 && v < a.V;
  const double q = in.q ? (inside ? (double)in.q[seq * in.qb + i * in.qr + v] : 0.0) : 1.0;
  return !(inside && uniform_at(in, (long)seq * a.per + i) * q < px);
}

enum { kDrawRow = 0, kDrawRest = 1, kDrawOther = 2 };   // r = p, max(p - q, 0), p without one token

// r of 8 logits from index v0 (logits outside the row are -inf: no weight, q not read). Without a cut every
// logit's weight is formed; with one, those of which some lane keeps its own.
template <bool HALF, bool CUT>
__device__ __forceinline__ void rest8(const SampleArgs& a, const RowInfo& r, double inv, const u32x4_t& x, int v0, int mode,
                                      const float* q, int skip, double (&out)[8]) {
  const double mc = -(double)r.m * a.c;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const u32 b = bits_of(x, j);
    const int k = key_of<HALF>(b), v = v0 + j;
    const bool kept = k > r.thr || (k == r.thr && v <= r.cut);
    double w = 0;
    if (!CUT || __any(kept)) {
      w = weight(val<HALF>(b), r.m, a.c, mc);
      if (mode == kDrawRest) w = __builtin_fmax(w * inv - (kept && v >= 0 && v < a.V ? (double)q[v] : 0.0), 0.0);
      else if (mode == kDrawOther && v == skip) w = 0;
      w = kept ? w : 0.0;
    }
    out[j] = w;
  }
}

struct DrawShared {
  double sums[kMaxSegs];
  double r[kListed];
  int list[kMaxSegs];                  // segments with a kept token; or the listed tokens, then in order of index
  double red[kRowWaves];
  double before;
  int red_i[kRowWaves];
  int seg, last, token, first;
};

// The token drawn from row ri of a sequence: the first whose running sum of r passes u times the whole.
// `rest`: segment sums of max(p - q, 0) (no cut), `idx` / `w`: the listed tokens (RowInfo::listed >= 0).
template <bool HALF, bool CUT>
__device__ __forceinline__ int draw_token(const SampleArgs& a, const RowInfo& r, int seq, int ri, int mode, const float* q,
                                          int skip, double u, const double* rest, const int* idx, const double* w_list,
                                          DrawShared& sh) {
  const int t = threadIdx.x, lane = t & 63;
  const u16* x = row_ptr(a, seq, ri);
  const int off = row_off(x);
  const long row = (long)seq * a.per + ri;
  const double inv = r.z > 0 ? 1.0 / r.z : 0.0;
  if (t == 0) {
    sh.token = 0;
    sh.seg = kMaxSegs;
    sh.last = -1;
  }
  if (CUT && r.listed >= 0) {           // one token a thread, in the order of their indexes
    const int n = r.listed;
    int me = 0;
    double v = 0;
    if (t < n) {
      me = get_far(idx + t);
      const double w = __builtin_bit_cast(double, get_far(reinterpret_cast<const uint64_t*>(w_list) + t));
      v = w;
      if (mode == kDrawRest) v = __builtin_fmax(w * inv - (double)q[me], 0.0);
      else if (mode == kDrawOther && me == skip) v = 0;
      sh.list[t] = me;
      sh.sums[t] = w;
    }
    __syncthreads();
    int at = 0;
    if (t < n)
      for (int i = 0; i < n; ++i) at += sh.list[i] < me;
    double all = 0, upto = 0;
    for (int tries = 0; tries < 2; ++tries) {
      if (t < n) {
        sh.r[at] = tries ? sh.sums[t] : v;
        sh.list[kListed + at] = me;
      }
      __syncthreads();
      block_scan(t < n ? sh.r[t] : 0.0, sh.red, upto, all);
      if (all > 0 || mode == kDrawRow) break;
      mode = kDrawRow;                  // r is zero throughout: p
    }
    if (t < n && sh.r[t] > 0) {
      atomicMax(&sh.last, t);
      if (upto > u * all) atomicMin(&sh.seg, t);
    }
    __syncthreads();
    const int pick = sh.seg < kMaxSegs ? sh.seg : sh.last;
    return pick >= 0 ? sh.list[kListed + pick] : 0;
  }
  // sums of r over the segments; where r is zero throughout, of p
  const float sm = t < a.nseg ? a.segm[row * a.nseg + t] : -INFINITY;
  double all = 0, before = 0, upto = 0, mine = 0;
  for (int tries = 0; tries < 2; ++tries) {
    if constexpr (CUT) {
      sh.sums[t] = 0;                   // kMaxSegs == kRowThreads
      __syncthreads();
      int n;
      {
        const int f = r.z > 0 && t < a.nseg && key_of_float<HALF>(sm) >= r.thr;
        int up;
        const int at = block_scan(f, sh.red_i, up, n);
        if (f) sh.list[at] = t;
      }
      __syncthreads();
      each_listed<HALF>(a, x, off, sh.list, n, [&](int i, const u32x4_t& v) {
        double w[8], sum = 0;
        rest8<HALF, true>(a, r, inv, v, sh.list[i] * kSegVals + 8 * lane - off, mode, q, skip, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += w[j];
        sum = wave_total(sum);
        if (lane == 0) sh.sums[sh.list[i]] = sum;
      });
    } else {
      if (t < a.nseg) {
        if (mode == kDrawRest) sh.sums[t] = __builtin_bit_cast(double, get_far(reinterpret_cast<const uint64_t*>(rest) + t));
        else sh.sums[t] = r.z > 0 ? a.segs[row * a.nseg + t] * weight(sm, r.m, a.c) : 0.0;
      }
      __syncthreads();
      if (mode == kDrawOther && skip >= 0 && skip < a.V && t < 64) {   // the token's own segment again, without it
        const int s = (skip + off) / kSegVals, v0 = s * kSegVals + 8 * lane - off;
        double w[8], sum = 0;
        rest8<HALF, false>(a, r, inv, load8<HALF>(x, v0, a.V), v0, mode, nullptr, skip, w);
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
  const double goal = u * all;
  if (mine > 0) {
    atomicMax(&sh.last, t);
    if (upto > goal) atomicMin(&sh.seg, t);
  }
  __syncthreads();
  const int s = sh.seg < kMaxSegs ? sh.seg : sh.last;
  if (s >= 0) {
    if (t == s) sh.before = before;
    __syncthreads();
    if (t < 64) {
      const int v0 = s * kSegVals + 8 * lane - off;
      double w[8], sum = 0;
      rest8<HALF, CUT>(a, r, inv, load8<HALF>(x, v0, a.V), v0, mode, q, skip, w);
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

struct CutShared {
  RowShared row;
  DrawShared draw;
};

// With a cut: one row a workgroup; the last of a sequence accepts and draws (VERIFY).
template <bool HALF, bool VERIFY>
__global__ __launch_bounds__(kRowThreads) void sample_cut_kernel(const SampleArgs a, const VerifyIn in, uint64_t* info,
                                                                 int* list_idx, double* list_w) {
  __shared__ CutShared sh;
  const int ri = blockIdx.x, seq = blockIdx.y, m = a.per - 1, t = threadIdx.x;
  const long row = (long)seq * a.per + ri;
  const int draft = VERIFY && ri < m ? in.draft[(long)seq * m + ri] : -1;
  const RowInfo mine = select_row<HALF>(a, seq, ri, draft, sh.row, VERIFY ? list_idx + row * kListed : nullptr,
                                        VERIFY ? list_w + row * kListed : nullptr);
  static_assert(sizeof(RowInfo) == 32, "four words");
  if (t < 4) {
    uint64_t w[4];
    __builtin_memcpy(w, &mine, 32);
    put_far(info + 4 * row + t, t == 0 ? w[0] : t == 1 ? w[1] : t == 2 ? w[2] : w[3]);
  }
  if constexpr (!VERIFY) return;
  if (t == 0 && ri < m) in.px[(long)seq * m + ri] = (float)mine.px;
  if (!arrives_last(a.arrived + seq, a.per, &sh.row.last)) return;
  const int len = drafts_of(a, in, seq);
  if (t == 0) sh.draw.first = len;
  __syncthreads();
  if (t < len) {                        // kMaxDraft < kRowThreads
    const double px = __builtin_bit_cast(double, get_far(info + 4 * ((long)seq * a.per + t) + 1));
    if (refused(a, in, seq, t, px)) atomicMin(&sh.draw.first, t);
  }
  __syncthreads();
  const int n = sh.draw.first;
  const long at = (long)seq * a.per + n;
  uint64_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = get_far(info + 4 * at + i);
  RowInfo r;
  __builtin_memcpy(&r, w, 32);
  const float* q = in.q && n < len ? in.q + seq * in.qb + n * in.qr : nullptr;
  const int skip = n < len ? in.draft[(long)seq * m + n] : -1;
  const int token = draw_token<HALF, true>(a, r, seq, n, n == len ? kDrawRow : q ? kDrawRest : kDrawOther, q, skip,
                                           uniform_at(in, (long)seq * a.per + m), nullptr, list_idx + at * kListed,
                                           list_w + at * kListed, sh.draw);
  write_tokens(a, in, seq, n, token);
}

struct WholeShared {
  double z[kMaxDraft + 1], px[kMaxDraft + 1];
  float m[kMaxDraft + 1];
  DrawShared draw;
  int last;
};

// Without a cut: workgroups over the segments of a sequence. Each joins its rows and accepts; where draft
// probabilities are given, each sums max(p - q, 0) over its segments of the refused row and the last draws.
template <bool HALF>
__global__ __launch_bounds__(kRowThreads) void sample_whole_kernel(const SampleArgs a, const VerifyIn in, double* rest) {
  __shared__ WholeShared sh;
  const int seq = blockIdx.y, m = a.per - 1, t = threadIdx.x, lane = t & 63;
  const int len = drafts_of(a, in, seq);
  for (int i = uniform(t >> 6); i < a.per; i += kRowWaves) {
    const long row = (long)seq * a.per + i;
    const int draft = i < m ? in.draft[(long)seq * m + i] : -1;
    const bool inside = draft >= 0 && draft < a.V;
    const float xd = inside ? val<HALF>(row_ptr(a, seq, i)[draft]) : -INFINITY;
    float mx;
    const double z = join_wave(a.segm + row * a.nseg, a.segs + row * a.nseg, a.nseg, a.c, mx);
    if (lane == 0) {
      sh.z[i] = z;
      sh.m[i] = mx;
      sh.px[i] = z > 0 && xd > -INFINITY ? weight(xd, mx, a.c) / z : 0.0;
    }
  }
  if (t == 0) sh.draw.first = len;
  __syncthreads();
  if (blockIdx.x == 0 && t < m) in.px[(long)seq * m + t] = (float)sh.px[t];
  if (t < len && refused(a, in, seq, t, sh.px[t])) atomicMin(&sh.draw.first, t);
  __syncthreads();
  const int n = sh.draw.first;
  RowInfo r;
  r.z = sh.z[n];
  r.m = sh.m[n];
  r.thr = kLowKey<HALF>;
  r.cut = kNoTies;
  r.listed = -1;
  const bool dense = in.q && n < len;
  const float* q = dense ? in.q + seq * in.qb + n * in.qr : nullptr;
  double* sums = rest + (long)seq * a.nseg;
  if (dense) {
    const u16* x = row_ptr(a, seq, n);
    const int off = row_off(x);
    const double inv = r.z > 0 ? 1.0 / r.z : 0.0;
    for (int s = blockIdx.x * kRowWaves + uniform(t >> 6); s < a.nseg; s += gridDim.x * kRowWaves) {
      const int v0 = s * kSegVals + 8 * lane - off;
      double w[8], sum = 0;
      rest8<HALF, false>(a, r, inv, load8<HALF>(x, v0, a.V), v0, kDrawRest, q, -1, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += w[j];
      sum = wave_total(sum);
      if (lane == 0) put_far(reinterpret_cast<uint64_t*>(sums) + s, __builtin_bit_cast(uint64_t, r.z > 0 ? sum : 0.0));
    }
    if (!arrives_last(a.arrived + seq, gridDim.x, &sh.last)) return;
  } else if (blockIdx.x) {
    return;
  }
  const int skip = n < len ? in.draft[(long)seq * m + n] : -1;
  const int token = draw_token<HALF, false>(a, r, seq, n, n == len ? kDrawRow : q ? kDrawRest : kDrawOther, q, skip,
                                            uniform_at(in, (long)seq * a.per + m), sums, nullptr, nullptr, sh.draw);
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
      rest8<HALF, CUT>(a, r, inv, v[i], v0, kDrawRow, nullptr, -1, w);
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
  size_t segs, rest, list_w, info, segm, list_idx, arrived, bytes;
};

Layout layout(int64_t rows, int64_t V, int64_t sequences) {
  const size_t n = (size_t)((V + 7 + kSegVals - 1) / kSegVals), listed = sequences ? (size_t)rows * kListed : 0;
  const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  Layout l;
  l.segs = 0;
  l.rest = up(l.segs + (size_t)rows * n * 8);
  l.list_w = up(l.rest + (size_t)sequences * n * 8);
  l.info = up(l.list_w + listed * 8);
  l.segm = up(l.info + (size_t)rows * sizeof(RowInfo));
  l.list_idx = up(l.segm + (size_t)rows * n * 4);
  l.arrived = up(l.list_idx + listed * 4);
  l.bytes = up(l.arrived + (size_t)sequences * 4);
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
  const dim3 grid(groups(a.nseg, 4), (unsigned)a.per, (unsigned)(a.rows / a.per)), block(kStatThreads);
  if (a.top_k) hipLaunchKernelGGL((sample_segments_kernel<HALF, 4, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((sample_segments_kernel<HALF, 4, true>), grid, block, 0, s, a);
}

template <bool HALF>
void probs(const SampleArgs& a, uint64_t* info, float* out, long ldo, hipStream_t s) {
  const dim3 grid(groups(a.nseg, 4), (unsigned)a.rows);
  launch_segments<HALF>(a, s);
  if (a.top_k || a.top_p < 1.0) {
    hipLaunchKernelGGL((sample_cut_kernel<HALF, false>), dim3(1, (unsigned)a.rows), dim3(kRowThreads), 0, s, a, VerifyIn{}, info,
                       nullptr, nullptr);
    hipLaunchKernelGGL((sample_probs_kernel<HALF, true, 4>), grid, dim3(kStatThreads), 0, s, a, info, out, ldo);
  } else {
    hipLaunchKernelGGL((sample_probs_kernel<HALF, false, 4>), grid, dim3(kStatThreads), 0, s, a, info, out, ldo);
  }
}

template <bool HALF>
void verify(const SampleArgs& a, const VerifyIn& in, char* w, const Layout& l, hipStream_t s) {
  const unsigned B = (unsigned)(a.rows / a.per);
  launch_segments<HALF>(a, s);
  if (a.top_k || a.top_p < 1.0) {
    hipLaunchKernelGGL((sample_cut_kernel<HALF, true>), dim3((unsigned)a.per, B), dim3(kRowThreads), 0, s, a, in,
                       reinterpret_cast<uint64_t*>(w + l.info), reinterpret_cast<int*>(w + l.list_idx),
                       reinterpret_cast<double*>(w + l.list_w));
  } else {
    // where there are draft probabilities, a workgroup a CU over the refused rows, at most one a wave and segment
    const unsigned most = (unsigned)((a.nseg + kRowWaves - 1) / kRowWaves), fill = B < 256 ? 256 / B : 1;
    const unsigned g = in.q ? (most < fill ? most : fill) : 1;
    hipLaunchKernelGGL((sample_whole_kernel<HALF>), dim3(g, B), dim3(kRowThreads), 0, s, a, in,
                       reinterpret_cast<double*>(w + l.rest));
  }
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
  a.arrived = nullptr;
  uint64_t* info = reinterpret_cast<uint64_t*>(static_cast<char*>(p->workspace) + l.info);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == DSPARK_DTYPE_F16) probs<true>(a, info, p->out, p->ldo, s);
  else probs<false>(a, info, p->out, p->ldo, s);
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
  a.arrived = reinterpret_cast<int*>(w + l.arrived);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == DSPARK_DTYPE_F16) verify<true>(a, in, w, l, s);
  else verify<false>(a, in, w, l, s);
  return check_launch(what);
}
