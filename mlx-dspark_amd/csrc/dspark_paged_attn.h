// Attention over paged caches for gfx950: few rows of each sequence (decoded tokens, verify blocks).
//
// out[row] = softmax(scale q . k^T) . v over the keys that the row sees: keys 0 .. len - n + i of its sequence for row i of
// n (causal), or all of them; fp32 scores, running maximum and sum in one pass over the keys. The rows of a sequence and
// KV head, R = n times the query heads of the group, are (token, query head), heads fastest.
//
// Bound by the bytes of K and V. 32 tokens behind 90 to 8192 positions, 32 / 8 heads of 128: 524 MB in 95 us (5.5 TB/s; 111 with
// loads that fill the caches); two behind 70001 and 100000 8-bit positions, 64 / 8 heads: 395 MB in 76 us. Hence:
//   * the work is the list of all (sequence, KV head, row group, 128 keys), dealt in equal runs to a fixed number of
//     workgroups, whatever the lengths: a workgroup's run covers the end of one KV head, whole ones, and the start of
//     another. What is not whole goes to the workspace as unnormalised fp32 outputs with their maxima and sums, two slots a
//     workgroup, and a second launch joins them in the order of the keys. Lengths stay on the device;
//   * a wave takes 32 of the 128 keys by itself: no barrier in the loop. The next keys and values are in flight in
//     registers while the present ones are multiplied; one page's 16 positions have one address, so page ids are kept 64 a
//     wave in a register and read by the lane number;
//   * S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32: a lane holds 4 + 4 keys of one row, which are, in place, what
//     the second product needs. K goes from memory to the operand, V through LDS (the transposing read), 16-byte
//     chunks XOR-swizzled by the row;
//   * 8-bit pages are turned into the model's type as they are used: one conversion for two values with the page's power of
//     two in it, exact for every page that a model of that type wrote, but for values past fp16's largest: keys take what fp16 does not
//     hold of their power of two to the scores (key_unit), values become infinite, and their rows are computed again.
// Probabilities go to the matrix cores as two pieces of the type (16 bits of bf16, 20 and more of fp16, there of p 2^15), over 8-bit pages
// too: at these row counts the second piece costs nothing.
//
// Values that are not finite are only let through where a row sees them: a row with such an output, or one that sees keys and has
// no probability (scores of -inf), is computed again in plain fp32 from the keys it sees (plain_row).
#pragma once

#include "dspark_attn.h"
#include "dspark_paged.h"

namespace dspark {
namespace paged {

using attn::BF16;
using attn::F16;

constexpr int kAttnThreads = 256;
constexpr int kWaves = 4;
constexpr int kWaveKeys = 32;                       // keys of a wave's step
constexpr int kUnit = kWaves * kWaveKeys;           // of a workgroup's
constexpr float kLowest = -3.402823466e38f;
constexpr u32 kMostUnits = 1u << 30;                // of a call

struct AttnArgs {
  Seqs s;
  Pages k, v;
  const u16* q;
  u16* out;
  long qrow, qhead, orow, ohead;                    // element strides
  float* opart;                                     // [workgroup][2 slots][16 RT rows][D], unnormalised
  float* mpart;                                     // [workgroup][2 slots][16 RT rows]: maxima, then sums
  int Hq, Hk, gqa, causal;
  int whole;                                        // a workgroup takes whole (sequence, KV head, row group)s: nothing to join
  int least;                                        // units of a run, at least
  int rows_up_to;                                   // sequences with more rows of a KV head are another kernel's
  int clear;                                        // rows of no sequence: zeros
  float scale_log2;
};

// A sequence's share of the work list
struct Work {
  int start, n, len, full;                          // first row, rows, keys that the table has, and as given
  int rows, groups, tiles;                          // rows and row groups of a KV head, units along the keys
};

template <int RT>
__device__ __forceinline__ Work work_of(const AttnArgs& a, int b) {
  const Seq q = sequence(a.s, b);
  Work w{q.start, q.n, q.len, q.full, q.n * a.gqa, 0, 0};
  if (w.rows > a.rows_up_to || q.n == 0) w.rows = 0;
  w.groups = (w.rows + 16 * RT - 1) / (16 * RT);
  w.tiles = a.whole ? 1 : (q.len + kUnit - 1) / kUnit;
  return w;
}

__device__ __forceinline__ Work lane_work(const Work& w, int l) {
  auto at = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
  return Work{at(w.start), at(w.n), at(w.len), at(w.full), at(w.rows), at(w.groups), at(w.tiles)};
}

__device__ __forceinline__ u32 units_of(const AttnArgs& a, const Work& w) {
  const unsigned long long n = (unsigned long long)a.Hk * (unsigned)w.groups * (unsigned)w.tiles;
  return n > kMostUnits ? kMostUnits + 1 : (u32)n;
}

// The work of all sequences: that of the first 64 is looked up once, a lane each
template <int RT>
struct Works {
  const AttnArgs& a;
  Work first;

  __device__ __forceinline__ explicit Works(const AttnArgs& args) : a(args), first(work_of<RT>(args, min((int)__lane_id(), args.s.B - 1))) {}
  __device__ __forceinline__ u32 units(int b) const {        // of sequence b = 64 i + lane
    return b >= a.s.B ? 0u : b < 64 ? units_of(a, first) : units_of(a, work_of<RT>(a, b));
  }
  __device__ __forceinline__ Work at(int b) const {          // b: the wave's
    if (b < 64) return lane_work(first, b);
    return lane_work(work_of<RT>(a, b), 0);
  }
  // Units of all sequences, and of those before `upto`; none where they are more than a call may have (the entry point
  // checks that: only sequences that share their rows come to that here)
  __device__ __forceinline__ int all(int upto, int* before) const {
    const int lane = __lane_id();
    u32 sum = 0, some = 0;
    for (int b0 = 0; b0 < a.s.B; b0 += 64) {
      const u32 n = units(b0 + lane);
      sum = __builtin_elementwise_add_sat(sum, n);
      if (b0 + lane < upto) some += n;
    }
    const u32 total = (u32)__builtin_amdgcn_readlane((int)wave_scan(sum), 63);
    if (total > kMostUnits) return 0;
    if (before) *before = __builtin_amdgcn_readlane((int)wave_scan(some), 63);
    return (int)total;
  }
};

__device__ __forceinline__ int run_of(const AttnArgs& a, int units, int workgroups) {
  const int even = (units + workgroups - 1) / workgroups;
  return even > a.least ? even : a.least;
}

template <class T, bool CODES>
__device__ __forceinline__ float element(const Pages& p, long at, float unit) {
  if constexpr (CODES) return __builtin_amdgcn_cvt_f32_fp8((int)(unsigned char)p.data[at], 0) * unit;
  else return attn::to_f32<T>(reinterpret_cast<const u16*>(p.data)[at]);
}

// One row again, by one wave, in plain fp32 over the keys it sees: largest score, sum, then probabilities times values.
template <class T, int D, bool CODES>
__device__ __forceinline__ void plain_row(const AttnArgs& a, int b, int t, int head, int keys) {
  const int lane = __lane_id(), h = head / a.gqa;
  const u16* q = a.q + t * a.qrow + head * a.qhead;
  u16* o = a.out + t * a.orow + head * a.ohead + lane * (D / 64);
  bool some = false;                                         // a key that is there
  for (int p = lane; (long)p << a.s.log2P < keys; p += 64) some |= page_of(a.s, b, (long)p << a.s.log2P) >= 0;
  if (!__builtin_amdgcn_ballot_w64(some)) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c) o[c] = 0;
    return;
  }
  auto unit = [&](const Pages& p, int id) {
    return CODES ? scale_of(p.exps[id * p.epage + h * p.ehead]) : 1.f;
  };
  auto score = [&](int key) {
    const int id = key < keys ? page_of(a.s, b, key) : -1;
    if (id < 0) return -__builtin_inff();
    const long at = id * a.k.page + h * a.k.head + (key & (a.s.P - 1)) * a.k.row;
    const float u = unit(a.k, id);
    float s = 0.f;
#pragma unroll 1
    for (int d = 0; d < D; ++d) s = __builtin_fmaf(attn::to_f32<T>(q[d]), element<T, CODES>(a.k, at + d, u), s);
    return s;
  };
  auto seen = [&](int key) { return key < keys && page_of(a.s, b, key) >= 0; };
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll 1
  for (int k0 = 0; k0 < keys; k0 += 64) m = fmaxf(m, score(k0 + lane));
#pragma unroll 1
  for (int x = 1; x < 64; x *= 2) m = fmaxf(m, shfl_xor(m, x));
  auto weight = [&](int key) { return seen(key) ? __builtin_amdgcn_exp2f((score(key) - m) * a.scale_log2) : 0.f; };
#pragma unroll 1
  for (int k0 = 0; k0 < keys; k0 += 64) l += weight(k0 + lane);
#pragma unroll 1
  for (int x = 1; x < 64; x *= 2) l += shfl_xor(l, x);
  float sum[D / 64] = {};
#pragma unroll 1
  for (int k0 = 0; k0 < keys; k0 += 64) {
    const float p = weight(k0 + lane) / l;
#pragma unroll 1
    for (int j = 0; j < min(64, keys - k0); ++j) {
      const int id = page_of(a.s, b, k0 + j);
      if (id < 0) continue;
      const float pj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), j)), u = unit(a.v, id);
      const long at = id * a.v.page + h * a.v.head + ((k0 + j) & (a.s.P - 1)) * a.v.row + lane * (D / 64);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) sum[c] = __builtin_fmaf(pj, element<T, CODES>(a.v, at + c, u), sum[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < D / 64; ++c) o[c] = attn::from_f32<T>(sum[c]);
}

// Keys that row i of a sequence's n sees
template <class W>
__device__ __forceinline__ int keys_seen(const AttnArgs& a, const W& w, int i) {
  if (!a.causal) return w.len;
  const int k = w.full - w.n + i + 1;                        // full > 0
  return k < 0 ? 0 : k < w.len ? k : w.len;
}

// 16 codes as 16 values of T
template <class T>
__device__ __forceinline__ void decode(u32x4_t c, float unit, u32x4_t& lo, u32x4_t& hi) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u32 x, y;
    if constexpr (T::kF16) {
      x = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], unit, false));
      y = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], unit, true));
    } else {
      x = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], unit, false));
      y = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], unit, true));
    }
    if (i < 2) lo[2 * i] = x, lo[2 * i + 1] = y;
    else hi[2 * i - 4] = x, hi[2 * i - 3] = y;
  }
}

// What a page's power of two leaves of itself where its keys become values of T, and what multiplies their scores instead: fp16
// has all codes, 2^-9 to 448 in size, times 2^-15 to 2^7. (fp16 rows of 63489 and more become 256 2^8 = 65536: as an fp16 infinity such a
// key had no weight, or all of it.)
template <class T>
__device__ __forceinline__ float key_unit(float unit) { return T::kF16 ? fminf(fmaxf(unit, 0x1p-15f), 0x1p7f) : unit; }
template <class T>
__device__ __forceinline__ float key_rest(float unit) {
  return key_unit<T>(unit) == unit ? 1.f : unit * (unit < 1.f ? 0x1p15f : 0x1p-7f);
}

// The 16-byte chunk c of row r of a V tile lies at chunk c ^ tile_swz(r): a transposing read takes two chunks of 16 rows
template <int D>
__device__ __forceinline__ int tile_swz(int r) { return D == 64 ? ((r >> 1) & 3) << 1 : (r & 7) << 1; }

__device__ __forceinline__ u32x2_t lds_transposed(const u16* p) {
  typedef short s16x4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}

// What a wave writes to LDS for itself is in place before it reads it
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Zeros in rows of no sequence
template <int D>
__device__ __forceinline__ void clear_rows(const AttnArgs& a) {
  constexpr int CH = D / 8;
  const int lane = __lane_id();
  if (all_rows_taken(a.s)) return;
  for (int t = blockIdx.x; t < a.s.T; t += gridDim.x) {
    bool has = false;
    for (int b0 = 0; b0 < a.s.B; b0 += 64) {
      const Seq q = sequence(a.s, min(b0 + lane, a.s.B - 1));
      has |= q.n > 0 && t >= q.start && t < q.start + q.n;
    }
    if (__builtin_amdgcn_ballot_w64(has)) continue;
    for (int i = threadIdx.x; i < a.Hq * CH; i += kAttnThreads)
      *reinterpret_cast<u32x4_t*>(a.out + t * a.orow + i / CH * a.ohead + 8 * (i % CH)) = u32x4_t{0u, 0u, 0u, 0u};
  }
}

template <class T, int D, int RT, bool CODES>
__global__ __launch_bounds__(kAttnThreads, RT * D > 256 || D == 256 ? 1 : 2) void rows_kernel(const AttnArgs a) {
  constexpr int ROWS = 16 * RT, NC = D / 32, ND = D / 16;
  constexpr int KL = CODES ? D / 64 : D / 32;                // 16-byte loads of a lane for 16 keys
  constexpr int VCH = CODES ? D / 16 : D / 8;                // 16-byte chunks of a row in memory
  constexpr int VL = kWaveKeys * VCH / 64;                   // of a lane for the wave's keys
  __shared__ __attribute__((aligned(16))) u16 tiles[kWaves][kWaveKeys * D];      // V; then the waves' outputs
  __shared__ float wm[kWaves][ROWS], wl[kWaves][ROWS];
  __shared__ int again[ROWS];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int c16 = lane & 15, q4 = lane >> 4;
  u16* const vt = tiles[wave];

  if (a.clear) clear_rows<D>(a);
  const Works<RT> works(a);
  const int units = works.all(0, nullptr), run = a.whole ? 1 : run_of(a, units, gridDim.x);
  if ((long)blockIdx.x * run >= units) return;
  int u = blockIdx.x * run;
  const int u_end = min(u + run, units);
  int b, local;
  if (!locate((u32)u, a.s.B, [&](int i) { return works.units(i); }, b, local)) return;
  Work w = works.at(b);

  while (u < u_end) {
    // the KV head and row group, and the units [t0, t1) of it
    const int seg = local / w.tiles, t0 = local - seg * w.tiles;
    const int t1 = min(w.tiles, t0 + (u_end - u));
    const int h = seg / w.groups, r0 = (seg - h * w.groups) * ROWS;
    const int key0 = t0 * kUnit, key1 = a.whole ? w.len : min(w.len, t1 * kUnit);

    u32x4_t qf[RT][NC];
    int lim[RT];                                             // keys that this lane's rows see
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = min(r0 + 16 * rt + c16, w.rows - 1), i = r / a.gqa;
      lim[rt] = keys_seen(a, w, i);
      const u16* qp = a.q + (w.start + i) * a.qrow + (h * a.gqa + r - i * a.gqa) * a.qhead;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        qf[rt][c] = CODES ? ldg128(qp + 64 * (c >> 1) + 16 * q4 + 8 * (c & 1)) : ldg128(qp + 32 * c + 8 * q4);
    }
    const int all_see = uniform(keys_seen(a, w, min(r0, w.rows - 1) / a.gqa));

    // page ids (and scales) of 64 pages, a lane each
    const int* const row = a.s.table + b * a.s.ldt;
    int ids = -1, ids_at = -(1 << 30);                        // of page ids_at + lane
    float ku = 1.f, vu = 1.f;
    auto fetch_ids = [&](int first) {
      ids_at = first;
      const int p = first + lane;
      const int id = p <= (w.len - 1) >> a.s.log2P ? row[p] : -1;
      ids = (unsigned)id < (unsigned)a.s.pool ? id : -1;
      if constexpr (CODES) {
        ku = vu = 0.f;
        if (ids >= 0) {
          ku = scale_of(a.k.exps[ids * a.k.epage + h * a.k.ehead]);
          vu = scale_of(a.v.exps[ids * a.v.epage + h * a.v.ehead]);
        }
      }
    };

    u32x4_t kr[2][KL], vr[VL];
    int id0 = -1, id1 = -1;                                  // pages of the two 16-key halves in flight
    float ku0 = 1.f, ku1 = 1.f, vu0 = 1.f, vu1 = 1.f;
    auto lane_of = [&](float x, int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l)); };
    auto find_pages = [&](int key) {
      const int p0 = key >> a.s.log2P, p1 = (key + 16) >> a.s.log2P;
      if (p0 < ids_at || p1 >= ids_at + 64) fetch_ids(p0);
      id0 = __builtin_amdgcn_readlane(ids, p0 - ids_at);
      id1 = __builtin_amdgcn_readlane(ids, p1 - ids_at);
      if constexpr (CODES) {
        ku0 = lane_of(ku, p0 - ids_at), ku1 = lane_of(ku, p1 - ids_at);
        vu0 = lane_of(vu, p0 - ids_at), vu1 = lane_of(vu, p1 - ids_at);
      }
    };
    constexpr int ES = CODES ? 1 : 2;
    auto at = [&](const Pages& p, int id, int key) {         // of a half's first row; pages that are not there: any
      return p.data + (max(id, 0) * p.page + h * p.head + (key & (a.s.P - 1)) * p.row) * ES;
    };
    auto load_k = [&](int key) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const char* p = at(a.k, s ? id1 : id0, key + 16 * s) + (c16 * (int)a.k.row * ES + 16 * q4);
#pragma unroll
        for (int c = 0; c < KL; ++c) kr[s][c] = ldg128_nt(p + 64 * c);
      }
    };
    auto load_v = [&](int key) {
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const int chunk = j * 64 + lane, r = chunk / VCH;    // rows of one load lie in one half
        const bool second = j >= VL / 2;
        vr[j] = ldg128_nt(at(a.v, second ? id1 : id0, key + (second ? 16 : 0)) + ((r & 15) * (int)a.v.row * ES + 16 * (chunk % VCH)));
      }
    };

    f32x4_t o[RT][ND];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = kLowest;
      l[rt] = 0.f;
#pragma unroll
      for (int t = 0; t < ND; ++t) o[rt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    int key = key0 + wave * kWaveKeys;
    if (key < key1) {
      find_pages(key);
      load_k(key);
      load_v(key);
    }
    while (key < key1) {
      const bool bad0 = id0 < 0, bad1 = id1 < 0;
      // S^T of the two halves
      f32x4_t s[RT][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KL; ++c) {
          if constexpr (CODES) {
            u32x4_t lo, hi;
            decode<T>(kr[j][c], key_unit<T>(j ? ku1 : ku0), lo, hi);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              s[rt][j] = attn::mfma<T>(lo, qf[rt][2 * c], s[rt][j]);
              s[rt][j] = attn::mfma<T>(hi, qf[rt][2 * c + 1], s[rt][j]);
            }
          } else {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt][j] = attn::mfma<T>(kr[j][c], qf[rt][c], s[rt][j]);
          }
        }
        if constexpr (CODES && T::kF16) {
          const float rest = key_rest<T>(j ? ku1 : ku0);
          if (rest != 1.f) {                                 // wave-uniform
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt][j] *= rest;
          }
        }
      }
      // V of these keys to LDS; rows past the sequence's are nobody's, and zero
      wave_lds_fence();
      const bool short_tile = key + kWaveKeys > w.len;
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const int chunk = j * 64 + lane, r = chunk / VCH, c = chunk % VCH;
        u32x4_t x = vr[j];
        if constexpr (CODES) {
          u32x4_t lo, hi;
          decode<T>(x, j >= VL / 2 ? vu1 : vu0, lo, hi);
          if (short_tile && key + r >= w.len) lo = hi = u32x4_t{0u, 0u, 0u, 0u};
          *reinterpret_cast<u32x4_t*>(vt + r * D + (((2 * c) ^ tile_swz<D>(r)) << 3)) = lo;
          *reinterpret_cast<u32x4_t*>(vt + r * D + (((2 * c + 1) ^ tile_swz<D>(r)) << 3)) = hi;
        } else {
          if (short_tile && key + r >= w.len) x = u32x4_t{0u, 0u, 0u, 0u};
          *reinterpret_cast<u32x4_t*>(vt + r * D + ((c ^ tile_swz<D>(r)) << 3)) = x;
        }
      }
      wave_lds_fence();
      const int cur = key;
      key += kUnit;
      if (key < key1) {
        find_pages(key);
        load_k(key);
        load_v(key);
      }

      u32x4_t ph[RT], pl[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (cur + kWaveKeys > all_see || bad0 || bad1) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (cur + 16 * j + 4 * q4 + i >= lim[rt] || (j ? bad1 : bad0)) s[rt][j][i] = -__builtin_inff();
        }
        float mx = m[rt];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rt][j][i]);
        mx = max_xor32(max_xor16(mx));
        if (__builtin_amdgcn_ballot_w64(mx > m[rt])) {
          const float alpha = __builtin_amdgcn_exp2f((m[rt] - mx) * a.scale_log2);
          m[rt] = mx;
          l[rt] *= alpha;
#pragma unroll
          for (int t = 0; t < ND; ++t) o[rt][t] *= alpha;
        }
        float p[8];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = __builtin_amdgcn_exp2f((s[rt][j][i] - mx) * a.scale_log2);
            if constexpr (T::kF16) x *= 32768.f;
            p[4 * j + i] = x;
            l[rt] += x;
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const u32 hi = attn::pack2<T>(p[2 * i], p[2 * i + 1]);
          ph[rt][i] = hi;
          pl[rt][i] = attn::pack2<T>(p[2 * i] - attn::to_f32<T>(hi & 0xFFFFu), p[2 * i + 1] - attn::to_f32<T>(hi >> 16));
        }
      }
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        const int r = 4 * q4 + (c16 >> 2);
        const u16* vp = vt + r * D + (((2 * t + ((c16 & 3) >> 1)) ^ tile_swz<D>(r)) << 3) + 4 * (c16 & 1);
        const u32x2_t lo = lds_transposed(vp), hi = lds_transposed(vp + 16 * D);
        const u32x4_t vf = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          o[rt][t] = attn::mfma<T>(vf, ph[rt], o[rt][t]);
          o[rt][t] = attn::mfma<T>(vf, pl[rt], o[rt][t]);
        }
      }
    }

    // the waves' parts together: a common maximum, then sums row tile by row tile
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] += shfl_xor(l[rt], 16);
      l[rt] += shfl_xor(l[rt], 32);
      if (q4 == 0) {
        wm[wave][16 * rt + c16] = m[rt];
        wl[wave][16 * rt + c16] = l[rt];
      }
    }
    if (tid < ROWS) again[tid] = 0;
    __syncthreads();
    const bool complete = t0 == 0 && t1 == w.tiles;
    const long slot = (2 * (long)blockIdx.x + (t0 == 0 ? 1 : 0)) * ROWS;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int rw = 16 * rt + c16;
      const float mt = fmaxf(fmaxf(wm[0][rw], wm[1][rw]), fmaxf(wm[2][rw], wm[3][rw]));
      const float f = __builtin_amdgcn_exp2f((m[rt] - mt) * a.scale_log2);
      f32x4_t* const mine = reinterpret_cast<f32x4_t*>(vt);
#pragma unroll
      for (int t = 0; t < ND; ++t) mine[t * 64 + lane] = o[rt][t] * f;
      __syncthreads();
      float lt = 0.f;                                        // of the row whose outputs this thread sums
#pragma unroll
      for (int i = 0; i < kWaves; ++i) lt += wl[i][rw] * __builtin_amdgcn_exp2f((wm[i][rw] - mt) * a.scale_log2);
      const int r = r0 + rw, i = r / a.gqa;
      if (r < w.rows) {
        const float inv = lt > 0.f ? 1.f / lt : 0.f;
        float zero = lt > 0.f || lim[rt] == 0 ? lt - lt : 1.f;       // NaN once an output is not finite
        for (int x = wave; x < ND; x += kWaves) {
          f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < kWaves; ++k) sum += reinterpret_cast<const f32x4_t*>(tiles[k])[x * 64 + lane];
          if (complete) {
#pragma unroll
            for (int k = 0; k < 4; ++k) zero = __builtin_fmaf(sum[k], 0.f, zero);
            *reinterpret_cast<u32x2_t*>(a.out + (w.start + i) * a.orow + (h * a.gqa + r - i * a.gqa) * a.ohead + 16 * x + 4 * q4) =
                u32x2_t{attn::pack2<T>(sum[0] * inv, sum[1] * inv), attn::pack2<T>(sum[2] * inv, sum[3] * inv)};
          } else {
            *reinterpret_cast<f32x4_t*>(a.opart + (slot + rw) * D + 16 * x + 4 * q4) = sum;
          }
        }
        if (complete) {
          if (zero != 0.f) again[rw] = 1;
        } else if (wave == 0 && q4 == 0) {
          a.mpart[2 * slot + rw] = mt;
          a.mpart[2 * slot + ROWS + rw] = lt;
        }
      }
      __syncthreads();
    }
    if (complete) {
      __threadfence_block();
      for (int r = wave; r < ROWS; r += kWaves)
        if (again[r]) {
          const int i = (r0 + r) / a.gqa;
          plain_row<T, D, CODES>(a, b, w.start + i, h * a.gqa + r0 + r - i * a.gqa, keys_seen(a, w, i));
        }
    }
    __syncthreads();

    u += t1 - t0;
    local += t1 - t0;
    if (u < u_end && local == a.Hk * w.groups * w.tiles) {
      local = 0;
      do {
        ++b;
        w = works.at(b);
      } while (w.rows == 0 && b < a.s.B - 1);
      if (w.rows == 0) return;
    }
  }
}

// Parts of a row, joined by a wave: out = sum_z 2^(m_z - m) o_z / sum_z 2^(m_z - m) l_z in the order of the keys. `part(z)`:
// where part z's row stands among the outputs; its maximum (times `c` in the exponent) and sum at `stat(z)` and `stat(z)` +
// `sums`. A lane looks at a part's maximum and sum, while N parts' outputs are on their way.
template <int C>
struct Joined {
  float v[C];                    // unnormalised columns of the lane
  float m, l;
};
template <int D, int N, class Part, class Stat>
__device__ __forceinline__ Joined<D / 64> join_parts(const float* o, const float* stats, int sums, float c, int parts, int first,
                                                     int step, Part part, Stat stat) {
  constexpr int C = D / 64;
  typedef float cols_t __attribute__((ext_vector_type(C)));
  const int lane = __lane_id();
  cols_t x[N];
  auto load = [&](int z) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      x[k] = *reinterpret_cast<const cols_t*>(o + part(min(z + k * step, parts - 1)) * D + C * lane);
  };
  load(first);
  float ms = stats[stat(min(lane, parts - 1))], ls = stats[stat(min(lane, parts - 1)) + sums];
  Joined<C> r;
#pragma unroll
  for (int i = 0; i < C; ++i) r.v[i] = 0.f;
  r.m = ms;
  for (int z = lane + 64; z < parts; z += 64) r.m = fmaxf(r.m, stats[stat(z)]);
#pragma unroll
  for (int y = 1; y < 64; y *= 2) r.m = fmaxf(r.m, shfl_xor(r.m, y));
  r.l = 0.f;
  for (int z0 = 0; z0 < parts; z0 += 64) {
    if (z0) {
      const int z = min(z0 + lane, parts - 1);
      ms = stats[stat(z)], ls = stats[stat(z) + sums];
    }
    const float f = z0 + lane < parts ? __builtin_amdgcn_exp2f((ms - r.m) * c) : 0.f;
    r.l += f * ls;
    const int n = min(64, parts - z0);
    for (int j = first; j < n; j += step * N) {
      if (z0 + j != first) load(z0 + j);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float fk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(j + k * step, n - 1)));
        // (a part of weight 0 may hold what is not finite: it would have to count, were it there)
#pragma unroll
        for (int i = 0; i < C; ++i) r.v[i] = j + k * step < n ? __builtin_fmaf(fk, x[k][i], r.v[i]) : r.v[i];
      }
    }
  }
#pragma unroll
  for (int y = 1; y < 64; y *= 2) r.l += shfl_xor(r.l, y);
  return r;
}

// A joined row to its place, by a wave
template <class T, int D, bool CODES>
__device__ __forceinline__ void put_row(const AttnArgs& a, const float (&v)[D / 64], float l, int b, int t, int head, int keys) {
  constexpr int C = D / 64;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  u16* op = a.out + t * a.orow + head * a.ohead + C * (int)__lane_id();
  float zero = l > 0.f || keys == 0 ? l - l : 1.f;
  u16 x[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    zero = __builtin_fmaf(v[i], 0.f, zero);
    x[i] = attn::from_f32<T>(v[i] * inv);
  }
  if constexpr (C == 4) *reinterpret_cast<u32x2_t*>(op) = u32x2_t{x[0] | (u32)x[1] << 16, x[2] | (u32)x[3] << 16};
  else if constexpr (C == 2) *reinterpret_cast<u32*>(op) = x[0] | (u32)x[1] << 16;
  else op[0] = x[0];
  if (__builtin_amdgcn_ballot_w64(zero != 0.f)) plain_row<T, D, CODES>(a, b, t, head, keys);
}

// Joins the parts of a KV head's rows. Few parts, up to 8 on the average: a wave a row (32 tokens behind 600 to 2500 positions
// 48.7 -> 46.4 us with the first launch, 16 blocks of 4 to 8 rows 48 -> 39); many: a workgroup a row, whose waves take every
// fourth part (one token behind 100000 positions has 64).
template <class T, int D, int RT, bool CODES, bool FEW>
__global__ __launch_bounds__(kAttnThreads) void join_kernel(const AttnArgs a, int workgroups) {
  constexpr int ROWS = 16 * RT, C = D / 64, AT_ONCE = FEW ? 4 : C == 4 ? 8 : 16, STEP = FEW ? kWaves : 1;
  __shared__ float sm[kWaves][FEW ? 1 : D];
  const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
  const int b = blockIdx.x / a.Hk, h = blockIdx.x - b * a.Hk;
  const Works<RT> works(a);
  const Work w = works.at(b);
  if ((int)blockIdx.y * STEP >= w.rows) return;
  int before = 0;
  const int units = works.all(b, &before);
  if (!units) return;
  const int run = run_of(a, units, workgroups);
  for (int r = (int)blockIdx.y * STEP + (FEW ? wave : 0); r < w.rows; r += gridDim.y * STEP) {
    const int group = r / ROWS, rw = r - group * ROWS, i = r / a.gqa;
    const int u0 = before + (h * w.groups + group) * w.tiles, u1 = u0 + w.tiles;
    const int j0 = u0 / run, j1 = (u1 - 1) / run;
    if (j0 == j1) continue;
    auto slot = [&](int z) { return (2 * (long)(j0 + z) + (z == 0 ? 1 : 0)) * ROWS; };
    Joined<C> x = join_parts<D, AT_ONCE>(a.opart, a.mpart, ROWS, a.scale_log2, j1 - j0 + 1, FEW ? 0 : wave, FEW ? 1 : kWaves,
                                         [&](int z) { return slot(z) + rw; }, [&](int z) { return 2 * slot(z) + rw; });
    if constexpr (!FEW) {
#pragma unroll
      for (int c = 0; c < C; ++c) sm[wave][C * lane + c] = x.v[c];
      __syncthreads();
#pragma unroll
      for (int c = 0; c < C; ++c) x.v[c] = (sm[0][C * lane + c] + sm[1][C * lane + c]) + (sm[2][C * lane + c] + sm[3][C * lane + c]);
    }
    if (FEW || wave == 0) put_row<T, D, CODES>(a, x.v, x.l, b, w.start + i, h * a.gqa + r - i * a.gqa, keys_seen(a, w, i));
    if (!FEW) __syncthreads();
  }
}

template <class T, int D, int RT, bool CODES>
int launch_rows(const AttnArgs& a, int workgroups, int most_rows, hipStream_t s) {
  hipLaunchKernelGGL((rows_kernel<T, D, RT, CODES>), dim3((unsigned)workgroups), dim3(kAttnThreads), 0, s, a);
  const int st = check_launch("paged_attention");
  if (st || a.whole) return st;
  const unsigned x = (unsigned)(a.s.B * a.Hk), y = (unsigned)std::min(most_rows, 16 * RT);      // more rows: a loop
  if (workgroups <= 8 * (long)x)                                 // parts of a row, on the average
    hipLaunchKernelGGL((join_kernel<T, D, RT, CODES, true>), dim3(x, (y + kWaves - 1) / kWaves), dim3(kAttnThreads), 0, s, a, workgroups);
  else hipLaunchKernelGGL((join_kernel<T, D, RT, CODES, false>), dim3(x, y), dim3(kAttnThreads), 0, s, a, workgroups);
  return check_launch("paged_attention(join)");
}

// Each (element type, head dim) in its own translation unit
template <class T, int D>
int launch(const AttnArgs& a, int rt, bool codes, int workgroups, int most_rows, hipStream_t s);

#define DSPARK_PAGED_ATTN(T, D)                                                                                       \
  template <>                                                                                                        \
  int launch<T, D>(const AttnArgs& a, int rt, bool codes, int workgroups, int most_rows, hipStream_t s)
DSPARK_PAGED_ATTN(BF16, 64);
DSPARK_PAGED_ATTN(BF16, 128);
DSPARK_PAGED_ATTN(BF16, 256);
DSPARK_PAGED_ATTN(F16, 64);
DSPARK_PAGED_ATTN(F16, 128);
DSPARK_PAGED_ATTN(F16, 256);

template <class T, int D>
int launch_rt(const AttnArgs& a, int rt, bool codes, int workgroups, int most_rows, hipStream_t s) {
#define DSPARK_ROWS(RT) \
  (codes ? launch_rows<T, D, RT, true>(a, workgroups, most_rows, s) : launch_rows<T, D, RT, false>(a, workgroups, most_rows, s))
  if constexpr (D <= 128) {
    if (rt == 4) return DSPARK_ROWS(4);
  }
  return rt >= 2 ? DSPARK_ROWS(2) : DSPARK_ROWS(1);
#undef DSPARK_ROWS
}

}  // namespace paged
}  // namespace dspark
