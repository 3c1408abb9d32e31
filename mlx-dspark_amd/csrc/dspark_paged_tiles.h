// Attention over paged caches for gfx950: many rows of each sequence (prompt chunks).
//
// The same attention as dspark_paged_attn.h, bound by the matrix cores and, close behind, by the softmax's instructions.
// Hence, as for prompts over contiguous caches:
//   * a workgroup of 4 waves takes 128 rows of a (sequence, KV head), (token, query head) heads fastest, 32 a wave, so
//     that 64 keys and values in LDS serve them all; S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16, where the scores
//     of a lane (32 keys of one row) are, in place, what the second product needs;
//   * K and V tiles are double buffered, one barrier a tile; each wave brings 16 positions, which lie in one page: pages of
//     the model's type go to LDS without passing registers, 8-bit codes through registers, where they are turned into the
//     model's type once for the workgroup;
//   * sequences of unequal lengths: those with more keys than one to one and a half times the average share of a workgroup
//     slot are split along the keys, into parts that a second launch joins (fp32, in the order of the keys).
//     Everything is found on the device from the lengths as they are;
//   * items with many keys first: sequences by their length, long causal tiles first within one. Consecutive items are a
//     tile's KV heads, which go to consecutive XCDs: with 8 heads each XCD's L2 has the pages of one.
// Probabilities are two pieces of the type, as in dspark_paged_attn.h: the second costs a third of the products, and one
// bf16 piece alone would add an error of the size of the output's own rounding. Codes of a page with a scale of 2^-25 to 2^-3
// (values up to 56) are fp16 numbers when multiplied by 2^10, and one fp16 piece of a probability is off by an eighth of a bf16
// rounding (2^-11 of it; one 2^21 under the reference is subnormal there, and off by 2^-32 of the reference): so 8-bit pages of
// bf16 models go to LDS as fp16 and take one product, and a workgroup that comes to a page that does not fit begins again with
// two bf16 pieces (seven chunks of 1 to 700 rows: 182 -> 165 us; with values past 56 throughout 101 -> 117 in seven others, with one
// page of zeros, whose scale is 2^-110, in one sequence of them 126). Pages that are not there begin again too. For bf16 pages
// what the conversion costs is what the products save.
//
// The running maximum is only raised (and the outputs rescaled) where it grew by more than 2^8: fp32 sums do not mind
// probabilities up to 2^8, and with 32 rows a wave some row's maximum moves in most tiles.
// 2048 rows behind 2953 keys, 32 / 8 heads of 128, bf16: 196 us (680 TFLOP/s of the two products, 1020 with the pieces); seven
// chunks of 1 to 700 rows over 8-bit pages, 16 / 4 heads of 128: 130 us; six verify blocks of 18 to 96 rows of a KV head behind
// 1500 to 10007 fp16 positions, 24 / 4 heads of 256: 154 MB in 56 us with what joins them (4 more when waves without rows
// multiplied too). Tried and not kept: two groups of four waves in a workgroup, one in its products while the other is in its
// softmax, a barrier between the phases (198 -> 234 us: as many cycles a tile, and lengths that fit together worse).
#pragma once

#include "dspark_attn_prefill.h"
#include "dspark_paged_attn.h"

namespace dspark {
namespace paged {

constexpr int kTileRows = 128;    // rows of a workgroup
constexpr int kTileKeys = 64;
template <int D>
constexpr int kSlots = D == 256 ? 256 : 512;     // workgroups that run together: two a CU, at head dim 256 one
constexpr int kParts = 704;       // parts of split sequences, at most: 2 * 512 / 1.5 and what rounding adds
constexpr int kLeastTiles = 8;    // key tiles of a part, at least

constexpr int kAluMayCross = 0x2 | 0x4;     // of a scheduling barrier: vector and scalar arithmetic

typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct TileArgs {
  AttnArgs a;                     // rows_up_to: sequences with more rows of a KV head are these kernels'
  float* opart;                   // [part][128 rows][D], unnormalised; then maxima and sums
  float* mpart;
};

struct TileWork {
  int start, n, len, full, rows, row_tiles, key_tiles;
};

__device__ __forceinline__ TileWork tile_work(const AttnArgs& a, int b) {
  const Seq q = sequence(a.s, b);
  TileWork w{q.start, q.n, q.len, q.full, q.n * a.gqa, 0, (q.len + kTileKeys - 1) / kTileKeys};
  if (w.rows <= a.rows_up_to) w.rows = 0;
  w.row_tiles = (w.rows + kTileRows - 1) / kTileRows;
  return w;
}

// The list of items: how many key tiles a part may have, and what every sequence has. That of the first 64 is looked up
// once, a lane each.
template <int D>
struct TileList {
  const AttnArgs& a;
  TileWork first;
  // Key tiles that a part may have: 1.5 times the average share of a slot. With one workgroup a CU (head dim 256) the least
  // from the share on with which all items run together, if that is less: six verify blocks of 18 to 96 rows 66.7 -> 62.4 us
  // (with two a CU, where a lone one runs faster, seven chunks lose 8% by it)
  int target;

  __device__ __forceinline__ explicit TileList(const AttnArgs& args) : a(args), first(tile_work(args, min((int)__lane_id(), args.s.B - 1))) {
    const int lane = __lane_id();
    float sum = 0.f;              // a rule, not a count: rounding does not matter
    for (int b = lane; b < a.s.B; b += 64) {
      const TileWork w = lanes(b);
      sum += (float)w.row_tiles * (float)w.key_tiles;
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2) sum += shfl_xor(sum, x);
    const float share = sum * (float)a.Hk / kSlots<D>;
    auto whole = [](float t) { return t < kLeastTiles ? kLeastTiles : t > 1e9f ? 1000000000 : (int)t + 1; };
    target = whole(1.5f * share);
    if (D == 256 && a.s.B <= 64) {
      const int mine = whole((1.f + (float)lane / 128.f) * share);       // a lane's try
      const float inv = 1.f / (float)mine;
      float items = 0.f;
      for (int b = 0; b < a.s.B; ++b)
        items += (float)__builtin_amdgcn_readlane(first.row_tiles, b) *
                 __builtin_ceilf((float)__builtin_amdgcn_readlane(first.key_tiles, b) * inv - 1e-6f);
      const unsigned long long fit = __builtin_amdgcn_ballot_w64(items * (float)a.Hk <= (float)kSlots<D>);
      if (fit) target = __builtin_amdgcn_readlane(mine, __builtin_ctzll(fit));
    }
    target = uniform(target);
  }
  __device__ __forceinline__ TileWork lanes(int b) const {   // of sequence b = 64 i + lane
    if (b < 64) return first;
    return tile_work(a, min(b, a.s.B - 1));
  }
  __device__ __forceinline__ TileWork at(int b) const {      // b: the wave's
    const TileWork w = b < 64 ? first : tile_work(a, b);
    const int l = b < 64 ? b : 0;
    auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
    return TileWork{of(w.start), of(w.n), of(w.len), of(w.full), of(w.rows), of(w.row_tiles), of(w.key_tiles)};
  }
  __device__ __forceinline__ int parts(const TileWork& w) const { return (w.key_tiles + target - 1) / target; }
  // Items of the list (and of the split ones among them) of a sequence
  __device__ __forceinline__ u32 items(int b) const {
    if (b >= a.s.B) return 0;
    const TileWork w = lanes(b);
    const unsigned long long n = (unsigned long long)a.Hk * (unsigned)w.row_tiles * (unsigned)parts(w);
    return n > kMostUnits ? kMostUnits + 1 : (u32)n;
  }
  __device__ __forceinline__ u32 split_items(int b) const { return b < a.s.B && parts(lanes(b)) > 1 ? items(b) : 0u; }
  __device__ __forceinline__ u32 all() const {
    u32 n = 0;
    for (int b0 = 0; b0 < a.s.B; b0 += 64) n = __builtin_elementwise_add_sat(n, items(b0 + (int)__lane_id()));
    return (u32)__builtin_amdgcn_readlane((int)wave_scan(n), 63);
  }
  // Parts before sequence b among the split sequences
  __device__ __forceinline__ int parts_before(int b) const {
    const int lane = __lane_id();
    u32 n = 0;
    for (int b0 = 0; b0 < b; b0 += 64)
      if (b0 + lane < b) n = __builtin_elementwise_add_sat(n, split_items(b0 + lane));
    const u32 sum = (u32)__builtin_amdgcn_readlane((int)wave_scan(n), 63);
    return (int)(sum > (u32)kParts ? (u32)kParts : sum);
  }
  // The sequence of the item, and its place among the sequence's, where sequences (64 at a time) stand in the order of
  // the keys that their items have, most first
  __device__ __forceinline__ bool locate(u32 item, int& b, int& local) const {
    const int lane = __lane_id();
    for (int b0 = 0; b0 < a.s.B; b0 += 64) {
      const int n = min(64, a.s.B - b0);
      const u32 count = items(b0 + lane);
      const TileWork w = lanes(b0 + lane);
      const int keys = lane < n ? w.key_tiles / max(parts(w), 1) : -1;
      int rank = 0;
      for (int j = 0; j < n; ++j) {
        const int k = __builtin_amdgcn_readlane(keys, j);
        rank += k > keys || (k == keys && j < lane) ? 1 : 0;
      }
      rank = lane < n ? rank : lane;
      const u32 c = (u32)__builtin_amdgcn_ds_permute(rank << 2, (int)count);
      const int from = __builtin_amdgcn_ds_permute(rank << 2, lane);
      const u32 upto = wave_scan(c);
      const u32 sum = (u32)__builtin_amdgcn_readlane((int)upto, 63);
      if (item < sum) {
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > item));
        b = uniform(b0 + __builtin_amdgcn_readlane(from, at));
        local = uniform((int)(item - (u32)__builtin_amdgcn_readlane((int)(upto - c), at)));
        return true;
      }
      item -= sum;
    }
    return false;
  }
};

// 16 bytes a lane from `base` + `off` to LDS, the wave's 1 KB from `to` on. In assembly, and waited for by hand: the
// compiler takes every later LDS read for one of these bytes and would have it wait for the copies just begun.
__device__ __forceinline__ void copy_to_lds(const char* base, u32 off, u16* to) {
  typedef __attribute__((address_space(3))) u16 lds_u16;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(base), "s"((u32)(uintptr_t)(lds_u16*)to)
               : "memory", "m0");
}

constexpr int kNarrow = 10;       // what codes are multiplied by as fp16: 2^10

// Eight probabilities as fp16
__device__ __forceinline__ u32x4_t one_piece(const f32x16_t& p, int r0) {
  u32x4_t o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = attn::pack2<F16>(p[r0 + 2 * i], p[r0 + 2 * i + 1]);
  return o;
}

// Eight probabilities as two pieces of T whose sum they are: the upper one cut off, so that both are positive
template <class T>
__device__ __forceinline__ void two_pieces(const f32x16_t& p, int r0, u32x4_t& hi, u32x4_t& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = p[r0 + 2 * i], b = p[r0 + 2 * i + 1];
    if constexpr (T::kF16) {
      const attn::f16x2_t h = __builtin_bit_cast(attn::f16x2_t, __builtin_amdgcn_cvt_pkrtz(a, b));
      const float m1 = __builtin_bit_cast(float, opaque_sgpr(0xBF800000u));     // keeps it one v_fma_mix
      hi[i] = __builtin_bit_cast(u32, h);
      lo[i] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)h.x, m1, a), __builtin_fmaf((float)h.y, m1, b)));
    } else {
      const u32 x = __builtin_bit_cast(u32, a), y = __builtin_bit_cast(u32, b);
      hi[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
      lo[i] = pack_bf16x2(a - __builtin_bit_cast(float, x & 0xFFFF0000u), b - __builtin_bit_cast(float, y & 0xFFFF0000u));
    }
  }
}

template <int D>
struct TileLds {
  u16 kv[2][2][kTileKeys * D];    // [buffer][K, V]
  u32 fits[2][4];                 // V of 16 positions fits fp16
  float rest[2][4];               // of fp16 models: key_rest of 16 positions
};

struct TileItem {
  TileWork w;
  int b, local, parts;            // its sequence, its place among the sequence's items, parts of a row tile
};

// The workgroup's item of the list
template <int D>
__device__ __forceinline__ bool find_item(const AttnArgs& a, TileItem& it) {
  const TileList<D> list(a);
  const u32 all = list.all();
  if (all > kMostUnits) return false;
  // Of the 512 that start together, two a CU, the second 256 in turned order: a long causal tile shares its CU with a
  // short one (2048 rows behind 2953 keys: 193.4 -> 191.6 us). At head dim 256 a CU has one, and the second 256 only start with
  // their shortest; that order was not measured
  const u32 nth = blockIdx.x >> 3, rounds = (all + 7) / 8;
  const u32 turned = nth / 32 == 1 && rounds > 32 ? 32 + min(63u, rounds - 1) - nth : nth;
  const u32 item = turned * 8 + (blockIdx.x & 7);
  if (nth >= rounds || item >= all) return false;
  if (!list.locate(item, it.b, it.local)) return false;
  it.w = list.at(it.b);
  it.parts = list.parts(it.w);
  return true;
}

// A workgroup's item; false if it was given up at a tile whose V does not fit fp16. `again`: rows of the wave that plain_rows
// has to compute
template <class T, int D, bool CODES, bool FP16>
__device__ __forceinline__ bool take_item(const TileArgs& ta, TileLds<D>& lds, u32& again) {
  using prefill::k_swz;
  using prefill::lds_tr;
  using prefill::mfma32;
  using prefill::v_swz;
  constexpr int KT = kTileKeys, SUB = KT / 32, CH = D / 8, ND = D / 32, NK = D / 16;
  constexpr int NJ = 16 * CH / 64;                           // 16-byte pieces of T that a lane brings of 16 positions
  constexpr int CJ = CODES ? D / 64 : 1;                     // of codes
  constexpr float kTop = 7.f;                                // probabilities times 2^7: up to 2^15
  constexpr float kUnscale = FP16 ? 1.f / (1 << kNarrow) : 1.f;
  auto& sm = lds.kv;
  auto& fits = lds.fits;
  const AttnArgs& a = ta.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int l31 = lane & 31, half = lane >> 5, l16 = lane & 15;

  TileItem it;
  if (!find_item<D>(a, it)) return true;
  const TileWork& w = it.w;
  const int b = it.b, parts = it.parts, z = it.local % parts, h = it.local / parts % a.Hk, tile = w.row_tiles - 1 - it.local / (parts * a.Hk);

  const int r0 = tile * kTileRows, rw = r0 + 32 * wave;
  const int r = min(rw + l31, w.rows - 1), tok = r / a.gqa, head = h * a.gqa + (r - tok * a.gqa);
  // keys that this lane's row sees, the wave's least and most, the workgroup's most
  const int lim = keys_seen(a, w, tok);
  const int wmin = uniform(keys_seen(a, w, min(rw, w.rows - 1) / a.gqa));
  const int wmax = rw < w.rows ? uniform(keys_seen(a, w, min(rw + 31, w.rows - 1) / a.gqa)) : 0;      // (none for a wave without rows)
  const int bmax = uniform(keys_seen(a, w, min(r0 + kTileRows - 1, w.rows - 1) / a.gqa));
  const int ntile = (bmax + KT - 1) / KT;
  const int t0 = (int)((long)ntile * z / parts), t1 = (int)((long)ntile * (z + 1) / parts);

  // page ids (and scales), 64 at a time
  const int* const row = a.s.table + b * a.s.ldt;
  const int last_page = (w.len - 1) >> a.s.log2P;
  int ids = -1, ids_at = -(1 << 30);
  bool whole_window = true;
  float ku = 1.f, vu = 1.f;
  auto fetch_ids = [&](int first) {
    ids_at = first;
    const int p = first + lane;
    const int id = p <= last_page ? row[p] : 0;
    ids = (unsigned)id < (unsigned)a.s.pool ? id : -1;
    whole_window = __builtin_amdgcn_ballot_w64(ids < 0) == 0;
    if constexpr (CODES) {
      ku = vu = 0.f;
      if (ids >= 0) {
        ku = scale_of(a.k.exps[ids * a.k.epage + h * a.k.ehead]);
        vu = scale_of(a.v.exps[ids * a.v.epage + h * a.v.ehead]);
      }
    }
  };
  auto window = [&](int t) {      // pages of tile t are in the window
    const int p0 = (t * KT) >> a.s.log2P, p1 = (t * KT + KT - 1) >> a.s.log2P;
    if (p0 < ids_at || p1 >= ids_at + 64) fetch_ids(p0);
  };

  // This wave's 16 positions of tile t: rows past the keys repeat the last one (and are masked)
  constexpr int ES = CODES ? 1 : 2;
  u32x4_t kc[CJ], vc[CJ];         // codes in flight
  float kc_unit = 1.f, vc_unit = 1.f;
  const char* v_at = nullptr;     // of the positions whose keys were brought last, and its last row
  int rmax = 0;
  auto bring_k = [&](int t, int buf) {
    window(t);
    const int pos = min(t * KT + 16 * wave, (w.len - 1) & ~15);
    rmax = min(15, w.len - 1 - pos);
    const int p = (pos >> a.s.log2P) - ids_at, id = max(__builtin_amdgcn_readlane(ids, p), 0);
    const long in = pos & (a.s.P - 1);
    const char* kp = a.k.data + (id * a.k.page + h * a.k.head + in * a.k.row) * ES;
    v_at = a.v.data + (id * a.v.page + h * a.v.head + in * a.v.row) * ES;
    if constexpr (CODES) {
#pragma unroll
      for (int j = 0; j < CJ; ++j) {
        const int i = j * 64 + lane, rr = i / (D / 16), c = i % (D / 16);
        kc[j] = ldg128(kp + min(rr, rmax) * (int)a.k.row + 16 * c);
      }
      auto unit = [&](float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), p)); };
      kc_unit = unit(ku);
      vc_unit = unit(vu);
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int i = j * 64 + lane, rr = i / CH;
        const u32 off = __umul24((u32)min(rr, rmax), (u32)a.k.row * 2) + (u32)((i % CH ^ k_swz<D>(16 * wave + rr)) << 4);    // < 2^28
        copy_to_lds(kp, off, &sm[buf][0][16 * wave * D + j * 512]);
      }
    }
  };
  auto bring_v = [&](int buf) {
    if constexpr (CODES) {
#pragma unroll
      for (int j = 0; j < CJ; ++j) {
        const int i = j * 64 + lane, rr = i / (D / 16), c = i % (D / 16);
        vc[j] = ldg128(v_at + min(rr, rmax) * (int)a.v.row + 16 * c);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int i = j * 64 + lane, rr = i / CH;
        const u32 off = __umul24((u32)min(rr, rmax), (u32)a.v.row * 2) + (u32)((i % CH ^ v_swz<D>(16 * wave + rr)) << 4);
        copy_to_lds(v_at, off, &sm[buf][1][16 * wave * D + j * 512]);
      }
    }
  };
  // What passes registers goes to LDS
  auto put = [&](int buf) {
    if constexpr (CODES) {
#pragma unroll
      for (int j = 0; j < CJ; ++j) {
        const int i = j * 64 + lane, rr = 16 * wave + i / (D / 16), c = 2 * (i % (D / 16));
        u32x4_t lo, hi;
        decode<T>(kc[j], key_unit<T>(kc_unit), lo, hi);
        *reinterpret_cast<u32x4_t*>(&sm[buf][0][rr * D + ((c ^ k_swz<D>(rr)) << 3)]) = lo;
        *reinterpret_cast<u32x4_t*>(&sm[buf][0][rr * D + (((c + 1) ^ k_swz<D>(rr)) << 3)]) = hi;
        if constexpr (FP16) decode<F16>(vc[j], vc_unit * (1 << kNarrow), lo, hi);
        else decode<T>(vc[j], vc_unit, lo, hi);
        *reinterpret_cast<u32x4_t*>(&sm[buf][1][rr * D + ((c ^ v_swz<D>(rr)) << 3)]) = lo;
        *reinterpret_cast<u32x4_t*>(&sm[buf][1][rr * D + (((c + 1) ^ v_swz<D>(rr)) << 3)]) = hi;
      }
      // codes are up to 448 in size and multiples of 2^-9
      if (FP16 && lane == 0) fits[buf][wave] = vc_unit <= 0.125f && vc_unit >= 1.f / (1 << 25);
      if (T::kF16 && lane == 0) lds.rest[buf][wave] = key_rest<T>(kc_unit);
    }
  };

  if (t0 < t1) {
    bring_k(t0, 0);
    bring_v(0);
  }
  u32x4_t qf[NK];
  const u16* qp = a.q + (w.start + tok) * a.qrow + head * a.qhead + 8 * half;
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) qf[kk] = ldg128(qp + 16 * kk);
  // vmcnt(0): the queries are here, or their first use, in the loop, would wait for a tile's copies in every round
  __builtin_amdgcn_s_waitcnt(0x0F70);
  __builtin_amdgcn_sched_barrier(0);

  f32x16_t o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  const float c = a.scale_log2;
  float m = kLowest, mc = -1e30f, l = 0.f;                   // reference of the exponents: raw, and times c; this half's sum
  const int kswz = k_swz<D>(l31), kbase = l31 * D;
  const int vrow = 4 * half + (l16 >> 2), vswz = v_swz<D>(l16 >> 2);
  const int vchunk = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1), vbase = vrow * D + 4 * (l16 & 1);

  if (t0 < t1) put(0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    // tile t has landed once every wave's copies have; every read of the other buffer is done
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    u32 gone = 0;                                            // 16-position groups of this tile in pages that are not there
    if (!whole_window) {
      window(t);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = (t * KT + 16 * i) >> a.s.log2P;
        if (p <= last_page && __builtin_amdgcn_readlane(ids, p - ids_at) < 0) gone |= 1u << i;
      }
    }
    const int key0 = t * KT;
    if constexpr (FP16) {
      const u32x4_t f = *reinterpret_cast<const u32x4_t*>(fits[buf]);
      if (!uniform((int)(f.x & f.y & f.z & f.w))) return false;
    }
    if (t + 1 < t1) bring_k(t + 1, buf ^ 1);
    if (key0 >= wmax) {                                      // wave-uniform
      if (t + 1 < t1) bring_v(buf ^ 1);
    } else {
      const u16* ks = sm[buf][0];
      const u16* vs = sm[buf][1];
      f32x16_t s[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
      // K operands are asked for KA steps ahead of their products, V operands of DB column blocks one (left to itself the
      // compiler reads one and waits for it). Two of each at head dim 256, where what is past 256 registers moves between two
      // files (513 rows behind 2462 positions: 87.6 -> 84.5 us)
      constexpr int KA = D == 256 ? 2 : NK < 4 ? NK : 4;
      u32x4_t kf[KA][SUB];
      auto read_k = [&](int kk) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
          kf[kk % KA][u] = *reinterpret_cast<const u32x4_t*>(ks + u * 32 * D + kbase + (((2 * kk + half) ^ kswz) << 3));
      };
#pragma unroll
      for (int kk = 0; kk < KA; ++kk) read_k(kk);
      __builtin_amdgcn_sched_barrier(kAluMayCross);
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) s[u] = mfma32<T>(kf[kk % KA][u], qf[kk], s[u]);
        if (kk + KA < NK) read_k(kk + KA);
        __builtin_amdgcn_sched_barrier(kAluMayCross);
      }
      if constexpr (CODES && T::kF16) {
        const u32x4_t f = *reinterpret_cast<const u32x4_t*>(lds.rest[buf]);
        const int one = __builtin_bit_cast(int, 1.f);
        const int f0 = uniform((int)f.x), f1 = uniform((int)f.y), f2 = uniform((int)f.z), f3 = uniform((int)f.w);
        if (f0 != one || f1 != one || f2 != one || f3 != one) {
#pragma unroll
          for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i)                     // (positions 16 (2 u + i / 8) ..)
              s[u][i] *= __builtin_bit_cast(float, u ? i < 8 ? f2 : f3 : i < 8 ? f0 : f1);
        }
      }
      if (t + 1 < t1) bring_v(buf ^ 1);             // (its registers are free now)
      auto v_frag = [&](int uj, int d) {                     // V^T of keys 16 uj .. 16 uj + 15, columns 32 d ..
        const u16* vp = vs + 16 * uj * D + vbase + (((4 * d + vchunk) ^ vswz) << 3);
        const u32x2_t lo = lds_tr(vp), hi = lds_tr(vp + 8 * D);
        return u32x4_t{lo.x, lo.y, hi.x, hi.y};
      };
      constexpr int DB = D == 256 ? 2 : ND < 4 ? ND : 4, NG = 2 * SUB * (ND / DB);    // V operands of a step, steps
      u32x4_t vf[2][DB];
      auto read_v = [&](int g) {
#pragma unroll
        for (int d = 0; d < DB; ++d) vf[g & 1][d] = v_frag(g / (ND / DB), g % (ND / DB) * DB + d);
      };
      read_v(0);
      __builtin_amdgcn_sched_barrier(kAluMayCross);
      if (key0 + KT > wmin || gone) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int k = 32 * u + 8 * (i >> 2) + 4 * half + (i & 3);
            if (key0 + k >= lim || (gone >> (k >> 4) & 1)) s[u][i] = -__builtin_inff();
          }
      }
      float mx = s[0][0];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
      mx = max_xor32(mx);
      // (the first keys that a row sees raise it from its lowest)
      if (__builtin_amdgcn_ballot_w64(mx > m && __builtin_fmaf(mx, c, -mc) > 8.f)) {
        const float to = fmaxf(m, mx), toc = to == kLowest ? -1e30f : to * c;
        const float alpha = __builtin_amdgcn_exp2f(mc - toc);
        m = to;
        mc = toc;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
      }
      const float up = kTop - mc;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], c, up));
          s[u][i] = p;
          sum += p;
        }
      l += sum;
      u32x4_t ph, pl;
      if constexpr (FP16) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const int uj = g / (ND / DB), d0 = g % (ND / DB) * DB;
          if (g + 1 < NG) read_v(g + 1);
          __builtin_amdgcn_sched_barrier(kAluMayCross);
          if (d0 == 0) ph = one_piece(s[uj >> 1], 8 * (uj & 1));
#pragma unroll
          for (int d = 0; d < DB; ++d) o[d0 + d] = mfma32<F16>(vf[g & 1][d], ph, o[d0 + d]);
        }
      } else {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const int uj = g / (ND / DB), d0 = g % (ND / DB) * DB;
          if (g + 1 < NG) read_v(g + 1);
          __builtin_amdgcn_sched_barrier(kAluMayCross);
          if (d0 == 0) two_pieces<T>(s[uj >> 1], 8 * (uj & 1), ph, pl);
#pragma unroll
          for (int d = 0; d < DB; ++d) o[d0 + d] = mfma32<T>(vf[g & 1][d], ph, o[d0 + d]);
#pragma unroll
          for (int d = 0; d < DB; ++d) o[d0 + d] = mfma32<T>(vf[g & 1][d], pl, o[d0 + d]);
        }
      }
    }
    if (t + 1 < t1) put(buf ^ 1);
  }

  l += shfl_xor(l, 32);
  const bool own = rw + l31 < w.rows;
  if (parts > 1) {
    const int part = TileList<D>(a).parts_before(b) + it.local;   // (kept from the start, the list costs registers)
    if (part >= kParts || !own) return true;
    const long pr = (long)part * kTileRows + 32 * wave + l31;
    if (half == 0) {
      ta.mpart[2 * pr] = mc;
      ta.mpart[2 * pr + 1] = l;
    }
    float* op = ta.opart + pr * D + 4 * half;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4_t*>(op + 32 * d + 8 * g) =
            f32x4_t{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]} * kUnscale;
    return true;
  }
  const float inv = l > 0.f ? kUnscale / l : 0.f;
  float zero = l > 0.f || lim == 0 ? l - l : 1.f;            // NaN once an output is not finite
  if (own) {
    u16* op = a.out + (w.start + tok) * a.orow + head * a.ohead + 4 * half;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
#pragma unroll
        for (int i = 0; i < 4; ++i) zero = __builtin_fmaf(o[d][4 * g + i], 0.f, zero);
        *reinterpret_cast<u32x2_t*>(op + 32 * d + 8 * g) =
            u32x2_t{attn::pack2<T>(o[d][4 * g] * inv, o[d][4 * g + 1] * inv),
                    attn::pack2<T>(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv)};
      }
  }
  const unsigned long long bad = __builtin_amdgcn_ballot_w64(own && zero != 0.f);
  again = (u32)bad | (u32)(bad >> 32);
  return true;
}

// Rows of the wave again, in plain fp32. The item is found anew: kept, what this needs would cost registers in take_item's loop
template <class T, int D, bool CODES>
__device__ __forceinline__ void plain_rows(const AttnArgs& a, u32 rows) {
  TileItem it;
  if (!find_item<D>(a, it)) return;
  const int h = it.local / it.parts % a.Hk, tile = it.w.row_tiles - 1 - it.local / (it.parts * a.Hk);
  const int rw = tile * kTileRows + 32 * uniform((int)threadIdx.x >> 6);
  __threadfence_block();
  for (; rows; rows &= rows - 1) {
    const int i = rw + __builtin_ctz(rows), ti = i / a.gqa;
    plain_row<T, D, CODES>(a, it.b, it.w.start + ti, h * a.gqa + i - ti * a.gqa, keys_seen(a, it.w, ti));
  }
}

template <class T, int D, bool CODES>
__global__ __launch_bounds__(kAttnThreads, D == 256 ? 1 : 2) void tiles_kernel(const TileArgs ta) {
  __shared__ __attribute__((aligned(16))) TileLds<D> lds;
  if (ta.a.clear) clear_rows<D>(ta.a);
  u32 again = 0;
  // (At head dim 256 the two paths together are past the registers of one wave)
  if constexpr (CODES && !T::kF16 && D <= 128) {
    if (!take_item<T, D, CODES, true>(ta, lds, again)) {
      __syncthreads();            // every wave has read what does not fit
      asm volatile("" ::: "memory");
      take_item<T, D, CODES, false>(ta, lds, again);
    }
  } else {
    take_item<T, D, CODES, false>(ta, lds, again);
  }
  if (again) plain_rows<T, D, CODES>(ta.a, again);
}

// Joins the parts of split sequences; a wave a row
template <class T, int D, bool CODES>
__global__ __launch_bounds__(kAttnThreads) void join_tiles_kernel(const TileArgs ta) {
  constexpr int C = D / 64;
  const AttnArgs& a = ta.a;
  const int lane = __lane_id(), wave = uniform((int)(threadIdx.x >> 6));
  const TileList<D> list(a);
  if (list.all() > kMostUnits) return;
  int base = 0;                   // parts before sequence b0
  for (int b0 = 0; b0 < a.s.B && base < kParts; b0 += 64) {
    // a lane has a sequence's parts and rows, and those before
    const TileWork w = list.lanes(b0 + lane);
    const u32 count = list.split_items(b0 + lane), rows = count ? (u32)a.Hk * (u32)w.rows : 0u;
    const u32 upto = wave_scan(count), rows_upto = wave_scan(rows);
    const u32 all = (u32)__builtin_amdgcn_readlane((int)rows_upto, 63);
    for (u32 x = blockIdx.x * kWaves + wave; x < all; x += gridDim.x * kWaves) {
      const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(rows_upto > x)), b = b0 + l;
      auto of = [&](u32 y) { return __builtin_amdgcn_readlane((int)y, l); };
      const long before = (long)base + (u32)of(upto - count);
      if (before + (u32)of(count) > kParts) break;
      const TileWork v = TileWork{of(w.start), of(w.n), of(w.len), of(w.full), of(w.rows), of(w.row_tiles), of(w.key_tiles)};
      const int parts = list.parts(v), i = (int)(x - (u32)of(rows_upto - rows)), h = i / v.rows, r = i - h * v.rows;
      const int tile = r / kTileRows, at = r - tile * kTileRows;
      const int first = (int)before + ((v.row_tiles - 1 - tile) * a.Hk + h) * parts;
      const Joined<C> y = join_parts<D, 4>(ta.opart, ta.mpart, 1, 1.f, parts, 0, 1,
                                           [&](int z) { return (long)(first + z) * kTileRows + at; },
                                           [&](int z) { return 2 * ((long)(first + z) * kTileRows + at); });
      const int tok = r / a.gqa;
      put_row<T, D, CODES>(a, y.v, y.l, b, v.start + tok, h * a.gqa + r - tok * a.gqa, keys_seen(a, v, tok));
    }
    const u32 sum = (u32)__builtin_amdgcn_readlane((int)upto, 63);
    base = sum > (u32)(kParts - base) ? kParts : base + (int)sum;
  }
}

// Each (element type, head dim) in its own translation unit
template <class T, int D>
int launch_tiles(const TileArgs& ta, bool codes, unsigned items, hipStream_t s);

#define DSPARK_PAGED_TILES(T, D) \
  template <>                   \
  int launch_tiles<T, D>(const TileArgs& ta, bool codes, unsigned items, hipStream_t s)
DSPARK_PAGED_TILES(BF16, 64);
DSPARK_PAGED_TILES(BF16, 128);
DSPARK_PAGED_TILES(BF16, 256);
DSPARK_PAGED_TILES(F16, 64);
DSPARK_PAGED_TILES(F16, 128);
DSPARK_PAGED_TILES(F16, 256);

template <class T, int D, bool CODES>
int launch_tiles_of(const TileArgs& ta, unsigned items, hipStream_t s) {
  hipLaunchKernelGGL((tiles_kernel<T, D, CODES>), dim3(items), dim3(kAttnThreads), 0, s, ta);
  const int st = check_launch("paged_attention(tiles)");
  if (st) return st;
  hipLaunchKernelGGL((join_tiles_kernel<T, D, CODES>), dim3(2048), dim3(kAttnThreads), 0, s, ta);
  return check_launch("paged_attention(join tiles)");
}

}  // namespace paged
}  // namespace dspark
