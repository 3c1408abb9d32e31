// A step's rows into a paged cache, rotated to their positions on the way, and pages read back (gfx950).
//
// Rotation, of the pairs (i, i + half) or, interleaved, (2i, 2i + 1) of a head's first 2 half values:
//   a = position * f_i in fp64;  c, s = cos a, sin a times the factor, rounded to fp32;
//   y1 = x1 c - x2 s,  y2 = x1 s + x2 c: three fp32 operations, each rounded, then the model's type.
// cos and sin are taken in fp64 (a reduced by multiples of pi / 2 in two parts, Cody and Waite; then the Taylor series,
// which at pi / 4 is down to 2^-60 after nine terms), so that their fp32 values are the rounded true ones but for one in
// 2^25: a row has the same bits wherever it is rotated, and its 8-bit codes with it.
//
// 8-bit pages: E of a page and head is the least exponent with |x| <= 448 2^E for the finite values of the rows new in it,
// at least kLeastExp and the page's own where it holds rows of the sequence before them; codes are e4m3(x 2^-E), those
// of the earlier rows shifted where E grew. Infinities and NaN become NaN codes, and so does what is put behind rows of a NaN scale.
//
// Bound by bytes. Rows: a workgroup forms cos and sin of its row once in LDS for all heads. 8-bit pages: a workgroup a
// (page, KV head, keys or values), since the scale needs all its rows first; they wait in LDS. Its threads take the
// angles that they need themselves, as no other head shares them there (what rows become goes past the caches, 19.5 -> 19.0 us for the
// 2048 below; read past them too they took 18.4 there, but the chunks 20.2 with their read for 18.1); a page's chain of loads and angles is what takes
// the time of a step with fewer pages than the card has compute units (workgroups of 512 and 1024 threads shorten it by
// 15% there, and cost as much and more where there are many). bf16: one row of 32 / 8 heads of 128 3.5 us, 2048 rows of 64 / 8
// 19 us (4.4 TB/s); 8-bit pages, 48 single rows 5 us, chunks of 77 to 600 rows of 24 / 4 heads of 256 14 us.
#include <algorithm>

#include "dspark_paged.h"

// The rotation's products and sums stay separate roundings.
#pragma clang fp contract(off)

namespace dspark {
namespace paged {
namespace {

constexpr int kThreads = 256;

struct Rows {                    // [T, heads, D]; strides in elements
  const char* x;
  long row, head;
};

struct AppendArgs {
  Seqs s;
  Pages kp, vp;
  Rows q, k, v;
  char* qo;
  long qo_row, qo_head;
  int clear;                     // rows of no sequence: zeros in qo
  int Hq, Hk, D, half;           // half = 0: nothing is rotated
  const double* freqs;
  double scale;
  const void* pos;               // null: the positions that the rows are written to
  int pos64;
  long pstride;
  int page_blocks;               // workgroups of the pages, which come before those of the rows
  int parts;                     // workgroups of a row
};

template <int DT>
__device__ __forceinline__ float get(u32 v) {
  if constexpr (DT == DSPARK_DTYPE_F16) return (float)__builtin_bit_cast(_Float16, (u16)v);
  else return bf2f(v & 0xFFFFu);
}
template <int DT>
__device__ __forceinline__ u32 put(float v) {
  if constexpr (DT == DSPARK_DTYPE_F16) return __builtin_bit_cast(u16, (_Float16)v);
  else return f2bf(v);
}

// fp32(cos a), fp32(sin a), times the factor before the rounding
__device__ __forceinline__ float2 cos_sin(double a, double scale) {
  const double k = __builtin_rint(a * 0.63661977236758138);
  const double r = __builtin_fma(-k, 6.123233995736766e-17, __builtin_fma(-k, 1.5707963267948966, a));
  const double z = r * r;
  double s = 1.0 / 355687428096000.0, c = -1.0 / 6402373705728000.0;       // 1 / 17!, -1 / 18!
  constexpr double fs[] = {-1.0 / 1307674368000.0, 1.0 / 6227020800.0, -1.0 / 39916800.0, 1.0 / 362880.0, -1.0 / 5040.0,
                           1.0 / 120.0, -1.0 / 6.0};
  constexpr double fc[] = {1.0 / 20922789888000.0, -1.0 / 87178291200.0, 1.0 / 479001600.0, -1.0 / 3628800.0, 1.0 / 40320.0,
                           -1.0 / 720.0, 1.0 / 24.0, -0.5};
#pragma unroll
  for (int i = 0; i < 7; ++i) s = __builtin_fma(s, z, fs[i]);
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_fma(c, z, fc[i]);
  s = __builtin_fma(s * z, r, r);
  c = __builtin_fma(c, z, 1.0);
  const int quarter = (int)(k - 4.0 * __builtin_floor(k * 0.25));
  double cs = quarter & 1 ? s : c, sn = quarter & 1 ? c : s;
  cs = quarter == 1 || quarter == 2 ? -cs : cs;
  sn = quarter >= 2 ? -sn : sn;
  return make_float2((float)(cs * scale), (float)(sn * scale));
}

__device__ __forceinline__ long rotary_position(const AppendArgs& a, int t, long p) {
  if (!a.pos) return p;
  return a.pos64 ? static_cast<const int64_t*>(a.pos)[t * a.pstride] : (long)static_cast<const int32_t*>(a.pos)[t * a.pstride];
}

// Item c of a head's row, rotated: rotating items are 8 pairs (half layout: 8 values at d and 8 at d + half) or the 4
// pairs of 8 values (interleaved), the others 8 values as they are. Two or one 16-byte accesses.
struct Item {
  u32x4_t lo, hi;
  int d, d2;                     // d2 < 0: no second part
};

template <bool INTER>
__device__ __forceinline__ Item load_item(const AppendArgs& a, const u16* x, int c) {
  Item it;
  const int rot = INTER ? a.half / 4 : a.half / 8;
  it.d = c < rot ? 8 * c : 2 * a.half + 8 * (c - rot);
  it.d2 = !INTER && c < rot ? it.d + a.half : -1;
  it.lo = ldg128(x + it.d);
  if (it.d2 >= 0) it.hi = ldg128(x + it.d2);
  return it;
}

template <int DT, bool INTER, class F>
__device__ __forceinline__ void turn_item(const AppendArgs& a, Item& it, F turn) {
  if (INTER ? it.d >= 2 * a.half : it.d2 < 0) return;
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 cs = turn(it.d / 2 + i);
      const float u = get<DT>(it.lo[i]), v = get<DT>(it.lo[i] >> 16);
      it.lo[i] = put<DT>(u * cs.x - v * cs.y) | put<DT>(u * cs.y + v * cs.x) << 16;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32 y1[2], y2[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 cs = turn(it.d + 2 * i + j);
        const float u = get<DT>(it.lo[i] >> (16 * j)), v = get<DT>(it.hi[i] >> (16 * j));
        y1[j] = put<DT>(u * cs.x - v * cs.y);
        y2[j] = put<DT>(u * cs.y + v * cs.x);
      }
      it.lo[i] = y1[0] | y1[1] << 16;
      it.hi[i] = y2[0] | y2[1] << 16;
    }
  }
}

__device__ __forceinline__ void stg128_nt(void* p, u32x4_t v) { __builtin_nontemporal_store(v, static_cast<u32x4_t*>(p)); }
__device__ __forceinline__ void stg128(void* p, u32x4_t v) { *static_cast<u32x4_t*>(p) = v; }

// One row: its queries rotated, and into pages of the model's type its keys and values
template <int DT, bool INTER, bool KV>
__device__ __forceinline__ void append_row(const AppendArgs& a, float2* tab) {
  const int unit = blockIdx.x - a.page_blocks, t = unit / a.parts, part = unit - t * a.parts, lane = __lane_id();
  const int plain = a.D / 8, log_plain = __builtin_ctz(plain);
  const int rot = INTER ? a.half / 4 : a.half / 8, per = rot + (a.D - 2 * a.half) / 8;
  const int heads = a.Hq + (KV ? a.Hk : 0), turned = heads * per, all = turned + (KV ? a.Hk * plain : 0);
  // its sequence
  int b = -1, n0 = 0, n1 = 0;
  for (int b0 = 0; b0 < a.s.B && b < 0; b0 += 64) {
    const int i = min(b0 + lane, a.s.B - 1);
    const Seq q = sequence(a.s, i);
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(b0 + lane < a.s.B && q.n > 0 && t >= q.start && t < q.start + q.n);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      b = uniform(b0 + l);
      n0 = __builtin_amdgcn_readlane(q.start, l);
      n1 = __builtin_amdgcn_readlane(q.n, l);
    }
  }
  if (b < 0) {                   // a row of no sequence
    for (int i = part * kThreads + threadIdx.x; a.clear && i < a.Hq * plain; i += a.parts * kThreads)
      stg128(reinterpret_cast<u16*>(a.qo) + t * a.qo_row + (i >> log_plain) * a.qo_head + 8 * (i & (plain - 1)), u32x4_t{0u, 0u, 0u, 0u});
    return;
  }
  const long p = (long)a.s.lens[b] - n1 + (t - n0), rp = rotary_position(a, t, p);
  for (int i = threadIdx.x; i < a.half; i += kThreads) tab[i] = cos_sin((double)rp * a.freqs[i], a.scale);
  __syncthreads();
  const int id = KV ? page_of(a.s, b, p) : -1;
  const long off = p & (a.s.P - 1);
  for (int i = part * kThreads + threadIdx.x; i < all; i += a.parts * kThreads) {
    if (i < turned) {
      const int h = i / per, c = i - h * per;
      const bool key = h >= a.Hq;
      if (key && id < 0) continue;
      const Rows& r = key ? a.k : a.q;
      const int hs = key ? h - a.Hq : h;
      Item it = load_item<INTER>(a, reinterpret_cast<const u16*>(r.x) + t * r.row + hs * r.head, c);
      turn_item<DT, INTER>(a, it, [&](int j) { return tab[j]; });
      u16* y = key ? reinterpret_cast<u16*>(a.kp.data) + id * a.kp.page + hs * a.kp.head + off * a.kp.row
                   : reinterpret_cast<u16*>(a.qo) + t * a.qo_row + hs * a.qo_head;
      stg128_nt(y + it.d, it.lo);
      if (it.d2 >= 0) stg128_nt(y + it.d2, it.hi);
    } else if (id >= 0) {
      const int j = i - turned, h = j >> log_plain, c = j & (plain - 1);
      stg128_nt(reinterpret_cast<u16*>(a.vp.data) + id * a.vp.page + h * a.vp.head + off * a.vp.row + 8 * c,
             ldg128(reinterpret_cast<const u16*>(a.v.x) + t * a.v.row + h * a.v.head + 8 * c));
    }
  }
}

// Bits of the largest finite size among 8 values
template <int DT>
__device__ __forceinline__ u32 largest(u32x4_t v, u32 m) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u32 x = __builtin_bit_cast(u32, get<DT>(v[i] >> (16 * j))) & 0x7FFFFFFFu;
      m = x < 0x7F800000u && x > m ? x : m;
    }
  return m;
}

// 8 values times 2^-E as codes
template <int DT>
__device__ __forceinline__ u32x2_t codes8(u32x4_t v, float unit) {
  u32x2_t o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32 a = v[2 * i], b = v[2 * i + 1];
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(get<DT>(a) * unit, get<DT>(a >> 16) * unit, 0, false);
    o[i] = (u32)__builtin_amdgcn_cvt_pk_fp8_f32(get<DT>(b) * unit, get<DT>(b >> 16) * unit, c, true);
  }
  return o;
}

__device__ __forceinline__ u32 shift_codes(u32 c, float by) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  const int r = __builtin_amdgcn_cvt_pk_fp8_f32(lo.x * by, lo.y * by, 0, false);
  return (u32)__builtin_amdgcn_cvt_pk_fp8_f32(hi.x * by, hi.y * by, r, true);
}

// The rows new in one page of one KV head, keys or values
template <int DT, bool INTER>
__device__ __forceinline__ void append_page8(const AppendArgs& a, u16* stash, u32* joined) {
  const int item = blockIdx.x, kind = item & 1, h = (item >> 1) % a.Hk;
  int b, j;
  const auto count = [&](int i) {
    const Seq q = sequence(a.s, i);
    if (!q.n) return 0u;
    const long p0 = first_position(q), p1 = p0 + q.n;      // of the rows, their end
    return p1 <= 0 ? 0u : (u32)(((p1 - 1) >> a.s.log2P) - ((p0 < 0 ? 0 : p0) >> a.s.log2P) + 1);
  };
  if (!locate((u32)((item >> 1) / a.Hk), a.s.B, count, b, j)) return;
  const Seq q = sequence(a.s, b);
  const long p0 = first_position(q), base = (((p0 < 0 ? 0 : p0) >> a.s.log2P) + j) << a.s.log2P;
  const int id = page_of(a.s, b, base);
  if (id < 0) return;
  const int lo = (int)(p0 > base ? p0 - base : 0), hi = (int)(p0 + q.n < base + a.s.P ? p0 + q.n - base : a.s.P);
  const int t0 = q.start + (int)(base + lo - p0), rows = hi - lo;
  const Pages& pg = kind ? a.vp : a.kp;
  const Rows& src = kind ? a.v : a.k;
  unsigned char* ep = pg.exps + id * pg.epage + h * pg.ehead;
  const int half = kind ? 0 : a.half, D = a.D, log8 = __builtin_ctz(D / 8);
  const int rot = INTER ? half / 4 : half / 8, per = rot + (D - 2 * half) / 8;
  u32 m = 0;
  if (half) {
    const auto load = [&](int i) {
      const int r = i / per;
      return load_item<INTER>(a, reinterpret_cast<const u16*>(src.x) + (t0 + r) * src.row + h * src.head, i - r * per);
    };
    Item next = {};
    if ((int)threadIdx.x < rows * per) next = load(threadIdx.x);
    for (int i = threadIdx.x; i < rows * per;) {
      Item it = next;
      const int r = i / per;
      i += kThreads;
      if (i < rows * per) next = load(i);
      const double at = (double)rotary_position(a, t0 + r, base + lo + r);
      turn_item<DT, INTER>(a, it, [&](int f) { return cos_sin(at * a.freqs[f], a.scale); });
      m = largest<DT>(it.lo, m);
      stg128(stash + r * D + it.d, it.lo);
      if (it.d2 >= 0) {
        m = largest<DT>(it.hi, m);
        stg128(stash + r * D + it.d2, it.hi);
      }
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < rows << log8; i += kThreads) {
      const int r = i >> log8, c = i - (r << log8);
      const u32x4_t v = ldg128(reinterpret_cast<const u16*>(src.x) + (t0 + r) * src.row + h * src.head + 8 * c);
      m = largest<DT>(v, m);
      stg128(stash + 8 * i, v);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const u32 o = (u32)__builtin_amdgcn_ds_bpermute((__lane_id() ^ d) << 2, (int)m);
    m = o > m ? o : m;
  }
  if (__lane_id() == 0) joined[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) m = joined[i] > m ? joined[i] : m;
  // 448 = 1.75 2^8
  int e = max((int)(m >> 23) - 127 - 8 + ((m & 0x7FFFFFu) > 0x600000u ? 1 : 0), kLeastExp);
  const int old = lo ? (int)*ep - 127 : kLeastExp;
  e = max(e, old);
  const float unit = e > 127 ? __builtin_nanf("") : scale_of((u32)(127 - e));
  unsigned char* to = reinterpret_cast<unsigned char*>(pg.data) + id * pg.page + h * pg.head;
  for (int i = threadIdx.x; i < rows << log8; i += kThreads) {
    const int r = i >> log8, c = i - (r << log8);
    *reinterpret_cast<u32x2_t*>(to + (lo + r) * pg.row + 8 * c) = codes8<DT>(*reinterpret_cast<const u32x4_t*>(stash + 8 * i), unit);
  }
  if (lo && e > old) {
    const int by = old - e;
    const float f = by < -126 ? 0.f : scale_of((u32)(by + 127));
    for (int i = threadIdx.x; i < lo << (log8 - 1); i += kThreads) {
      const int r = i >> (log8 - 1), c = i - (r << (log8 - 1));
      u32x4_t* p = reinterpret_cast<u32x4_t*>(to + r * pg.row + 16 * c);
      u32x4_t v = *p;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = shift_codes(v[k], f);
      *p = v;
    }
  }
  __syncthreads();               // every wave has read the old exponent
  if (threadIdx.x == 0) *ep = (unsigned char)(e + 127);
}

template <int DT, bool INTER, bool CODES>
__global__ __launch_bounds__(kThreads) void append_kernel(const AppendArgs a) {
  extern __shared__ __attribute__((aligned(16))) char dynamic[];      // (cos, sin) pairs of a row, or a page's rows
  if constexpr (CODES) {
    __shared__ u32 joined[kThreads / 64];
    if ((int)blockIdx.x < a.page_blocks) {
      append_page8<DT, INTER>(a, reinterpret_cast<u16*>(dynamic), joined);
      return;
    }
  }
  append_row<DT, INTER, !CODES>(a, reinterpret_cast<float2*>(dynamic));
}

// Pages by id as dense values [N, Hk, P, D], zeros for ids that the pool does not have
struct ReadArgs {
  Pages side[2];
  u16* out[2];
  const int* ids;
  int N, Hk, P, D, pool;
  long items;                    // of 8 values, of one side
};

template <int DT, bool CODES>
__global__ __launch_bounds__(kThreads) void read_kernel(const ReadArgs a) {
  const Pages& pg = a.side[blockIdx.y];
  const int per_head = a.P * a.D / 8;
  for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < a.items; i += (long)gridDim.x * kThreads) {
    const long nh = i / per_head;
    const int in = (int)(i - nh * per_head), r = in / (a.D / 8), c = in - r * (a.D / 8);
    const long n = nh / a.Hk;
    const int h = (int)(nh - n * a.Hk), id = a.ids[n];
    u32x4_t v = {0u, 0u, 0u, 0u};
    if ((unsigned)id < (unsigned)a.pool) {
      const long at = id * pg.page + h * pg.head + r * pg.row + 8 * c;
      if constexpr (CODES) {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(pg.data + at);
        const float unit = scale_of(pg.exps[id * pg.epage + h * pg.ehead]);
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f32x2_t x = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], false), y = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], true);
          v[2 * k] = put<DT>(x.x * unit) | put<DT>(x.y * unit) << 16;
          v[2 * k + 1] = put<DT>(y.x * unit) | put<DT>(y.y * unit) << 16;
        }
      } else {
        v = ldg128(reinterpret_cast<const u16*>(pg.data) + at);
      }
    }
    stg128(a.out[blockIdx.y] + 8 * i, v);
  }
}

}  // namespace

int take_pages(const char* what, const dspark_pages* p, int64_t pool, int64_t Hk, int64_t P, int64_t D, bool codes, Pages* out) {
  if (!p->data || (codes && !p->exponents)) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  const int64_t wide = codes ? 16 : 8;
  if (!aligned(p->data, 16)) return fail(DSPARK_ERR_ALIGN, "%s: pages must be 16-byte aligned", what);
  for (int i = 0; i < 3; ++i)
    if (p->strides[i] < 0 || p->strides[i] % wide || (i == 2 && p->strides[i] > (1 << 22)))
      return fail(DSPARK_ERR_ALIGN, "%s: page strides must be multiples of 16 bytes", what);
  *out = Pages{static_cast<char*>(p->data), codes ? static_cast<unsigned char*>(p->exponents) : nullptr, p->strides[0],
               p->strides[1], p->strides[2], p->exponent_strides[0], p->exponent_strides[1]};
  return DSPARK_OK;
}

int check_pool(const char* what, int64_t pool, int64_t Hk, int64_t P, int64_t D) {
  if (D != 64 && D != 128 && D != 256) return fail(DSPARK_ERR_SHAPE, "%s: head_dim %ld (64, 128 or 256)", what, (long)D);
  if (P != 16 && P != 32 && P != 64 && P != 128)
    return fail(DSPARK_ERR_SHAPE, "%s: pages of %ld positions (16, 32, 64 or 128)", what, (long)P);
  if (Hk < 1 || Hk > 1024 || pool < 1 || pool >= (1L << 31))
    return fail(DSPARK_ERR_SHAPE, "%s: %ld pages of %ld heads", what, (long)pool, (long)Hk);
  return DSPARK_OK;
}

int take_seqs(const char* what, const dspark_sequences* p, int64_t P, int64_t pool, Seqs* out) {
  if (!p->table || !p->starts || !p->lens) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  if (p->count < 1 || p->count > 4096 || p->width < 1 || p->width > (1 << 24) || p->rows < 1 || p->rows >= (1 << 22) ||
      p->ld_table < p->width || p->width * P > (1L << 30))
    return fail(DSPARK_ERR_SHAPE, "%s: %ld sequences (up to 4096) of %ld pages, %ld rows (up to 2^22)", what, (long)p->count,
                (long)p->width, (long)p->rows);
  *out = Seqs{p->table, p->starts, p->lens, p->ld_table, (int)p->count, (int)p->width, (int)p->rows, (int)P,
              __builtin_ctz((unsigned)P), (int)pool};
  return DSPARK_OK;
}

}  // namespace paged
}  // namespace dspark

using namespace dspark;

namespace {

template <int DT, bool INTER>
void launch_append(const paged::AppendArgs& a, bool codes, unsigned blocks, size_t lds, hipStream_t s) {
  const dim3 grid(blocks), block(paged::kThreads);
  if (codes) hipLaunchKernelGGL((paged::append_kernel<DT, INTER, true>), grid, block, lds, s, a);
  else hipLaunchKernelGGL((paged::append_kernel<DT, INTER, false>), grid, block, lds, s, a);
}
template <int DT>
void launch_append(const paged::AppendArgs& a, bool inter, bool codes, unsigned blocks, size_t lds, hipStream_t s) {
  inter ? launch_append<DT, true>(a, codes, blocks, lds, s) : launch_append<DT, false>(a, codes, blocks, lds, s);
}

int take_rows(const char* what, const void* x, const int64_t st[2], paged::Rows* out) {
  if (!aligned(x, 16) || st[0] % 8 || st[1] % 8) return fail(DSPARK_ERR_ALIGN, "%s: rows must be 16-byte aligned, their strides too", what);
  *out = paged::Rows{static_cast<const char*>(x), st[0], st[1]};
  return DSPARK_OK;
}

}  // namespace

extern "C" int dspark_paged_append(const dspark_paged_append_args* p, dspark_stream stream) {
  const char* what = "paged_append";
  if (!p || !p->k || !p->v || (p->Hq > 0 && (!p->q || !p->q_out)) || (p->dims > 0 && !p->freqs))
    return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  if (p->dtype != DSPARK_DTYPE_BF16 && p->dtype != DSPARK_DTYPE_F16)
    return fail(DSPARK_ERR_UNSUPPORTED, "%s: dtype %ld", what, (long)p->dtype);
  paged::AppendArgs a = {};
  const bool codes = p->codes != 0, inter = p->interleaved != 0;
  int st = paged::check_pool(what, p->pool, p->Hk, p->P, p->D);
  if (st || (st = paged::take_seqs(what, &p->seqs, p->P, p->pool, &a.s)) ||
      (st = paged::take_pages(what, &p->k_pages, p->pool, p->Hk, p->P, p->D, codes, &a.kp)) ||
      (st = paged::take_pages(what, &p->v_pages, p->pool, p->Hk, p->P, p->D, codes, &a.vp)) ||
      (st = take_rows(what, p->k, p->k_strides, &a.k)) || (st = take_rows(what, p->v, p->v_strides, &a.v)))
    return st;
  if (p->Hq < 0 || p->Hq > 4096) return fail(DSPARK_ERR_SHAPE, "%s: Hq=%ld", what, (long)p->Hq);
  if (p->dims < 0 || p->dims > p->D || p->dims % (inter ? 8 : 16))
    return fail(DSPARK_ERR_SHAPE, "%s: rotated part %ld of %ld (a multiple of 16, interleaved of 8)", what, (long)p->dims, (long)p->D);
  if (p->Hq) {
    if ((st = take_rows(what, p->q, p->q_strides, &a.q))) return st;
    paged::Rows o;
    if ((st = take_rows(what, p->q_out, p->q_out_strides, &o))) return st;
    a.qo = static_cast<char*>(p->q_out);
    a.qo_row = o.row;
    a.qo_head = o.head;
    a.clear = p->q_clear != 0;
  }
  a.Hq = (int)p->Hq;
  a.Hk = (int)p->Hk;
  a.D = (int)p->D;
  a.half = (int)(p->dims / 2);
  a.freqs = p->freqs;
  a.scale = p->scale;
  a.pos = p->positions;
  a.pos64 = p->positions_i64 != 0;
  a.pstride = p->position_stride;
  const int rot = inter ? a.half / 4 : a.half / 8, per = rot + (a.D - 2 * a.half) / 8;
  const int items = (a.Hq + (codes ? 0 : a.Hk)) * per + (codes ? 0 : a.Hk * (a.D / 8));
  a.parts = a.s.T >= 512 ? 1 : (items + paged::kThreads - 1) / paged::kThreads;
  if (a.parts < 1) a.parts = 1;
  long blocks = items ? (long)a.s.T * a.parts : 0;
  size_t lds = (size_t)a.half * sizeof(float2);
  if (codes) {
    // a sequence's rows reach into one page more than they fill, at each end
    const long pages = std::min<long>(a.s.T, a.s.T / p->P + 2L * a.s.B) * a.Hk * 2;
    a.page_blocks = (int)std::min<long>(pages, INT32_MAX);
    blocks += pages;
    lds = std::max(lds, (size_t)(std::min<long>(p->P, a.s.T) * p->D * 2));
  }
  if (blocks >= (1L << 31) / paged::kThreads) return fail(DSPARK_ERR_SHAPE, "%s: %ld workgroups", what, blocks);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == DSPARK_DTYPE_BF16) launch_append<DSPARK_DTYPE_BF16>(a, inter, codes, (unsigned)blocks, lds, s);
  else launch_append<DSPARK_DTYPE_F16>(a, inter, codes, (unsigned)blocks, lds, s);
  return check_launch(what);
}

extern "C" int dspark_paged_read(const dspark_paged_read_args* p, dspark_stream stream) {
  const char* what = "paged_read";
  if (!p || !p->ids || !p->k_out || !p->v_out) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  if (p->dtype != DSPARK_DTYPE_BF16 && p->dtype != DSPARK_DTYPE_F16)
    return fail(DSPARK_ERR_UNSUPPORTED, "%s: dtype %ld", what, (long)p->dtype);
  paged::ReadArgs a = {};
  const bool codes = p->codes != 0;
  int st = paged::check_pool(what, p->pool, p->Hk, p->P, p->D);
  if (st || (st = paged::take_pages(what, &p->k_pages, p->pool, p->Hk, p->P, p->D, codes, &a.side[0])) ||
      (st = paged::take_pages(what, &p->v_pages, p->pool, p->Hk, p->P, p->D, codes, &a.side[1])))
    return st;
  if (p->count < 1 || p->count >= (1L << 31)) return fail(DSPARK_ERR_SHAPE, "%s: %ld pages", what, (long)p->count);
  if (!aligned(p->k_out, 16) || !aligned(p->v_out, 16)) return fail(DSPARK_ERR_ALIGN, "%s: outputs must be 16-byte aligned", what);
  a.out[0] = static_cast<u16*>(p->k_out);
  a.out[1] = static_cast<u16*>(p->v_out);
  a.ids = p->ids;
  a.N = (int)p->count;
  a.Hk = (int)p->Hk;
  a.P = (int)p->P;
  a.D = (int)p->D;
  a.pool = (int)p->pool;
  a.items = p->count * p->Hk * (p->P * p->D / 8);
  const unsigned blocks = (unsigned)std::min<long>((a.items + paged::kThreads - 1) / paged::kThreads, 1L << 16);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(blocks, 2), block(paged::kThreads);
  if (p->dtype == DSPARK_DTYPE_BF16) {
    if (codes) hipLaunchKernelGGL((paged::read_kernel<DSPARK_DTYPE_BF16, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((paged::read_kernel<DSPARK_DTYPE_BF16, false>), grid, block, 0, s, a);
  } else {
    if (codes) hipLaunchKernelGGL((paged::read_kernel<DSPARK_DTYPE_F16, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((paged::read_kernel<DSPARK_DTYPE_F16, false>), grid, block, 0, s, a);
  }
  return check_launch(what);
}
