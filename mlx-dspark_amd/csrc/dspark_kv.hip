// Rows quantized into a key/value cache as they are written, and the cache read back (gfx950), both
// tensors of a layer in one launch.
//
// A group is 64 values of a row; its scale and bias are rounded to the cache's type, its fields come from
// the rounded ones, every step one fp32 operation (dspark_rocm.quant.quantize_rows on this GPU, bit for
// bit: torch's quotient by a constant is the product with its rounded reciprocal here, so the fused
// q/k/v kernel, which divides, rounds about one scale in 2^16 to the other side):
//   scale = T((max - min) * fl(1 / (2^bits - 1))), bias = T(min), f = clamp(round_half_even((x - bias) / scale))
// with a scale of 0 dividing as 1; read back: T'(fl(f * scale) + bias). A NaN in a group makes its scale and
// bias NaN and its fields 0. "Bit for bit" is but for the sign of a bias of zero: a group whose least values are +0 and
// -0 gets -0 here, what its order gives in torch; the values read back are the same.
//
// Bound by bytes: 8 lanes hold a group, 8 values a lane (16 bytes of a 16-bit row), the group's extremes
// joined over the 8 lanes with DPP. 2048 rows of 4 x 256 in bf16 to 4 bits: 7.1 us for 10.8 MB, of which the launch and
// one round of loads are 4; 32768 rows of 8 x 128 read back to fp32 from 8 bits: 50 us for 340 MB, 6.8 TB/s, the rate
// of a fill of the same size.
#include "dspark_common.h"

// A product and a sum stay two roundings: a fused one does not overflow between them.
#pragma clang fp contract(off)

namespace dspark {
namespace {

constexpr int kKvThreads = 256;
// Stores of a thread that reads back (one row written and 32768 of 8 x 128 read back, both kernels from a replayed graph:
// 51.7 us at 2, 85.4 at 1, 52.9 at 4; 16 written and 4017 read back: 9.8, 14.9, 11.2).
constexpr int kKvOut = 2;

struct KvSide {                                // keys or values
  char* x;                                     // plain rows (read, or the output of a read back)
  long xb, xh, xt;                             // strides of batch, head, row, in elements
  u32* w;
  u16* s;
  u16* b;
  long wb, wh, wt, sb, sh, st;
};

struct KvArgs {
  KvSide side[2];
  int B, H, D8;                                // D8 = D / 8
  u32 items;                                   // rows * D8 of one head
};

template <int DT>
__device__ __forceinline__ float kv_get(u32 bits) {
  if constexpr (DT == DSPARK_DTYPE_F16) return (float)__builtin_bit_cast(_Float16, (u16)bits);
  else return bf2f(bits);
}
template <int DT>
__device__ __forceinline__ u16 kv_put(float v) {
  if constexpr (DT == DSPARK_DTYPE_F16) return __builtin_bit_cast(u16, (_Float16)v);
  else return f2bf(v);
}

// Joined over each aligned group of 8 lanes, in all of them (the exchanges of sum8_lanes).
__device__ __forceinline__ float min8_lanes(float v) {
  v = fminf(v, dpp_mov<0xB1>(v));
  v = fminf(v, dpp_mov<0x4E>(v));
  return fminf(v, dpp_mov<0x141>(v));
}
__device__ __forceinline__ float max8_lanes(float v) {
  v = fmaxf(v, dpp_mov<0xB1>(v));
  v = fmaxf(v, dpp_mov<0x4E>(v));
  return fmaxf(v, dpp_mov<0x141>(v));
}

// SRC: type of the rows; DST: type of scales and biases; ALIGNED: 16-byte rows, 8-byte words
template <int SRC, int DST, int BITS, bool ALIGNED>
__global__ __launch_bounds__(kKvThreads) void kv_quantize_kernel(const KvArgs a) {
  const u32 i = blockIdx.x * kKvThreads + threadIdx.x;
  if (i >= a.items) return;                    // whole groups: items is a multiple of 8
  const int bh = blockIdx.y % (a.B * a.H), b = bh / a.H, h = bh % a.H;
  const KvSide& s = a.side[blockIdx.y >= (unsigned)(a.B * a.H)];
  const u32 t = i / (u32)a.D8, c = i - t * a.D8;
  float v[8];
  const long at = b * s.xb + h * s.xh + (long)t * s.xt + 8 * c;
  if constexpr (SRC == DSPARK_DTYPE_F32) {
    const float* x = reinterpret_cast<const float*>(s.x) + at;
    if constexpr (ALIGNED) {
      const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(x), hi = *reinterpret_cast<const f32x4_t*>(x + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = lo[j];
        v[4 + j] = hi[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = x[j];
    }
  } else {
    const u16* x = reinterpret_cast<const u16*>(s.x) + at;
    if constexpr (ALIGNED) {
      const u32x4_t r = ldg128(x);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = kv_get<SRC>(r[j] & 0xFFFFu);
        v[2 * j + 1] = kv_get<SRC>(r[j] >> 16);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = kv_get<SRC>(x[j]);
    }
  }
  constexpr float kLevels = (float)((1 << BITS) - 1);
  float lo = v[0], hi = v[0], bad = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo = fminf(lo, v[j]);
    hi = fmaxf(hi, v[j]);
    bad = v[j] != v[j] ? 1.f : bad;
  }
  lo = min8_lanes(lo);
  hi = max8_lanes(hi);
  if (max8_lanes(bad) != 0.f) lo = hi = __builtin_nanf("");
  float range = (hi - lo) * (1.0f / kLevels);
  asm("" : "+v"(range));                       // in fp32 first: else product and conversion to fp16 are one instruction, rounded once
  const u16 sbits = kv_put<DST>(range), bbits = kv_put<DST>(lo);
  const float sc = kv_get<DST>(sbits), bias = kv_get<DST>(bbits);
  const float div = sc == 0.f ? 1.f : sc;
  u32 f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    f[j] = (u32)fminf(fmaxf(rintf(__fdiv_rn(v[j] - bias, div)), 0.f), kLevels);
  u32* w = s.w + b * s.wb + h * s.wh + (long)t * s.wt + (BITS / 4) * c;
  if constexpr (BITS == 8) {
    const u32x2_t two = {f[0] | (f[1] << 8) | (f[2] << 16) | (f[3] << 24), f[4] | (f[5] << 8) | (f[6] << 16) | (f[7] << 24)};
    if constexpr (ALIGNED) {
      *reinterpret_cast<u32x2_t*>(w) = two;
    } else {
      w[0] = two[0];
      w[1] = two[1];
    }
  } else {
    u32 one = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) one |= f[j] << (4 * j);
    *w = one;
  }
  if ((c & 7) == 0) {
    const long g = b * s.sb + h * s.sh + (long)t * s.st + (c >> 3);
    s.s[g] = sbits;
    s.b[g] = bbits;
  }
}

// SRC: type of scales and biases; DST: type of the rows written; ALIGNED as above. An item is one store of 16 bytes
// (4 or 8 values), the lanes' next to each other; a thread takes kOut of them, their loads first.
template <int SRC, int DST, int BITS, bool ALIGNED>
__global__ __launch_bounds__(kKvThreads) void kv_dequantize_kernel(const KvArgs a) {
  constexpr int W = DST == DSPARK_DTYPE_F32 ? 4 : 8, kOut = kKvOut, kPerWord = 32 / BITS;
  const u32 i0 = blockIdx.x * (kKvThreads * kOut) + threadIdx.x, items = a.items * (8 / W), per = a.D8 * (8 / W);
  const int bh = blockIdx.y % (a.B * a.H), b = bh / a.H, h = bh % a.H;
  const KvSide& s = a.side[blockIdx.y >= (unsigned)(a.B * a.H)];
  u32 w[kOut][2], t[kOut], c[kOut];
  u16 sc[kOut], bi[kOut];
#pragma unroll
  for (int k = 0; k < kOut; ++k) {
    const u32 i = i0 + k * kKvThreads;
    if (i >= items) continue;
    t[k] = i / per;
    c[k] = (i - t[k] * per) * W;        // first value
    const u32* p = s.w + b * s.wb + h * s.wh + (long)t[k] * s.wt + c[k] / kPerWord;
    if constexpr (W > kPerWord) {
      if constexpr (ALIGNED) {
        const u32x2_t two = ldg64(p);
        w[k][0] = two[0];
        w[k][1] = two[1];
      } else {
        w[k][0] = p[0];
        w[k][1] = p[1];
      }
    } else {
      w[k][0] = *p >> (W < kPerWord ? (c[k] & (kPerWord - 1)) * BITS : 0);
    }
    const long g = b * s.sb + h * s.sh + (long)t[k] * s.st + (c[k] >> 6);
    sc[k] = s.s[g];
    bi[k] = s.b[g];
  }
#pragma unroll
  for (int k = 0; k < kOut; ++k) {
    if (i0 + k * kKvThreads >= items) break;
    const float scale = kv_get<SRC>(sc[k]), bias = kv_get<SRC>(bi[k]);
    float v[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const u32 q = (w[k][j / kPerWord] >> (BITS * (j % kPerWord))) & ((1u << BITS) - 1);
      v[j] = (float)q * scale + bias;
    }
    const long at = b * s.xb + h * s.xh + (long)t[k] * s.xt + c[k];
    if constexpr (DST == DSPARK_DTYPE_F32) {
      float* y = reinterpret_cast<float*>(s.x) + at;
      if constexpr (ALIGNED) {
        __builtin_nontemporal_store(f32x4_t{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4_t*>(y));
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) y[j] = v[j];
      }
    } else {
      u16* y = reinterpret_cast<u16*>(s.x) + at;
      if constexpr (ALIGNED) {
        u32x4_t o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = (u32)kv_put<DST>(v[2 * j]) | ((u32)kv_put<DST>(v[2 * j + 1]) << 16);
        __builtin_nontemporal_store(o, reinterpret_cast<u32x4_t*>(y));
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) y[j] = kv_put<DST>(v[j]);
      }
    }
  }
}

template <bool WRITE, int A, int C, int BITS, bool AL>
void launch_kv(const KvArgs& a, hipStream_t s) {
  const u32 per = WRITE ? kKvThreads : kKvThreads * kKvOut;
  const u32 items = WRITE ? a.items : a.items * (C == DSPARK_DTYPE_F32 ? 2 : 1);
  const dim3 grid((items + per - 1) / per, (unsigned)(2 * a.B * a.H)), block(kKvThreads);
  if constexpr (WRITE) hipLaunchKernelGGL((kv_quantize_kernel<A, C, BITS, AL>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((kv_dequantize_kernel<A, C, BITS, AL>), grid, block, 0, s, a);
}

template <bool WRITE, int A, int C>
void launch_kv(const KvArgs& a, int bits, bool al, hipStream_t s) {
  if (bits == 8) al ? launch_kv<WRITE, A, C, 8, true>(a, s) : launch_kv<WRITE, A, C, 8, false>(a, s);
  else al ? launch_kv<WRITE, A, C, 4, true>(a, s) : launch_kv<WRITE, A, C, 4, false>(a, s);
}

// The arguments both directions share; `al`: everything a wide access touches is aligned for it.
int kv_args(const char* what, const dspark_kv_args* p, KvArgs& a, bool& al) {
  if (!p) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  const int64_t B = p->B, H = p->H, T = p->T, D = p->D, xdt = p->x_dtype, cdt = p->cache_dtype;
  if (p->bits != 4 && p->bits != 8) return fail(DSPARK_ERR_UNSUPPORTED, "%s: bits=%lld (4 or 8)", what, (long long)p->bits);
  if (p->group_size != 64) return fail(DSPARK_ERR_UNSUPPORTED, "%s: group_size=%lld (64)", what, (long long)p->group_size);
  if ((cdt != DSPARK_DTYPE_BF16 && cdt != DSPARK_DTYPE_F16) ||
      (xdt != DSPARK_DTYPE_BF16 && xdt != DSPARK_DTYPE_F16 && xdt != DSPARK_DTYPE_F32))
    return fail(DSPARK_ERR_UNSUPPORTED, "%s: rows of dtype %lld, a cache of dtype %lld", what, (long long)xdt, (long long)cdt);
  if (D < 64 || D % 64 || D > 4096) return fail(DSPARK_ERR_SHAPE, "%s: head_dim %lld (a multiple of 64 up to 4096)", what, (long long)D);
  if (B < 1 || H < 1 || B > 32767 || H > 32767 || 2 * B * H > 65535 || T < 1 || T > (1LL << 31) / D * 4)
    return fail(DSPARK_ERR_SHAPE, "%s: B=%lld H=%lld rows=%lld", what, (long long)B, (long long)H, (long long)T);
  const int es = xdt == DSPARK_DTYPE_F32 ? 4 : 2;
  al = true;
  for (int i = 0; i < 2; ++i) {
    const dspark_kv_side& k = i ? p->values : p->keys;
    if (!k.x || !k.words || !k.scales || !k.biases) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
    if (!aligned(k.x, es) || !aligned(k.words, 4) || !aligned(k.scales, 2) || !aligned(k.biases, 2))
      return fail(DSPARK_ERR_ALIGN, "%s: tensors need the alignment of their type", what);
    al = al && aligned(k.x, 16) && aligned(k.words, 8);
    for (int j = 0; j < 3; ++j) al = al && k.x_strides[j] % (16 / es) == 0 && k.word_strides[j] % 2 == 0;
    a.side[i] = KvSide{static_cast<char*>(k.x), k.x_strides[0], k.x_strides[1], k.x_strides[2], k.words,
                       static_cast<u16*>(k.scales), static_cast<u16*>(k.biases), k.word_strides[0], k.word_strides[1],
                       k.word_strides[2], k.scale_strides[0], k.scale_strides[1], k.scale_strides[2]};
  }
  a.B = (int)B;
  a.H = (int)H;
  a.D8 = (int)(D / 8);
  a.items = (u32)(T * (D / 8));
  return DSPARK_OK;
}

template <bool WRITE>
void launch_types(const KvArgs& a, int x_dtype, int c_dtype, int bits, bool al, hipStream_t s) {
  constexpr int bf = DSPARK_DTYPE_BF16, hf = DSPARK_DTYPE_F16, f = DSPARK_DTYPE_F32;
  const bool ch = c_dtype == hf;
  if constexpr (WRITE) {
    if (x_dtype == bf) ch ? launch_kv<WRITE, bf, hf>(a, bits, al, s) : launch_kv<WRITE, bf, bf>(a, bits, al, s);
    else if (x_dtype == hf) ch ? launch_kv<WRITE, hf, hf>(a, bits, al, s) : launch_kv<WRITE, hf, bf>(a, bits, al, s);
    else ch ? launch_kv<WRITE, f, hf>(a, bits, al, s) : launch_kv<WRITE, f, bf>(a, bits, al, s);
  } else {
    if (x_dtype == bf) ch ? launch_kv<WRITE, hf, bf>(a, bits, al, s) : launch_kv<WRITE, bf, bf>(a, bits, al, s);
    else if (x_dtype == hf) ch ? launch_kv<WRITE, hf, hf>(a, bits, al, s) : launch_kv<WRITE, bf, hf>(a, bits, al, s);
    else ch ? launch_kv<WRITE, hf, f>(a, bits, al, s) : launch_kv<WRITE, bf, f>(a, bits, al, s);
  }
}

}  // namespace
}  // namespace dspark

using namespace dspark;

extern "C" int dspark_kv_quantize(const dspark_kv_args* p, dspark_stream stream) {
  KvArgs a;
  bool al;
  const int st = kv_args("kv_quantize", p, a, al);
  if (st) return st;
  launch_types<true>(a, (int)p->x_dtype, (int)p->cache_dtype, (int)p->bits, al, static_cast<hipStream_t>(stream));
  return check_launch("kv_quantize");
}

extern "C" int dspark_kv_dequantize(const dspark_kv_args* p, dspark_stream stream) {
  KvArgs a;
  bool al;
  const int st = kv_args("kv_dequantize", p, a, al);
  if (st) return st;
  launch_types<false>(a, (int)p->x_dtype, (int)p->cache_dtype, (int)p->bits, al, static_cast<hipStream_t>(stream));
  return check_launch("kv_dequantize");
}
