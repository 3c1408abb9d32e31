// Rotary positions of queries and keys in one launch (gfx950).
//
//   a_i = position * freqs_i,   (y1, y2) = scale * (x1 cos a_i - x2 sin a_i, x1 sin a_i + x2 cos a_i)
// for the pairs (i, i + half) or, interleaved, (2i, 2i + 1) of a head's first 2 half values; the others
// are copied. cos and sin of a position serve every head of its row: a workgroup forms them once for its
// rows in LDS. The angle is reduced in fp64, in turns: at position 1e6 an fp32 product is off by 0.06 rad,
// the fp64 one by 1e-10; its sine and cosine are fp32, within a few units of their own size also near zero. The rotation
// is fp32, rounded once to the tensors' type.
//
// Bound by the bytes of x and y: 16 bytes a lane and access where addresses and strides allow, else one
// value.
#include "dspark_common.h"

namespace dspark {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeHalf = 128;                 // pairs of a head
constexpr int kRopeRows = 4;                   // most rows of a workgroup
constexpr int kRopeTab = kRopeRows * kRopeHalf;

struct RopeSide {                              // queries or keys
  const char* x;
  char* y;
  long xb, xh, xl, yb, yh, yl;                 // strides of batch, head, row
};

struct RopeArgs {
  RopeSide s[2];
  int heads0, heads;                           // of s[0], of both
  int L, D, half, rows;                        // rows = B * L
  int per;                                     // items of a head
  int rot;                                     // of these, items that rotate
  int tok;                                     // rows of a workgroup
  const void* pos;
  int pos64;
  long pb, pl;                                 // strides of the positions
  long pos0;                                   // without pos: row l stands at pos0 + l
  const double* freqs;
  double scale;
};

template <int DT> struct Elem;
template <> struct Elem<DSPARK_DTYPE_BF16> {
  using t = u16;
  static __device__ __forceinline__ float get(u16 v) { return bf2f(v); }
  static __device__ __forceinline__ u16 put(float v) { return f2bf(v); }
};
template <> struct Elem<DSPARK_DTYPE_F16> {
  using t = u16;
  static __device__ __forceinline__ float get(u16 v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ u16 put(float v) { return __builtin_bit_cast(u16, (_Float16)v); }
};
template <> struct Elem<DSPARK_DTYPE_F32> {
  using t = float;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

template <typename T, int W>
__device__ __forceinline__ void store(T* p, const Pack<T, W>& v) {
  static_assert(sizeof(v) == 16, "one access");
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, v), reinterpret_cast<u32x4_t*>(p));
}

// (cos, sin) of a workgroup's rows
__device__ __forceinline__ void fill_table(const RopeArgs& a, float2* tab, int r0, int nr) {
  for (int i = threadIdx.x; i < nr * a.half; i += kRopeThreads) {
    const int r = r0 + i / a.half, f = i % a.half, b = r / a.L, l = r % a.L;
    long p = a.pos0 + l;
    if (a.pos) {
      const long at = b * a.pb + l * a.pl;
      p = a.pos64 ? static_cast<const int64_t*>(a.pos)[at] : (long)static_cast<const int32_t*>(a.pos)[at];
    }
    const double turns = (double)p * (a.freqs[f] * 0.15915494309189535);
    const double halves = 2.0 * (turns - __builtin_rint(turns));
    const float hi = (float)halves;
    float sn, cs;
    sincospif(hi, &sn, &cs);
    // What fp32 leaves of the angle (up to 1e-7 rad: all of a cosine near zero), to first order, and the factor in fp64:
    // one rounding of each.
    const double lo = 3.141592653589793 * (halves - (double)hi);
    tab[i] = make_float2((float)(((double)cs - lo * (double)sn) * a.scale), (float)(((double)sn + lo * (double)cs) * a.scale));
  }
}

template <int DT>
__device__ __forceinline__ void turn(const float2 cs, typename Elem<DT>::t& x1, typename Elem<DT>::t& x2) {
  const float u = Elem<DT>::get(x1), v = Elem<DT>::get(x2);
  x1 = Elem<DT>::put(u * cs.x - v * cs.y);
  x2 = Elem<DT>::put(u * cs.y + v * cs.x);
}

// 16 bytes an access, W values, written past the caches (2048 rows of 72 x 128: 14.9 us, 15.8 with plain stores; a
// copy of the bytes: 14.7). An item of a head is W pairs (half layout: two accesses), the W / 2 pairs of W values
// (interleaved), or W copied values. A thread keeps its item over the heads of all its workgroup's rows, kOut of
// them at once: no division in the loop.
template <int DT, int W, bool INTER>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const RopeArgs a) {
  using T = typename Elem<DT>::t;
  using P = Pack<T, W>;
  constexpr int kOut = 3;
  __shared__ float2 tab[kRopeTab];
  __shared__ long at_x[2][kRopeRows], at_y[2][kRopeRows];
  const int r0 = blockIdx.x * a.tok, nr = min(a.tok, a.rows - r0), t = threadIdx.x;
  if (t < 2 * kRopeRows) {              // where a row starts, queries and keys
    const int side = t / kRopeRows, i = t % kRopeRows, r = min(r0 + i, a.rows - 1), b = r / a.L, l = r - b * a.L;
    const RopeSide& s = a.s[side];
    at_x[side][i] = b * s.xb + l * s.xl;
    at_y[side][i] = b * s.yb + l * s.yl;
  }
  fill_table(a, tab, r0, nr);
  __syncthreads();
  const int heads_at_once = kRopeThreads / a.per, first = t / a.per, c = t - first * a.per;
  if (first >= heads_at_once) return;
  const int step = gridDim.y * heads_at_once;
  const bool rot = c < a.rot;
  const int d = rot ? c * W : 2 * a.half + (c - a.rot) * W;
  int h = blockIdx.y * heads_at_once + first, r = 0;
  while (h >= a.heads) {
    h -= a.heads;
    ++r;
  }
  while (r < nr) {
    P x1[kOut], x2[kOut];
    T* y[kOut];
    int row[kOut];
#pragma unroll
    for (int i = 0; i < kOut; ++i) {
      row[i] = r;
      if (r >= nr) continue;
      const int side = h >= a.heads0, hs = h - (side ? a.heads0 : 0);
      const RopeSide& s = a.s[side];
      const T* x = reinterpret_cast<const T*>(s.x) + at_x[side][r] + hs * s.xh + d;
      y[i] = reinterpret_cast<T*>(s.y) + at_y[side][r] + hs * s.yh + d;
      x1[i] = *reinterpret_cast<const P*>(x);
      if (!INTER && rot) x2[i] = *reinterpret_cast<const P*>(x + a.half);
      h += step;
      while (h >= a.heads) {
        h -= a.heads;
        ++r;
      }
    }
#pragma unroll
    for (int i = 0; i < kOut; ++i) {
      if (row[i] >= nr) break;
      const float2* cs = tab + row[i] * a.half;
      if (rot) {
#pragma unroll
        for (int e = 0; e < W; e += INTER ? 2 : 1) {
          if constexpr (INTER) turn<DT>(cs[(d + e) >> 1], x1[i].v[e], x1[i].v[e + 1]);
          else turn<DT>(cs[d + e], x1[i].v[e], x2[i].v[e]);
        }
      }
      store(y[i], x1[i]);
      if (!INTER && rot) store(y[i] + a.half, x2[i]);
    }
  }
}

// The same a value at a time, for addresses, strides and sizes that have no 16 bytes together: an item is a pair or a
// copied value.
template <int DT, bool INTER>
__global__ __launch_bounds__(kRopeThreads) void rope_single_kernel(const RopeArgs a) {
  using T = typename Elem<DT>::t;
  __shared__ float2 tab[kRopeTab];
  const int r0 = blockIdx.x * a.tok, nr = min(a.tok, a.rows - r0);
  fill_table(a, tab, r0, nr);
  __syncthreads();
  const int per_row = a.heads * a.per, n = nr * per_row;
  for (int i = blockIdx.y * kRopeThreads + threadIdx.x; i < n; i += gridDim.y * kRopeThreads) {
    const int tr = i / per_row, j = i - tr * per_row;
    int h = j / a.per;
    const int c = j - h * a.per;
    const int r = r0 + tr, b = r / a.L, l = r - b * a.L;
    const int side = h >= a.heads0;
    h -= side ? a.heads0 : 0;
    const RopeSide& s = a.s[side];
    const T* x = reinterpret_cast<const T*>(s.x) + b * s.xb + h * s.xh + l * s.xl;
    T* y = reinterpret_cast<T*>(s.y) + b * s.yb + h * s.yh + l * s.yl;
    if (c >= a.rot) {                   // beyond the rotated part
      y[a.half + c] = x[a.half + c];
    } else {
      const int d1 = INTER ? 2 * c : c, d2 = INTER ? 2 * c + 1 : c + a.half;
      T u = x[d1], v = x[d2];
      turn<DT>(tab[tr * a.half + c], u, v);
      y[d1] = u;
      y[d2] = v;
    }
  }
}

template <int DT, int W>
void launch_rope(RopeArgs a, bool inter, hipStream_t s) {
  a.rot = inter ? (W == 1 ? a.half : 2 * a.half / W) : a.half / W;
  a.per = a.rot + (a.D - 2 * a.half) / W;
  // Rows of a workgroup: one, its heads spread over workgroups until there are two a CU where rows are few. Many rows
  // of few heads share one until a thread has two items (2048 rows of 10 heads x 64: 4.0 us, 4.5 at one row each;
  // of 72 x 128: 15.5 at two rows, 14.9 at one).
  const int row_items = a.heads * a.per, fit = (2 * kRopeThreads + row_items - 1) / row_items;
  a.tok = a.rows >= 1024 ? (fit < kRopeRows ? fit : kRopeRows) : 1;
  const unsigned gx = (unsigned)((a.rows + a.tok - 1) / a.tok);
  const unsigned most = (unsigned)((a.tok * a.heads * a.per + kRopeThreads - 1) / kRopeThreads);
  const unsigned gy = gx >= 512 ? 1u : (most < 512 / gx ? most : (512 / gx ? 512 / gx : 1u));
  const dim3 grid(gx, gy), block(kRopeThreads);
  if constexpr (W == 1) {
    if (inter) hipLaunchKernelGGL((rope_single_kernel<DT, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rope_single_kernel<DT, false>), grid, block, 0, s, a);
  } else {
    if (inter) hipLaunchKernelGGL((rope_kernel<DT, W, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rope_kernel<DT, W, false>), grid, block, 0, s, a);
  }
}

}  // namespace
}  // namespace dspark

using namespace dspark;

extern "C" int dspark_rope(const dspark_rope_args* p, dspark_stream stream) {
  const char* what = "rope";
  if (!p || !p->q || !p->q_out || !p->freqs || (p->Hk > 0 && (!p->k || !p->k_out))) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  const int64_t dt = p->dtype, B = p->B, L = p->L, D = p->D, dims = p->dims, Hq = p->Hq, Hk = p->Hk;
  if (dt != DSPARK_DTYPE_BF16 && dt != DSPARK_DTYPE_F16 && dt != DSPARK_DTYPE_F32)
    return fail(DSPARK_ERR_UNSUPPORTED, "%s: dtype %lld", what, (long long)dt);
  if (D < 2 || D > 1024 || dims < 2 || dims > 2 * kRopeHalf || dims % 2 || dims > D)
    return fail(DSPARK_ERR_SHAPE, "%s: head_dim %lld (2..1024), rotated part %lld (even, up to it and to 256)", what, (long long)D, (long long)dims);
  // a workgroup a row: fewer than 2^32 threads
  if (B < 1 || L < 1 || B > (1 << 24) || L > (1 << 24) || B * L >= (1 << 24) || Hq < 1 || Hk < 0 || Hq > 4096 || Hk > 4096 ||
      Hq + Hk > 4096)
    return fail(DSPARK_ERR_SHAPE, "%s: B=%lld L=%lld Hq=%lld Hk=%lld", what, (long long)B, (long long)L, (long long)Hq, (long long)Hk);
  const int64_t es = dt == DSPARK_DTYPE_F32 ? 4 : 2, wide = 16 / es;
  const bool inter = p->interleaved != 0;
  RopeArgs a = {};
  bool vec = D % wide == 0 && (inter ? dims : dims / 2) % wide == 0;
  for (int i = 0; i < (Hk ? 2 : 1); ++i) {
    const void* x = i ? p->k : p->q;
    void* y = i ? p->k_out : p->q_out;
    const int64_t *xs = i ? p->k_strides : p->q_strides, *ys = i ? p->k_out_strides : p->q_out_strides;
    if (!aligned(x, es) || !aligned(y, es)) return fail(DSPARK_ERR_ALIGN, "%s: tensors need the alignment of their type", what);
    vec = vec && aligned(x, 16) && aligned(y, 16);
    for (int j = 0; j < 3; ++j) vec = vec && xs[j] % wide == 0 && ys[j] % wide == 0;
    a.s[i] = RopeSide{static_cast<const char*>(x), static_cast<char*>(y), xs[0], xs[1], xs[2], ys[0], ys[1], ys[2]};
  }
  a.heads0 = (int)Hq;
  a.heads = (int)(Hq + Hk);
  a.L = (int)L;
  a.D = (int)D;
  a.half = (int)(dims / 2);
  a.rows = (int)(B * L);
  a.pos = p->positions;
  a.pos64 = p->positions_i64 != 0;
  a.pb = p->position_strides[0];
  a.pl = p->position_strides[1];
  a.pos0 = p->pos0;
  a.freqs = p->freqs;
  a.scale = p->scale;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dt == DSPARK_DTYPE_BF16) vec ? launch_rope<DSPARK_DTYPE_BF16, 8>(a, inter, s) : launch_rope<DSPARK_DTYPE_BF16, 1>(a, inter, s);
  else if (dt == DSPARK_DTYPE_F16) vec ? launch_rope<DSPARK_DTYPE_F16, 8>(a, inter, s) : launch_rope<DSPARK_DTYPE_F16, 1>(a, inter, s);
  else vec ? launch_rope<DSPARK_DTYPE_F32, 4>(a, inter, s) : launch_rope<DSPARK_DTYPE_F32, 1>(a, inter, s);
  return check_launch(what);
}
