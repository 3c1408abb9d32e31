// Host side of the attention over paged caches: launch rules and the C entry points.
#include <algorithm>
#include <cmath>

#include "dspark_paged_tiles.h"

namespace dspark {
namespace paged {
namespace {

struct Plan {
  int rt, workgroups, most_rows, whole, least;   // few rows (workgroups = 0: not launched)
  int rows_up_to;                                // of a sequence and KV head that are few
  unsigned items;                                // many rows: workgroups, 0: not launched
  size_t part_floats, tile_floats;
};

Plan make_plan(long B, long Hq, long Hk, long D, long T, long max_rows, long max_len, bool codes) {
  Plan p{};
  const long gqa = Hq / Hk, rows = std::min(T, max_rows) * gqa;
  const bool tiles_too = rows > (D == 256 ? 32 : 64);
  // Beside prompt chunks the few-rows kernel has decoded tokens only: one row tile, and what is more goes to the other.
  // Pages of the model's type up to head dim 128: both are bound by the bytes, and the one launch takes all (32 / 8 heads of
  // 128, a chunk of 512 rows and 31 tokens behind 100 to 8000: 182 -> 168 us, a chunk of 256 and 127 tokens 181 -> 150; a
  // chunk of 100 and three behind 30000 122 -> 129). 8-bit pages and head dim 256 lose: 137 -> 155 us, 236 -> 252.
  const bool one_launch = B == 1 || (!codes && D <= 128);
  p.rows_up_to = !tiles_too ? 1 << 30 : one_launch ? 0 : 16;
  p.rt = tiles_too || rows <= 16 ? 1 : rows <= 32 || D == 256 ? 2 : 4;
  if (tiles_too) {
    const long long_ones = std::min(B, T * gqa / (p.rows_up_to + 1) + 1);
    p.items = (unsigned)(((T * gqa / kTileRows + long_ones) * Hk + kParts + 7) / 8 * 8);
    p.tile_floats = (size_t)kParts * kTileRows * (D + 2);
    if (one_launch) return p;
  }
  const long tiles = (max_len + kUnit - 1) / kUnit, height = 16 * p.rt;
  const long groups = T * gqa / height + std::min(B, T);                // of all sequences, at most
  p.most_rows = (int)std::min(T * gqa, std::max(tiles_too ? 16L : rows, 1L));
  p.whole = tiles <= 4;
  p.least = p.rt == 4 ? 4 : 2;
  if (p.whole) {
    p.workgroups = (int)std::min(groups * Hk, 1L << 30);
  } else {
    p.workgroups = (int)std::min(p.rt * D > 256 || D == 256 ? 256L : 512L, std::max(1L, groups * Hk * tiles));
    p.part_floats = (size_t)p.workgroups * 2 * height * (D + 2);
  }
  return p;
}

int check(long B, long Hq, long Hk, long D, long T, long max_rows, long max_len) {
  if (D != 64 && D != 128 && D != 256) return fail(DSPARK_ERR_SHAPE, "paged_attention: head_dim %ld (64, 128 or 256)", D);
  if (B < 1 || B > 4096 || Hk < 1 || Hk > 1024 || Hq < 1 || Hq > 4096 || Hq % Hk || T < 1 || T >= (1 << 22) || max_rows < 1 ||
      max_len < 1 || max_len > (1 << 30))
    return fail(DSPARK_ERR_SHAPE, "paged_attention: B=%ld Hq=%ld Hk=%ld rows=%ld max_rows=%ld max_len=%ld", B, Hq, Hk, T, max_rows, max_len);
  const long groups = T * (Hq / Hk) / 16 + B;
  if (groups * Hk > (1 << 22) || groups * Hk * ((max_len + kUnit - 1) / kUnit) > (long)kMostUnits)
    return fail(DSPARK_ERR_SHAPE, "paged_attention: %ld rows of %ld sequences over %ld positions are too much for one call", T, B, max_len);
  return DSPARK_OK;
}

}  // namespace
}  // namespace paged
}  // namespace dspark

using namespace dspark;

extern "C" size_t dspark_paged_attention_workspace(int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t rows, int64_t max_rows,
                                                   int64_t max_len) {
  if (paged::check(B, Hq, Hk, D, rows, max_rows, max_len)) return 0;
  size_t floats = 64;
  for (const bool codes : {false, true}) {
    const paged::Plan p = paged::make_plan(B, Hq, Hk, D, rows, max_rows, max_len, codes);
    floats = std::max({floats, p.part_floats, p.tile_floats});
  }
  return floats * sizeof(float);
}

extern "C" int dspark_paged_attention(const dspark_paged_attention_args* p, dspark_stream stream) {
  const char* what = "paged_attention";
  if (!p || !p->q || !p->out || !p->workspace) return fail(DSPARK_ERR_ARG, "%s: null pointer", what);
  if (p->dtype != DSPARK_DTYPE_BF16 && p->dtype != DSPARK_DTYPE_F16)
    return fail(DSPARK_ERR_UNSUPPORTED, "%s: dtype %ld", what, (long)p->dtype);
  if (!(p->scale > 0.0) || !std::isfinite((float)p->scale) || (float)p->scale == 0.f)
    return fail(DSPARK_ERR_ARG, "%s: scale %g (finite and > 0)", what, p->scale);
  paged::AttnArgs a = {};
  const bool codes = p->codes != 0;
  int st = paged::check_pool(what, p->pool, p->Hk, p->P, p->D);
  if (st || (st = paged::take_seqs(what, &p->seqs, p->P, p->pool, &a.s))) return st;
  const long max_len = (long)a.s.width * a.s.P;
  if ((st = paged::check(a.s.B, p->Hq, p->Hk, p->D, a.s.T, p->max_rows, max_len)) ||
      (st = paged::take_pages(what, &p->k_pages, p->pool, p->Hk, p->P, p->D, codes, &a.k)) ||
      (st = paged::take_pages(what, &p->v_pages, p->pool, p->Hk, p->P, p->D, codes, &a.v)))
    return st;
  for (int i = 0; i < 2; ++i)
    if (p->q_strides[i] % 8 || p->out_strides[i] % 8)
      return fail(DSPARK_ERR_ALIGN, "%s: strides of queries and outputs must be multiples of 16 bytes", what);
  if (!aligned(p->q, 16) || !aligned(p->out, 16) || !aligned(p->workspace, 16))
    return fail(DSPARK_ERR_ALIGN, "%s: queries, outputs and workspace must be 16-byte aligned", what);
  const paged::Plan plan = paged::make_plan(a.s.B, p->Hq, p->Hk, p->D, a.s.T, p->max_rows, max_len, codes);
  const size_t need = std::max(plan.part_floats, plan.tile_floats) * sizeof(float);      // one after the other
  if ((size_t)p->workspace_bytes < need)
    return fail(DSPARK_ERR_WORKSPACE, "%s: workspace %ld < %zu bytes", what, (long)p->workspace_bytes, need);
  a.q = static_cast<const u16*>(p->q);
  a.out = static_cast<u16*>(p->out);
  a.qrow = p->q_strides[0], a.qhead = p->q_strides[1];
  a.orow = p->out_strides[0], a.ohead = p->out_strides[1];
  a.opart = static_cast<float*>(p->workspace);
  a.mpart = a.opart + (size_t)plan.workgroups * 2 * 16 * plan.rt * p->D;
  a.Hq = (int)p->Hq;
  a.Hk = (int)p->Hk;
  a.gqa = a.Hq / a.Hk;
  a.causal = p->causal != 0;
  a.whole = plan.whole;
  a.least = plan.least;
  a.rows_up_to = plan.rows_up_to;
  a.clear = p->clear != 0;
  a.scale_log2 = (float)(p->scale * 1.44269504088896340736);
  hipStream_t s = static_cast<hipStream_t>(stream);
  using paged::BF16;
  using paged::F16;
  const bool bf = p->dtype == DSPARK_DTYPE_BF16;
  if (plan.workgroups) {
#define DSPARK_PAGED_CALL(D) \
  (bf ? paged::launch<BF16, D>(a, plan.rt, codes, plan.workgroups, plan.most_rows, s) \
      : paged::launch<F16, D>(a, plan.rt, codes, plan.workgroups, plan.most_rows, s))
    st = p->D == 64 ? DSPARK_PAGED_CALL(64) : p->D == 128 ? DSPARK_PAGED_CALL(128) : DSPARK_PAGED_CALL(256);
#undef DSPARK_PAGED_CALL
    if (st) return st;
    a.clear = 0;
  }
  if (!plan.items) return DSPARK_OK;
  paged::TileArgs ta{a, static_cast<float*>(p->workspace), nullptr};
  ta.mpart = ta.opart + (size_t)paged::kParts * paged::kTileRows * p->D;
#define DSPARK_PAGED_CALL(D) \
  (bf ? paged::launch_tiles<BF16, D>(ta, codes, plan.items, s) : paged::launch_tiles<F16, D>(ta, codes, plan.items, s))
  return p->D == 64 ? DSPARK_PAGED_CALL(64) : p->D == 128 ? DSPARK_PAGED_CALL(128) : DSPARK_PAGED_CALL(256);
#undef DSPARK_PAGED_CALL
}
