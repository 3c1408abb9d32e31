// Paged key/value caches: what the kernels that append to them, attend over them and read them share (gfx950).
//
// A cache is a pool of pages of P positions (a power of two) for every KV head; sequence b's position p lies in row
// p % P of page table[b][p / P]. A step's rows of all sequences stand one after the other: starts[b] .. starts[b + 1] - 1
// are sequence b's, the last ones of the lens[b] positions that it has with them. Pages are of the model's type, or hold
// e4m3 codes c that stand for c 2^E, with one exponent E for each page and head (e8m0: a byte E + 127, NaN for 255). With a power of
// two the codes' own precision is all there is to lose: a page whose exponent grows shifts its codes' exponents, and
// nothing is rounded that stays normal.
//
// starts, lens, table and page ids come from device memory: whatever they hold, nothing outside the tensors is read or
// written. A sequence whose rows are not within the call's has none; positions before the first, past the table or in a
// page that the pool does not have are not there.
#pragma once

#include "dspark_common.h"

namespace dspark {
namespace paged {

constexpr int kLeastExp = -110;  // of a page: its smallest code stands for 2^-119, which bf16 and fp32 have as a normal number

struct Pages {                   // keys or values
  char* data;                    // elements of the model's type, or codes
  unsigned char* exps;           // null: the model's type
  long page, head, row;          // strides in elements
  long epage, ehead;
};

// 2^(e - 127), NaN for 255: what a scale byte stands for
__device__ __forceinline__ float scale_of(u32 e) {
  return __builtin_bit_cast(float, e == 0 ? 0x400000u : e == 255 ? 0x7FC00000u : e << 23);
}

// The sequences of a call
struct Seqs {
  const int* table;              // [B][width], row stride ldt
  const int* starts;             // [B + 1]
  const int* lens;               // [B]
  long ldt;
  int B, width, T;               // T: rows of the call
  int P, log2P, pool;            // positions of a page, pages of the pool
};

struct Seq {
  int start, n, len;             // first row, rows, positions with them that the table has; n = 0 where they do not fit
  int full;                      // positions as given: the rows' own count from there
};

__device__ __forceinline__ Seq sequence(const Seqs& s, int b) {
  const int s0 = s.starts[b], s1 = s.starts[b + 1], len = s.lens[b];
  const bool ok = s0 >= 0 && s1 > s0 && s1 <= s.T && len > 0;
  const long most = (long)s.width << s.log2P;
  return Seq{s0, ok ? s1 - s0 : 0, (int)((long)len < most ? (long)len : most), len};
}

__device__ __forceinline__ long first_position(const Seq& q) { return (long)q.full - q.n; }

// Every row of the call is a sequence's: what a step usually is
__device__ __forceinline__ bool all_rows_taken(const Seqs& s) {
  const int lane = __lane_id();
  bool open = s.starts[0] != 0 || s.starts[s.B] != s.T;
  for (int b = lane; b < s.B; b += 64) {
    const int s0 = s.starts[b], s1 = s.starts[b + 1];
    open |= s1 < s0 || (s1 > s0 && s.lens[b] <= 0);
  }
  return !__builtin_amdgcn_ballot_w64(open);
}

// The page of a sequence's position, -1 where there is none
__device__ __forceinline__ int page_of(const Seqs& s, int b, long pos) {
  if (pos < 0 || pos >= ((long)s.width << s.log2P)) return -1;
  const int id = s.table[b * s.ldt + (pos >> s.log2P)];
  return (unsigned)id < (unsigned)s.pool ? id : -1;
}

// Sum of v over the lanes up to this one, at most 2^32 - 1
__device__ __forceinline__ u32 wave_scan(u32 v) {
  const int lane = __lane_id();
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u32 o = (u32)__builtin_amdgcn_ds_bpermute((lane - d) << 2, (int)v);
    v = __builtin_elementwise_add_sat(v, lane >= d ? o : 0u);
  }
  return v;
}

// The sequence that holds item `item` of a list in which every sequence b has count(b) items, and the item's place among
// them. Every wave finds it for itself; false past the list's end.
template <class F>
__device__ __forceinline__ bool locate(u32 item, int B, F count, int& b, int& local) {
  const int lane = __lane_id();
  for (int b0 = 0; b0 < B; b0 += 64) {
    const u32 c = b0 + lane < B ? count(b0 + lane) : 0u;
    const u32 upto = wave_scan(c);
    const u32 all = (u32)__builtin_amdgcn_readlane((int)upto, 63);
    if (item < all) {
      const int first = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > item));
      b = uniform(b0 + first);
      local = uniform((int)(item - (u32)__builtin_amdgcn_readlane((int)(upto - c), first)));
      return true;
    }
    item -= all;
  }
  return false;
}

// The parts of the entry points' arguments, checked (a dspark_status); defined in dspark_paged_append.hip
int check_pool(const char* what, int64_t pool, int64_t Hk, int64_t P, int64_t D);
int take_pages(const char* what, const dspark_pages* p, int64_t pool, int64_t Hk, int64_t P, int64_t D, bool codes, Pages* out);
int take_seqs(const char* what, const dspark_sequences* p, int64_t P, int64_t pool, Seqs* out);

}  // namespace paged
}  // namespace dspark
