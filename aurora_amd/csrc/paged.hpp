// What the paged K/V cache's kernels share: argument checks, the walk from a
// token to its sequence, and the elements of the pools.
#pragma once

#include "common.hpp"

namespace aurpaged {

// Sequence s of a batch, with every device value clamped to the host's bounds,
// so that a wrong length or offset reads and writes nothing out of range.
struct Seq {
  int lo, n;  // its first row among the new tokens, and their number
  int len;    // own tokens in the cache, the new ones among them
};

struct Batch {
  const int32_t* tok_off;
  const int32_t* own_len;
  const int32_t* pages;
  const int32_t* prefix_pages;
  int b, max_pages, n_tok, max_tok, max_own, prefix_len;
};

__device__ __forceinline__ Seq sequence(const Batch& a, int s) {
  Seq q;
  q.lo = min(max(a.tok_off[s], 0), a.n_tok);
  q.n = min(min(max(a.tok_off[s + 1], q.lo), a.n_tok) - q.lo, a.max_tok);
  q.len = min(max(a.own_len[s], 0), a.max_own);
  return q;
}

// The sequence of row t: how many sequences end at or before it (b: none holds it).
// For a whole block; every thread gets the answer.
__device__ __forceinline__ int sequence_of(const Batch& a, int t) {
  int s = 0;
  for (int i0 = 0; i0 < a.b; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    s += __syncthreads_count(i < a.b && a.tok_off[i + 1] <= t);
  }
  return s;
}

// Elements of a pool held in 8 bits: e4m3 numbers (sign, 4 bits of exponent, 3 of significand; up to 448 and down
// to 2^-9, a NaN, no infinity) times a power of two of their own for every 2^ssh tokens of a head, held as the
// byte e + 127 of 2^e.  A pool row's scales lie apart, [n_pages][n_kv_head][page_len >> ssh].
struct e4m3 {
  uint8_t bits;
};
__device__ __forceinline__ size_t scale_index(int row, int hk, int n_kv_head, int sh, int ssh) {
  return (((size_t)(row >> sh) * n_kv_head + hk) << (sh - ssh)) + ((row & ((1 << sh) - 1)) >> ssh);
}
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

// Work items of a launch stay below 2^32: so many blocks of 256.
constexpr uint32_t kMaxBlocks = 0x00ffffffu;

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Checks what the host can see of a cache and a batch and fills `out`; 0 or an error code.
int check_paged(aur_ctx* ctx, const char* who, const aur_paged_cache* c, const aur_paged_batch* b, Batch* out);

inline int log2_of(uint32_t pow2) { return __builtin_ctz(pow2); }

}  // namespace aurpaged
