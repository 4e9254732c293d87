// Types shared by the paged-cache operators (rotary append, attention).
//
// One layer's cache is a pool of pages, each holding `page_size` consecutive
// positions of one sequence for every KV head; block_table[b][j] names the
// page of positions j * page_size .. of sequence b. A batch is ragged: its
// new tokens are the rows of one [T, heads, D] tensor, sequence b owning rows
// cu_tokens[b] .. cu_tokens[b + 1] (or T / B rows each where cu_tokens is
// null).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "qi4_common.cuh"

namespace qi4 {

// The sequences of a launch. All of it is checked against T on use: whatever
// the arrays hold, no token index leaves [0, T).
struct Ragged {
  const int32_t* cu;       // [B + 1], or null: `per_seq` tokens each
  const int32_t* lengths;  // [B]
  int B, T, per_seq;
};

struct Tokens {
  int first, count;
};

__device__ __forceinline__ Tokens seq_tokens(const Ragged& r, int b) {
  if (!r.cu) return {b * r.per_seq, r.per_seq};
  const int t0 = min(max(__ldg(r.cu + b), 0), r.T);
  const int t1 = min(max(__ldg(r.cu + b + 1), t0), r.T);
  return {t0, t1 - t0};
}

// x / d for 0 <= x < 2^31 as a product and a shift (d set on the host): an
// integer division costs some 150 cycles of latency, and the work split, which
// runs before a kernel's first load, would hold ten of them.
struct FastDiv {
  unsigned mul, shift;  // mul 0: d = 1
  static FastDiv of(int64_t d) {
    if (d <= 1) return {0u, 0u};
    unsigned log = 0;
    while ((1ll << log) < d) ++log;
    // ceil(2^(31 + log) / d) is below 2^32, and exact for x below 2^31.
    return {(unsigned)(((1ull << (31 + log)) + (unsigned long long)d - 1) / (unsigned long long)d), log - 1};
  }
  __device__ __forceinline__ int operator()(int x) const { return mul ? (int)(__umulhi((unsigned)x, mul) >> shift) : x; }
};

// Device-side error bits of the paged operators (read by qi4_device_status).
constexpr int kErrCacheFull = QI4_DEVICE_CACHE_FULL;
constexpr int kErrBadPage = QI4_DEVICE_BAD_PAGE;
constexpr int kErrBadPosition = QI4_DEVICE_BAD_POSITION;

// Checks of a qi4_paged_kv that every operator makes (host); 0 or a QI4_ERR_* code.
int check_paged_kv(const qi4_paged_kv* kv, const char* what);

// SMs of the current device, once it is known to be an sm_100; 0 or a QI4_ERR_* code.
int require_device(int* sms);

// Reads and clears one translation unit's device error word on `stream` (synchronises).
int read_error_word(const void* symbol, cudaStream_t stream);

}  // namespace qi4
