// Rotary positions on new queries and keys, and the append of the new keys
// and values to a paged cache (sm_100a).
//
// Per token at position p of its sequence, for every query and key head x:
//   y[i]  = x[i] c - x[j] s,   y[j] = x[j] c + x[i] s,   c, s = cos, sin[row][m]
// over the m = 0 .. rot/2 - 1 pairs (i, j) = (m, m + rot/2), or (2m, 2m + 1)
// when interleaved; dimensions from rot on are copied. The products and sums
// are FP32 and each result is rounded once to the cache's type. The key and
// the value go to slot p % page_size of page block_table[b][p / page_size].
//
// A thread owns one unit: 16 dimensions of one head of one token, as two
// 16-byte chunks that hold whole pairs (the chunks m and m + rot/2 of 8
// dimensions each, or two adjacent chunks), so that both layouts read the
// same 8 cosines and sines and no value passes between threads. Bound by
// memory (each byte is read and written once); the loads of a thread's units
// are issued before the chain sequence -> length -> page that finds where
// they go, which is three dependent loads and the whole time of a small call.
#include <algorithm>

#include "paged.cuh"

namespace qi4 {

__device__ int g_append_error;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 64;  // tokens a CTA owns at most

struct AppendArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* q_out;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;  // strides, elements
  uint16_t* k_pages;
  uint16_t* v_pages;
  int64_t page_stride, head_stride, slot_stride;
  const int32_t* table;
  int64_t table_stride;
  int table_width, pages, page_size, page_shift;
  Ragged r;
  const int32_t* positions;  // [T] rows of cos / sin, or null: the position in the sequence
  const float* cos;
  const float* sin;
  int rope_rows, rot_units, half;  // rot / 16, rot / 2
  int Hq, Hkv, units_per_head;     // D / 16
  int tokens_per_cta;
  int interleaved;
};

template <bool F16>
__device__ __forceinline__ void unpack(uint4 w, float (&x)[8]) {
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(a[i] << 16);
      x[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
    }
  }
}

template <bool F16>
__device__ __forceinline__ uint4 pack(const float (&x)[8]) {
  uint32_t a[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F16)
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(a[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    else
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(a[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
  }
  return make_uint4(a[0], a[1], a[2], a[3]);
}

// The sequence of token t: the number of sequences that end at or before it
// (empty ones are passed over), counted by the warp 32 boundaries at a time.
__device__ __forceinline__ int owner_of(const Ragged& r, int t, int lane) {
  if (!r.cu) return t / r.per_seq;
  int before = 0;
  for (int j = lane; j < r.B; j += 32) before += __ldg(r.cu + j + 1) <= t;
  return __reduce_add_sync(0xffffffffu, before);
}

// ITER units per thread in flight.
template <bool F16, int ITER>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a) {
  __shared__ int64_t slot_of[kMaxTokens];  // element offset of the token's slot in the pool, or -1
  __shared__ int row_of[kMaxTokens];       // row of cos / sin
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int heads = a.Hq + 2 * a.Hkv, units = heads * a.units_per_head;
  const int t0 = blockIdx.x * a.tokens_per_cta;
  const int nt = min(a.tokens_per_cta, a.r.T - t0);
  const int total = nt * units;

  for (int base = 0; base < total; base += kThreads * ITER) {
    uint4 lo[ITER], hi[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int idx = base + i * kThreads + tid;
      if (idx >= total) break;
      const int tk = idx / units, rest = idx - tk * units, h = rest / a.units_per_head,
                u = rest - h * a.units_per_head;
      const int64_t t = t0 + tk;
      const uint16_t* src = h < a.Hq ? a.q + t * a.q_tok + h * a.q_head
                            : h < a.Hq + a.Hkv ? a.k + t * a.k_tok + (h - a.Hq) * a.k_head
                                               : a.v + t * a.v_tok + (h - a.Hq - a.Hkv) * a.v_head;
      const bool halves = h < a.Hq + a.Hkv && u < a.rot_units && !a.interleaved;
      const int c0 = halves ? 8 * u : 16 * u, c1 = halves ? c0 + a.half : c0 + 8;
      lo[i] = *reinterpret_cast<const uint4*>(src + c0);
      hi[i] = *reinterpret_cast<const uint4*>(src + c1);
    }
    if (base == 0) {  // where the CTA's tokens go, one warp per token at a time
      for (int j = warp; j < nt; j += kThreads / 32) {
        const int t = t0 + j;
        const int b = owner_of(a.r, t, lane);
        if (lane == 0) {
          int64_t slot = -1;
          int row = 0;
          if (b < a.r.B) {
            const Tokens s = seq_tokens(a.r, b);
            const int64_t at = (int64_t)__ldg(a.r.lengths + b) + (t - s.first);
            const int64_t pj = at >> a.page_shift;
            if (at < 0 || pj >= a.table_width) {
              atomicOr(&g_append_error, kErrCacheFull);
            } else {
              const int page = __ldg(a.table + b * a.table_stride + pj);
              if (page < 0 || page >= a.pages)
                atomicOr(&g_append_error, kErrBadPage);
              else
                slot = (int64_t)page * a.page_stride + (at & (a.page_size - 1)) * a.slot_stride;
            }
            const int64_t want = a.positions ? (int64_t)__ldg(a.positions + t) : at;
            row = (int)max((int64_t)0, min(want, (int64_t)a.rope_rows - 1));
            if (want != row && a.rot_units) atomicOr(&g_append_error, kErrBadPosition);
          }
          slot_of[j] = slot;
          row_of[j] = row;
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int idx = base + i * kThreads + tid;
      if (idx >= total) break;
      const int tk = idx / units, rest = idx - tk * units, h = rest / a.units_per_head,
                u = rest - h * a.units_per_head;
      const int64_t t = t0 + tk;
      const bool turned = h < a.Hq + a.Hkv && u < a.rot_units;
      const bool halves = turned && !a.interleaved;
      const int c0 = halves ? 8 * u : 16 * u, c1 = halves ? c0 + a.half : c0 + 8;
      uint4 w0 = lo[i], w1 = hi[i];
      if (turned) {
        const float4* cp = reinterpret_cast<const float4*>(a.cos + (int64_t)row_of[tk] * a.half + 8 * u);
        const float4* sp = reinterpret_cast<const float4*>(a.sin + (int64_t)row_of[tk] * a.half + 8 * u);
        const float4 ca = __ldg(cp), cb = __ldg(cp + 1), sa = __ldg(sp), sb = __ldg(sp + 1);
        const float c[8] = {ca.x, ca.y, ca.z, ca.w, cb.x, cb.y, cb.z, cb.w};
        const float s[8] = {sa.x, sa.y, sa.z, sa.w, sb.x, sb.y, sb.z, sb.w};
        float x[8], y[8], rx[8], ry[8];
        unpack<F16>(w0, x);
        unpack<F16>(w1, y);
        if (a.interleaved) {
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            rx[2 * m] = x[2 * m] * c[m] - x[2 * m + 1] * s[m];
            rx[2 * m + 1] = x[2 * m + 1] * c[m] + x[2 * m] * s[m];
            ry[2 * m] = y[2 * m] * c[m + 4] - y[2 * m + 1] * s[m + 4];
            ry[2 * m + 1] = y[2 * m + 1] * c[m + 4] + y[2 * m] * s[m + 4];
          }
        } else {
#pragma unroll
          for (int m = 0; m < 8; ++m) {
            rx[m] = x[m] * c[m] - y[m] * s[m];
            ry[m] = y[m] * c[m] + x[m] * s[m];
          }
        }
        w0 = pack<F16>(rx);
        w1 = pack<F16>(ry);
      }
      uint16_t* dst;
      if (h < a.Hq) {
        dst = a.q_out + t * a.o_tok + h * a.o_head;
      } else {
        if (slot_of[tk] < 0) continue;
        const bool key = h < a.Hq + a.Hkv;
        dst = (key ? a.k_pages : a.v_pages) + slot_of[tk] +
              (int64_t)(h - a.Hq - (key ? 0 : a.Hkv)) * a.head_stride;
      }
      *reinterpret_cast<uint4*>(dst + c0) = w0;
      *reinterpret_cast<uint4*>(dst + c1) = w1;
    }
  }
}

template <bool F16>
cudaError_t launch_append(const AppendArgs& a0, int sms, cudaStream_t stream) {
  AppendArgs a = a0;
  const int units = (a.Hq + 2 * a.Hkv) * a.units_per_head;
  // Two units in flight per thread once the call fills the GPU several times
  // over, one (the shortest path) below.
  const bool wide = (int64_t)a.r.T * units > (int64_t)sms * 8 * kThreads;
  a.tokens_per_cta = std::max(1, std::min(kMaxTokens, kThreads * (wide ? 2 : 1) / units));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.r.T + a.tokens_per_cta - 1) / a.tokens_per_cta), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return wide ? cudaLaunchKernelEx(&cfg, append_kernel<F16, 2>, a) : cudaLaunchKernelEx(&cfg, append_kernel<F16, 1>, a);
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int read_append_error(cudaStream_t stream) { return read_error_word(&g_append_error, stream); }

int check_paged_kv(const qi4_paged_kv* kv, const char* what) {
  if (!kv || !kv->k || !kv->v || !kv->block_table) {
    set_error("%s: the cache descriptor, its pages and its block table must be non-null", what);
    return QI4_ERR_ARGUMENT;
  }
  if (kv->dtype != QI4_DTYPE_F16 && kv->dtype != QI4_DTYPE_BF16) {
    set_error("%s takes FP16 or BF16 pages", what);
    return QI4_ERR_DTYPE;
  }
  if (kv->pages <= 0 || kv->kv_heads <= 0 || kv->head_dim <= 0 || kv->table_width <= 0 || kv->table_stride < 0) {
    set_error("%s: pages, kv_heads, head_dim and the table's width must be positive", what);
    return QI4_ERR_ARGUMENT;
  }
  if (kv->page_size < 8 || kv->page_size > 1024 || (kv->page_size & (kv->page_size - 1))) {
    set_error("%s: page_size must be a power of two from 8 to 1024 (got %d)", what, kv->page_size);
    return QI4_ERR_SHAPE;
  }
  if ((int64_t)kv->table_width * kv->page_size > (1ll << 30)) {
    set_error("%s: a block table covers at most 2^30 positions", what);
    return QI4_ERR_SHAPE;
  }
  if (!al16(kv->k) || !al16(kv->v) || kv->page_stride % 8 || kv->head_stride % 8 || kv->slot_stride % 8 ||
      kv->page_stride < 0 || kv->head_stride < 0 || kv->slot_stride < kv->head_dim) {
    set_error("%s: pages must be 16-byte aligned, with strides that are multiples of 8 elements", what);
    return QI4_ERR_ALIGNMENT;
  }
  return QI4_OK;
}

}  // namespace qi4

extern "C" QI4_API int qi4_rope_paged_append(const qi4_paged_kv* kv, const void* q, int64_t q_token_stride,
                                             int64_t q_head_stride, const void* k, int64_t k_token_stride,
                                             int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                             int64_t v_head_stride, void* q_out, int64_t out_token_stride,
                                             int64_t out_head_stride, int64_t T, int64_t B, int64_t Hq,
                                             const int32_t* cu_tokens, const int32_t* lengths,
                                             const int32_t* positions, const float* cos, const float* sin,
                                             int64_t rope_rows, int rot_dim, int interleaved, void* stream) {
  using namespace qi4;
  clear_error();
  int rc = check_paged_kv(kv, "rotary append");
  if (rc) return rc;
  if (T < 0 || B <= 0 || Hq < 0 || T > (1ll << 30) || B > (1ll << 30) || Hq > 65535) {
    set_error("rotary append: B must be positive and T, Hq not negative (at most 2^30, 65535)");
    return QI4_ERR_ARGUMENT;
  }
  if (T == 0) return QI4_OK;
  if (!k || !v || !lengths || (Hq && (!q || !q_out))) {
    set_error("rotary append: q, k, v, lengths and q_out must be non-null");
    return QI4_ERR_ARGUMENT;
  }
  if (!cu_tokens && T % B) {
    set_error("rotary append: without cu_tokens every sequence has T / B tokens (got T = %lld, B = %lld)",
              (long long)T, (long long)B);
    return QI4_ERR_SHAPE;
  }
  if (kv->head_dim % 16 || kv->head_dim > 1024 || rot_dim < 0 || rot_dim % 16 || rot_dim > kv->head_dim) {
    set_error("rotary append: head_dim must be a multiple of 16 (at most 1024) and rot_dim a multiple of 16 up to "
              "it (got %d, %d)", kv->head_dim, rot_dim);
    return QI4_ERR_SHAPE;
  }
  if (rot_dim && (!cos || !sin || rope_rows <= 0 || rope_rows > (1ll << 30))) {
    set_error("rotary append: cos and sin must be non-null with at least one row");
    return QI4_ERR_ARGUMENT;
  }
  const int64_t strides[] = {q_token_stride, q_head_stride,  k_token_stride,   k_head_stride,
                             v_token_stride, v_head_stride, out_token_stride, out_head_stride};
  bool ok = al16(q) && al16(k) && al16(v) && al16(q_out) && al16(cos) && al16(sin);
  for (int64_t s : strides) ok = ok && s % 8 == 0 && s >= 0;
  if (!ok) {
    set_error("rotary append: q, k, v, q_out, cos and sin must be 16-byte aligned, with token and head strides that "
              "are multiples of 8 elements");
    return QI4_ERR_ALIGNMENT;
  }
  int sms = 0;
  rc = require_device(&sms);
  if (rc) return rc;
  AppendArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.q_tok = q_token_stride, a.q_head = q_head_stride;
  a.k_tok = k_token_stride, a.k_head = k_head_stride;
  a.v_tok = v_token_stride, a.v_head = v_head_stride;
  a.o_tok = out_token_stride, a.o_head = out_head_stride;
  a.k_pages = static_cast<uint16_t*>(kv->k);
  a.v_pages = static_cast<uint16_t*>(kv->v);
  a.page_stride = kv->page_stride, a.head_stride = kv->head_stride, a.slot_stride = kv->slot_stride;
  a.table = kv->block_table, a.table_stride = kv->table_stride, a.table_width = kv->table_width;
  a.pages = kv->pages, a.page_size = kv->page_size, a.page_shift = __builtin_ctz((unsigned)kv->page_size);
  a.r = {cu_tokens, lengths, (int)B, (int)T, (int)(T / B)};
  a.positions = positions;
  a.cos = cos, a.sin = sin, a.rope_rows = (int)rope_rows;
  a.rot_units = rot_dim / 16, a.half = rot_dim / 2;
  a.Hq = (int)Hq, a.Hkv = kv->kv_heads, a.units_per_head = kv->head_dim / 16;
  a.interleaved = interleaved ? 1 : 0;
  a.tokens_per_cta = 1;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = kv->dtype == QI4_DTYPE_F16 ? launch_append<true>(a, sms, s) : launch_append<false>(a, sms, s);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("rotary append launch failed: %s", cudaGetErrorString(e));
    return QI4_ERR_LAUNCH;
  }
  return QI4_OK;
}
