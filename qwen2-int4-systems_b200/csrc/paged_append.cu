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
// A thread owns one unit at a time: 16 dimensions of one head of one token, as
// two 16-byte chunks that hold whole pairs (the chunks m and m + rot/2 of 8
// dimensions each, or two adjacent chunks), so that both layouts read the same
// 8 cosines and sines and no value passes between threads. Bound by memory
// (each byte is read and written once). A CTA owns up to 64 tokens; one thread
// per token follows the chain boundaries -> sequence -> length -> page that
// says where it goes, three dependent loads, once per CTA and behind the first
// two units' loads of every thread; from there each thread has the loads of
// two units ahead of it under way. Measured (device time): ragged prompts of up
// to 4001 tokens, 24 heads of 128 dims, 81 us (5.6 TB/s); one token each of 64
// sequences 2.8 us.
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
  FastDiv by_units, by_head, by_per_seq;
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

// The sequence of token t (the number of sequences that end at or before it,
// so that empty ones are passed over), or -1 where no sequence has it.
__device__ __forceinline__ int owner_of(const Ragged& r, const FastDiv& by_per_seq, int t) {
  if (!r.cu) return by_per_seq(t);
  int lo = 0, hi = r.B;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(r.cu + mid + 1) <= t)
      lo = mid + 1;
    else
      hi = mid;
  }
  if (lo >= r.B) return -1;
  const Tokens s = seq_tokens(r, lo);
  return t >= s.first && t < s.first + s.count ? lo : -1;
}

struct Unit {
  int64_t t;
  int tk, h, c0, c1;  // token of the CTA, head (q, then k, then v), the two chunks' dimensions
  bool turned;
  int u;
};

template <bool F16>
__global__ void __launch_bounds__(kThreads, 4) append_kernel(const AppendArgs a) {
  __shared__ int64_t slot_of[kMaxTokens];  // element offset of the token's slot in the pool, or -1
  __shared__ int row_of[kMaxTokens];       // row of cos / sin
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int units = (a.Hq + 2 * a.Hkv) * a.units_per_head;
  const int t0 = blockIdx.x * a.tokens_per_cta;
  const int nt = min(a.tokens_per_cta, a.r.T - t0);
  const int total = nt * units;

  auto unit = [&](int idx) {
    Unit x;
    x.tk = a.by_units(idx);
    const int rest = idx - x.tk * units;
    x.h = a.by_head(rest);
    x.u = rest - x.h * a.units_per_head;
    x.t = t0 + x.tk;
    x.turned = x.h < a.Hq + a.Hkv && x.u < a.rot_units;
    const bool halves = x.turned && !a.interleaved;
    x.c0 = halves ? 8 * x.u : 16 * x.u;
    x.c1 = halves ? x.c0 + a.half : x.c0 + 8;
    return x;
  };
  auto fetch = [&](int idx, uint4& lo, uint4& hi) {
    if (idx >= total) return;
    const Unit x = unit(idx);
    const uint16_t* src = x.h < a.Hq ? a.q + x.t * a.q_tok + x.h * a.q_head
                          : x.h < a.Hq + a.Hkv ? a.k + x.t * a.k_tok + (x.h - a.Hq) * a.k_head
                                               : a.v + x.t * a.v_tok + (x.h - a.Hq - a.Hkv) * a.v_head;
    lo = *reinterpret_cast<const uint4*>(src + x.c0);
    hi = *reinterpret_cast<const uint4*>(src + x.c1);
  };
  auto place = [&](int idx, uint4 w0, uint4 w1) {
    if (idx >= total) return;
    const Unit x = unit(idx);
    if (x.turned) {
      const float4* cp = reinterpret_cast<const float4*>(a.cos + (int64_t)row_of[x.tk] * a.half + 8 * x.u);
      const float4* sp = reinterpret_cast<const float4*>(a.sin + (int64_t)row_of[x.tk] * a.half + 8 * x.u);
      const float4 ca = __ldg(cp), cb = __ldg(cp + 1), sa = __ldg(sp), sb = __ldg(sp + 1);
      const float c[8] = {ca.x, ca.y, ca.z, ca.w, cb.x, cb.y, cb.z, cb.w};
      const float s[8] = {sa.x, sa.y, sa.z, sa.w, sb.x, sb.y, sb.z, sb.w};
      float e[8], f[8], re[8], rf[8];
      unpack<F16>(w0, e);
      unpack<F16>(w1, f);
      if (a.interleaved) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          re[2 * m] = e[2 * m] * c[m] - e[2 * m + 1] * s[m];
          re[2 * m + 1] = e[2 * m + 1] * c[m] + e[2 * m] * s[m];
          rf[2 * m] = f[2 * m] * c[m + 4] - f[2 * m + 1] * s[m + 4];
          rf[2 * m + 1] = f[2 * m + 1] * c[m + 4] + f[2 * m] * s[m + 4];
        }
      } else {
#pragma unroll
        for (int m = 0; m < 8; ++m) {
          re[m] = e[m] * c[m] - f[m] * s[m];
          rf[m] = f[m] * c[m] + e[m] * s[m];
        }
      }
      w0 = pack<F16>(re);
      w1 = pack<F16>(rf);
    }
    uint16_t* dst;
    if (x.h < a.Hq) {
      dst = a.q_out + x.t * a.o_tok + x.h * a.o_head;
    } else {
      if (slot_of[x.tk] < 0) return;
      const bool key = x.h < a.Hq + a.Hkv;
      dst = (key ? a.k_pages : a.v_pages) + slot_of[x.tk] + (int64_t)(x.h - a.Hq - (key ? 0 : a.Hkv)) * a.head_stride;
    }
    *reinterpret_cast<uint4*>(dst + x.c0) = w0;
    *reinterpret_cast<uint4*>(dst + x.c1) = w1;
  };

  uint4 lo[2], hi[2];
  fetch(tid, lo[0], hi[0]);
  fetch(tid + kThreads, lo[1], hi[1]);
  if (tid < nt) {
    const int t = t0 + tid, b = owner_of(a.r, a.by_per_seq, t);
    int64_t slot = -1;
    int row = 0;
    if (b >= 0) {
      const int64_t at = (int64_t)__ldg(a.r.lengths + b) + (t - seq_tokens(a.r, b).first);
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
    slot_of[tid] = slot;
    row_of[tid] = row;
  }
  __syncthreads();
  for (int base = tid; base < total; base += 2 * kThreads) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 w0 = lo[i], w1 = hi[i];
      fetch(base + (i + 2) * kThreads, lo[i], hi[i]);
      place(base + i * kThreads, w0, w1);
    }
  }
}

template <bool F16>
cudaError_t launch_append(const AppendArgs& a0, int sms, cudaStream_t stream) {
  AppendArgs a = a0;
  const int units = (a.Hq + 2 * a.Hkv) * a.units_per_head;
  // Few tokens per CTA while that gives every SM work (the chain above is then
  // the whole time), six rounds of units once the call fills the GPU: 36,238
  // tokens of 24 heads x 128 take 88 us with three rounds, 81 with six, 82 with
  // twelve (454 MB: 5.6 TB/s), 64 decode steps 2.8.
  const int64_t all = (int64_t)a.r.T * units;
  const int64_t per_cta = all <= (int64_t)sms * 4 * kThreads ? kThreads : 6 * kThreads;
  a.tokens_per_cta = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxTokens, per_cta / units));
  a.by_units = FastDiv::of(units);
  a.by_head = FastDiv::of(a.units_per_head);
  a.by_per_seq = FastDiv::of(a.r.per_seq);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.r.T + a.tokens_per_cta - 1) / a.tokens_per_cta), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, append_kernel<F16>, a);
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
      kv->page_stride < (kv->pages > 1) || kv->head_stride < (kv->kv_heads > 1) || kv->slot_stride < kv->head_dim) {
    set_error("%s: pages must be 16-byte aligned, with positive strides that are multiples of 8 elements", what);
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
  // Tokens or heads that share their memory can be read, but not written.
  ok = ok && out_token_stride >= (Hq && T > 1) && out_head_stride >= (Hq > 1);
  if (!ok) {
    set_error("rotary append: q, k, v, q_out, cos and sin must be 16-byte aligned, with token and head strides that "
              "are multiples of 8 elements, those of q_out positive");
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
