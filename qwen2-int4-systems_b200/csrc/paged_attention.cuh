// Work split and partial-result merging of the paged attention kernels.
//
// A batch is cut into items - one row tile (R consecutive rows of one
// sequence's tokens x the G query heads of one KV head, row = token * G + head)
// of one KV head - and every item into units of kBlockKeys keys. The units of
// all items, in one line, are dealt to the CTAs in equal runs, so sequences of
// any mixture of lengths keep all SMs equally busy; a CTA's run may end inside
// an item. An item wholly inside one run is finished there; the pieces of
// another go to a workspace as (weighted sums, max, sum of weights) and the
// CTA that delivers the last piece merges them all, in the order of the runs,
// whoever it is: the result does not depend on the order of arrival.
//
// The pieces of an item are counted in a 64-bit word (call number << 16 |
// pieces so far) that the merging CTA sets back to zero; a word that holds
// another call's number counts as zero. So the workspace needs no
// initialisation, and a captured graph may be replayed.
#pragma once

#include "paged.cuh"
#include "tma_util.cuh"

namespace qi4 {

constexpr int kBlockKeys = 128;  // keys of a unit

struct PagedArgs {
  const uint16_t* q;
  int64_t q_tok, q_head;  // strides, elements
  uint16_t* out;          // [T, Hq, D] contiguous
  const int32_t* table;
  int64_t table_stride;
  int table_width, pages, page_shift, box_shift;  // box: rows of one copy, min(page_size, kBlockKeys)
  Ragged r;
  int fixed_len;  // >= 0: every sequence has this many keys (lengths is not read)
  int Hkv, G, cap;
  int causal;
  float scale_log2;  // scale * log2(e)
  float* ws;         // pieces: two slots per CTA, each R x D sums then R x (max, sum)
  unsigned long long* counters;  // one per CTA
  unsigned long long call;       // number of this call, 1 .. 2^48 - 1
  // Keys that every row has seen already (a shared prefix): per row t * Hq + h
  // the D weighted sums, and (max, sum of weights); or null.
  const float* prior_acc;
  const float* prior_ml;
  // Non-null: the rows' state is written here instead of `out`.
  float* state_acc;
  float* state_ml;
};

struct Seq {
  int first, n, len;  // first token row, tokens, keys
  int tiles, blocks;  // row tiles, units of an item
  __device__ __forceinline__ int units(int Hkv) const { return n > 0 ? tiles * Hkv * blocks : 0; }
};

template <int R>
__device__ __forceinline__ Seq seq_info(const PagedArgs& a, int b) {
  const Tokens t = seq_tokens(a.r, b);
  int len = a.fixed_len >= 0 ? a.fixed_len : __ldg(a.r.lengths + b);
  len = min(max(len, 0), a.cap);
  return {t.first, t.count, len, (t.count * a.G + R - 1) / R, max(1, (len + kBlockKeys - 1) / kBlockKeys)};
}

// Keys that row `row` of the sequence sees.
__device__ __forceinline__ int visible(const PagedArgs& a, const Seq& s, int row) {
  return a.causal ? max(0, min(s.len, s.len - s.n + row / a.G + 1)) : s.len;
}

// The units of all sequences: their number, and the sequence that holds unit
// `u` with the units before it. Every lane of the warp takes part and gets
// the same result; 128 sequences at a time, their loads independent.
template <int R>
__device__ __forceinline__ long long total_units(const PagedArgs& a, int lane) {
  long long sum = 0;
  for (int b0 = 0; b0 < a.r.B; b0 += 128) {
    int w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = b0 + 4 * lane + i;
      w[i] = b < a.r.B ? seq_info<R>(a, b).units(a.Hkv) : 0;
    }
    long long mine = (long long)w[0] + w[1] + w[2] + w[3];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    sum += mine;
  }
  return sum;
}

template <int R>
__device__ __forceinline__ void find_unit(const PagedArgs& a, long long u, int lane, int& seq, long long& before) {
  long long base = 0;
  for (int b0 = 0; b0 < a.r.B; b0 += 128) {
    int w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = b0 + 4 * lane + i;
      w[i] = b < a.r.B ? seq_info<R>(a, b).units(a.Hkv) : 0;
    }
    const long long mine = (long long)w[0] + w[1] + w[2] + w[3];
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const long long all = __shfl_sync(0xffffffffu, incl, 31);
    if (u < base + all) {
      const unsigned hit = __ballot_sync(0xffffffffu, base + incl > u);
      const int src = __ffs(hit) - 1;
      long long at = base + incl - mine;
      int s = 0;
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (s == i && at + w[i] <= u) {
          at += w[i];
          ++s;
        }
      seq = __shfl_sync(0xffffffffu, b0 + 4 * lane + s, src);
      before = __shfl_sync(0xffffffffu, at, src);
      return;
    }
    base += all;
  }
  seq = a.r.B;
  before = base;
}

// CTA c of C owns units [run_start(c), run_start(c + 1)); run_of inverts it.
__device__ __forceinline__ long long run_start(int c, long long U, int C) { return (long long)c * U / C; }
__device__ __forceinline__ int run_of(long long u, long long U, int C) { return (int)(((u + 1) * C + U - 1) / U) - 1; }

// One CTA's walk over its units, item by item; every warp keeps its own copy.
template <int R>
struct Walk {
  long long U, u, end, item0;  // item0: first unit of the current item
  int C, c, b, rem;            // rem: units of sequence b before u
  Seq s;
  int kvh, tile, blk, nblk;    // this piece: units [blk, blk + nblk) of the item

  __device__ __forceinline__ bool begin(const PagedArgs& a, int lane) {
    U = total_units<R>(a, lane);
    C = (int)min((long long)gridDim.x, U);
    c = blockIdx.x;
    if (c >= C) return false;
    u = run_start(c, U, C);
    end = run_start(c + 1, U, C);
    long long before;
    find_unit<R>(a, u, lane, b, before);
    rem = (int)(u - before);
    s = seq_info<R>(a, min(b, a.r.B - 1));
    return true;
  }
  __device__ __forceinline__ bool next(const PagedArgs& a) {
    if (u >= end) return false;
    while (rem >= s.units(a.Hkv)) {
      rem -= s.units(a.Hkv);
      if (++b >= a.r.B) return false;
      s = seq_info<R>(a, b);
    }
    const int item = rem / s.blocks;
    blk = rem - item * s.blocks;
    tile = item / a.Hkv;
    kvh = item - tile * a.Hkv;
    nblk = (int)min((long long)(s.blocks - blk), end - u);
    item0 = u - blk;
    u += nblk;
    rem += nblk;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return blk == 0 && nblk == s.blocks; }
  __device__ __forceinline__ int rows(const PagedArgs& a) const { return min(R, s.n * a.G - tile * R); }
  __device__ __forceinline__ int64_t token(const PagedArgs& a, int r) const { return s.first + (tile * R + r) / a.G; }
  __device__ __forceinline__ int head(const PagedArgs& a, int r) const { return kvh * a.G + (tile * R + r) % a.G; }
  // Keys the tile's last row sees: none beyond is loaded.
  __device__ __forceinline__ int tile_visible(const PagedArgs& a) const {
    return visible(a, s, tile * R + rows(a) - 1);
  }
  // Blocks of this piece that hold visible keys.
  __device__ __forceinline__ int loaded(int vis) const {
    return max(0, min(nblk, (vis + kBlockKeys - 1) / kBlockKeys - blk));
  }
  __device__ __forceinline__ int first_cta() const { return run_of(item0, U, C); }
  __device__ __forceinline__ int pieces() const { return run_of(item0 + s.blocks - 1, U, C) - first_cta() + 1; }
  // Where CTA p's piece of the current item lies: its first or its second slot.
  __device__ __forceinline__ int slot(int p) const { return 2 * p + (run_start(p, U, C) >= item0 ? 0 : 1); }
};

// Counts one piece of `n`; true for the piece that completes the item.
__device__ __forceinline__ bool arrive_last(unsigned long long* word, unsigned long long call, int n) {
  unsigned long long old = *reinterpret_cast<volatile unsigned long long*>(word);
  for (;;) {
    const int seen = (old >> 16) == call ? (int)(old & 0xFFFF) : 0;
    const unsigned long long now = seen + 1 == n ? 0ull : (call << 16 | (unsigned)(seen + 1));
    const unsigned long long got = atomicCAS(word, old, now);
    if (got == old) return seen + 1 == n;
    old = got;
  }
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats rounded to the packed 16-bit type (lo in the low half).
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t d;
  if constexpr (F16)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// N dims (at d) of a finished row: weighted sums, max and sum of weights over
// its own keys. Joins the prior state, and writes the output or the state. A
// row that saw no key is zero.
template <int D, bool F16, int N>
__device__ __forceinline__ void finish_row(const PagedArgs& a, int64_t token, int head, int d, float (&acc)[N], float m,
                                           float l) {
  const int64_t row = token * (a.Hkv * a.G) + head;
  if (a.state_acc) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(a.state_acc + row * D + d + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
    if (d == 0) *reinterpret_cast<float2*>(a.state_ml + 2 * row) = make_float2(m, l);
    return;
  }
  if (a.prior_acc) {
    const float2 pm = *reinterpret_cast<const float2*>(a.prior_ml + 2 * row);
    const float top = fmaxf(m, pm.x);
    const float f = m == -INFINITY ? 0.f : exp2_approx(m - top), g = pm.x == -INFINITY ? 0.f : exp2_approx(pm.x - top);
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 p = *reinterpret_cast<const float4*>(a.prior_acc + row * D + d + i);
      acc[i] = acc[i] * f + p.x * g;
      acc[i + 1] = acc[i + 1] * f + p.y * g;
      acc[i + 2] = acc[i + 2] * f + p.z * g;
      acc[i + 3] = acc[i + 3] * f + p.w * g;
    }
    l = l * f + pm.y * g;
  }
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) w[i] = pack2<F16>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  if constexpr (N == 8)
    *reinterpret_cast<uint4*>(a.out + row * D + d) = make_uint4(w[0], w[1], w[2], w[3]);
  else
    *reinterpret_cast<uint2*>(a.out + row * D + d) = make_uint2(w[0], w[1]);
}

// Merges the pieces of the walk's current item and finishes its rows: a group
// of D / 4 lanes per row, warp `warp` of `nwarps`. Pieces in the order of
// their CTAs: the first CTA's, then the first slot of each later one.
template <int D, int R, bool F16, class W>
__device__ __forceinline__ void merge_pieces(const PagedArgs& a, const W& w, int warp, int nwarps, int lane) {
  constexpr int kLanes = D / 4, kPerWarp = 32 / kLanes;
  constexpr int64_t kSlot = (int64_t)R * (D + 2);
  const int np = w.pieces(), p0 = w.first_cta(), rows = w.rows(a);
  const float* first = a.ws + w.slot(p0) * kSlot;
  const float* later = a.ws + 2 * (int64_t)p0 * kSlot;  // piece p > 0 at later + 2 p kSlot
  const int d = (lane % kLanes) * 4;
  for (int r0 = warp * kPerWarp; r0 < rows; r0 += nwarps * kPerWarp) {
    const int r = min(r0 + lane / kLanes, rows - 1);
    const int64_t at_ml = (int64_t)R * D + 2 * r, at_acc = (int64_t)r * D + d;
    float top = -INFINITY;
    for (int p = lane % kLanes; p < np; p += kLanes) top = fmaxf(top, __ldcg((p ? later + 2 * p * kSlot : first) + at_ml));
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int q0 = 0; q0 < np; q0 += kLanes) {
      const int p = q0 + lane % kLanes;
      float2 ml = make_float2(-INFINITY, 0.f);
      if (p < np) ml = __ldcg(reinterpret_cast<const float2*>((p ? later + 2 * p * kSlot : first) + at_ml));
      const float fp = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - top);
      const float lp = ml.y * fp;
      const int cnt = min(kLanes, np - q0);
      const float* src = later + 2 * q0 * kSlot + at_acc;
#pragma unroll 16
      for (int j = 0; j < cnt; ++j) {
        const float f = __shfl_sync(0xffffffffu, fp, j, kLanes);
        l += __shfl_sync(0xffffffffu, lp, j, kLanes);
        const float4 v = __ldcg(reinterpret_cast<const float4*>(q0 + j ? src + 2 * j * kSlot : first + at_acc));
        acc[0] += v.x * f;
        acc[1] += v.y * f;
        acc[2] += v.z * f;
        acc[3] += v.w * f;
      }
    }
    if (r0 + lane / kLanes < rows) finish_row<D, F16, 4>(a, w.token(a, r), w.head(a, r), d, acc, top, l);
  }
}

// Launch of the tcgen05 kernel (paged_prefill.cu): tiles of kTcRows rows.
constexpr int kTcRows = 256;
cudaError_t launch_paged_tc(int D, bool f16, const CUtensorMap& k, const CUtensorMap& v, const PagedArgs& a, int ctas,
                            cudaStream_t s);

// One box {64 dims, rows, one head, one page} of the pool into shared memory.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int page,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(smem_addr(bar))
      : "memory");
}

}  // namespace qi4
