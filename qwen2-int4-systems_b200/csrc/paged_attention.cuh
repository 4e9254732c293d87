// Work split and partial-result merging of the paged attention kernels.
//
// A batch is cut into items - one row tile (up to R consecutive rows of one
// sequence's tokens x the G query heads of one KV head, row = token * G + head)
// of one KV head - and every item into units of kBlockKeys keys that its rows
// see. The units of all items, in one line, are dealt to the CTAs in equal
// runs, so sequences of any mixture of lengths keep all SMs equally busy; a
// CTA's run may end inside an item. An item wholly inside one run is finished there; the pieces of
// another go to a workspace as (weighted sums, max, sum of weights), and a
// second, small launch joins them in the order of the runs, so no result
// depends on timing. (It is resident before the first launch ends, by
// programmatic dependent launch. Counting the pieces in the kernel instead,
// the last CTA of an item joining them, cost 25 us where 74 CTAs met at one
// counter and one of them read all their pieces: 65 us for one sequence of
// 131,002 keys against 32 with the second launch.)
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
  struct SplitItem* splits;  // one per CTA: the item that begins in its run and ends beyond it
  // Keys that every row has seen already (a shared prefix): per row t * Hq + h
  // the D weighted sums, and (max, sum of weights); or null.
  const float* prior_acc;
  const float* prior_ml;
  // Non-null: the rows' state is written here instead of `out`.
  float* state_acc;
  float* state_ml;
};

// An item whose pieces are joined: `pieces` of them (0: none), the first in
// slot `slot`, piece p > 0 in slot 2 (cta + p). Row r of its tile is query row
// row0 + r of the sequence whose first token is `first`.
struct SplitItem {
  int pieces, slot, rows, first, row0, kvh;
};

// CTA c of C owns units [run_start(c), run_start(c + 1)); run_of inverts it.
__device__ __forceinline__ long long run_start(int c, long long U, int C) { return (long long)c * U / C; }
__device__ __forceinline__ int run_of(long long u, long long U, int C) { return (int)(((u + 1) * C + U - 1) / U) - 1; }

// One CTA's walk over its units, item by item; every warp keeps its own copy
// (all lanes alike). A tile has R rows, or the most whole tokens that R rows
// hold; an item has one unit per kBlockKeys keys that its last row sees, and
// one more in front that stands for its fixed cost (queries, sums, output) in
// the dealing and is no work: where a run ends behind it, the item begins
// with the next CTA.
template <int R>
struct Walk {
  long long U, u, end, item0;  // u: next unit; item0: the current item's first (fixed-cost) unit
  int C, tile_rows;
  int b, first, n, len, tiles;       // sequence b: first token, tokens, keys, row tiles
  int tile, kvh, blocks, at;         // item; at: next of its 1 + blocks units
  int blk, nblk;                     // this piece: blocks [blk, blk + nblk) of the item

  __device__ __forceinline__ void load(const PagedArgs& a, int seq) {
    b = seq;
    const Tokens t = seq_tokens(a.r, seq);
    first = t.first;
    n = t.count;
    len = a.fixed_len >= 0 ? a.fixed_len : __ldg(a.r.lengths + seq);
    len = min(max(len, 0), a.cap);
    tiles = (n * a.G + tile_rows - 1) / tile_rows;
  }
  // Keys that a row of the sequence sees.
  __device__ __forceinline__ int visible(const PagedArgs& a, int seq_row) const {
    return a.causal ? max(0, min(len, len - n + seq_row / a.G + 1)) : len;
  }
  __device__ __forceinline__ int blocks_of(const PagedArgs& a, int t) const {
    return max(1, (visible(a, min(n * a.G, (t + 1) * tile_rows) - 1) + kBlockKeys - 1) / kBlockKeys);
  }
  // Units of sequences b0 .. b0 + per - 1, one per group of 32 / per lanes (per
  // a power of two), each lane summing every (32 / per)-th tile; the sum of a
  // sequence ends up in the first lane of its group, 0 in the others.
  __device__ __forceinline__ long long group_units(const PagedArgs& a, int b0, int per, int lane) {
    const int lanes = 32 / per, seq = b0 + lane / lanes, sub = lane % lanes;
    long long sum = 0;
    if (seq < a.r.B) {
      load(a, seq);
      if (!a.causal) {
        if (sub == 0) sum = (long long)tiles * (1 + blocks_of(a, 0));
      } else {
        for (int t = sub; t < tiles; t += lanes) sum += 1 + blocks_of(a, t);
      }
    }
    for (int o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sub == 0 ? sum * a.Hkv : 0;
  }
  static __device__ __forceinline__ long long scan(long long x, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += v;
    }
    return x;
  }
  // False if the CTA has no units.
  __device__ __forceinline__ bool begin(const PagedArgs& a, int lane) {
    tile_rows = a.G <= R ? R / a.G * a.G : R;
    int per = 32;
    while (per > 1 && per / 2 >= a.r.B) per >>= 1;
    U = 0;
    long long mine = 0;
    for (int b0 = 0; b0 < a.r.B; b0 += per) {
      long long x = mine = group_units(a, b0, per, lane);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      U += x;
    }
    C = (int)min((long long)gridDim.x, U);
    if ((int)blockIdx.x >= C) return false;
    u = run_start(blockIdx.x, U, C);
    end = run_start(blockIdx.x + 1, U, C);
    // The sequence that holds unit u, then the tile.
    long long before = 0;
    int seq = 0;
    for (int b0 = 0; b0 < a.r.B; b0 += per) {
      if (a.r.B > per) mine = group_units(a, b0, per, lane);
      const long long incl = scan(mine, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, before + incl > u);
      if (hit) {
        const int src = __ffs(hit) - 1;
        seq = b0 + src / (32 / per);
        before += __shfl_sync(0xffffffffu, incl - mine, src);
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    load(a, seq);
    for (tile = 0; tile + 1 < tiles; tile += 32) {
      const long long units = tile + lane < tiles ? (long long)(1 + blocks_of(a, tile + lane)) * a.Hkv : 0;
      const long long incl = scan(units, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, before + incl > u);
      if (hit) {
        const int src = __ffs(hit) - 1;
        tile += src;
        before += __shfl_sync(0xffffffffu, incl - units, src);
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    blocks = blocks_of(a, tile);
    at = (int)(u - before);
    kvh = at / (1 + blocks);
    at -= kvh * (1 + blocks);
    return true;
  }
  // The next piece; false behind the last.
  __device__ __forceinline__ bool next(const PagedArgs& a) {
    for (;;) {
      if (u >= end) return false;
      if (at > blocks) {  // the next KV head, tile or sequence with tokens
        at = 0;
        if (++kvh == a.Hkv) {
          kvh = 0;
          if (++tile == tiles) {
            tile = 0;
            do {
              if (b + 1 >= a.r.B) return false;
              load(a, b + 1);
            } while (tiles == 0);
          }
          blocks = blocks_of(a, tile);
        }
      }
      const int take = (int)min((long long)(1 + blocks - at), end - u);
      item0 = u - at;
      blk = max(at - 1, 0);
      nblk = at + take - 1 - blk;
      u += take;
      at += take;
      if (nblk > 0) return true;
    }
  }
  __device__ __forceinline__ bool whole() const { return nblk == blocks; }
  __device__ __forceinline__ int rows(const PagedArgs& a) const { return min(tile_rows, n * a.G - tile * tile_rows); }
  __device__ __forceinline__ int row0() const { return tile * tile_rows; }
  __device__ __forceinline__ int64_t token(const PagedArgs& a, int r) const { return first + (row0() + r) / a.G; }
  __device__ __forceinline__ int head(const PagedArgs& a, int r) const { return kvh * a.G + (row0() + r) % a.G; }
  __device__ __forceinline__ int row_visible(const PagedArgs& a, int r) const { return visible(a, row0() + r); }
  // Keys the tile's last row sees: none beyond is loaded.
  __device__ __forceinline__ int tile_visible(const PagedArgs& a) const { return row_visible(a, rows(a) - 1); }
  // Blocks of this piece that hold visible keys: all, but for an item of one empty block.
  __device__ __forceinline__ int loaded(int vis) const { return vis > 0 ? nblk : 0; }
  // The CTAs that hold the item's blocks, and where CTA p's piece lies: its first or its second slot.
  __device__ __forceinline__ int first_cta() const { return run_of(item0 + 1, U, C); }
  __device__ __forceinline__ int pieces() const { return run_of(item0 + blocks, U, C) - first_cta() + 1; }
  __device__ __forceinline__ int slot(int p) const { return 2 * p + (run_start(p, U, C) >= item0 ? 0 : 1); }
};

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
  uint16_t* out = a.out + row * D + d;
  if constexpr (N == 16)  // one whole sector of 32 bytes
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  else
    *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
}

// What a CTA leaves for the joining launch, from its last piece (one thread).
template <int R>
__device__ __forceinline__ void note_split(const PagedArgs& a, const Walk<R>& w, bool any) {
  SplitItem it = {0, 0, 0, 0, 0, 0};
  if (any && w.blk == 0 && w.nblk > 0 && !w.whole())
    it = {w.pieces(), w.slot(blockIdx.x), w.rows(a), w.first, w.row0(), w.kvh};
  a.splits[blockIdx.x] = it;
}

// Joins the pieces of the item that begins in CTA blockIdx.x's run and ends
// beyond it, if there is one: a group of D / 4 lanes per row, the rows spread
// over the warps of the blocks (blockIdx.x, 0 ..).
constexpr int kJoinThreads = 256;
template <int D, int R, bool F16>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const SplitItem it = a.splits[blockIdx.x];
  constexpr int kLanes = D / 4, kPerWarp = 32 / kLanes;
  constexpr int64_t kSlot = (int64_t)R * (D + 2);
  const int lane = threadIdx.x & 31, d = (lane % kLanes) * 4, np = it.pieces;
  const float* first = a.ws + it.slot * kSlot;
  const float* later = a.ws + 2 * (int64_t)blockIdx.x * kSlot;
  for (int r0 = (blockIdx.y * (kJoinThreads / 32) + threadIdx.x / 32) * kPerWarp; r0 < it.rows;
       r0 += gridDim.y * (kJoinThreads / 32) * kPerWarp) {
    const int r = min(r0 + lane / kLanes, it.rows - 1);
    const int64_t at_ml = (int64_t)R * D + 2 * r, at_acc = (int64_t)r * D + d;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, l = 0.f;
    // 32 (16) pieces at a time, one lane each for their maxima and sums; the
    // running maximum is moved once per round.
    for (int q0 = 0; q0 < np; q0 += kLanes) {
      const int p = q0 + lane % kLanes;
      float2 ml = make_float2(-INFINITY, 0.f);
      if (p < np) ml = *reinterpret_cast<const float2*>((p ? later + 2 * p * kSlot : first) + at_ml);
      float m = fmaxf(top, ml.x);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float back = top == -INFINITY ? 0.f : exp2_approx(top - m);
      top = m;
      l *= back;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] *= back;
      const float fp = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - m);
      const float lp = ml.y * fp;
      const int cnt = min(kLanes, np - q0);
      const float* src = later + 2 * q0 * kSlot + at_acc;
#pragma unroll 16
      for (int j = 0; j < cnt; ++j) {
        const float f = __shfl_sync(0xffffffffu, fp, j, kLanes);
        l += __shfl_sync(0xffffffffu, lp, j, kLanes);
        const float4 v = *reinterpret_cast<const float4*>(q0 + j ? src + 2 * j * kSlot : first + at_acc);
        acc[0] += v.x * f;
        acc[1] += v.y * f;
        acc[2] += v.z * f;
        acc[3] += v.w * f;
      }
    }
    if (r0 + lane / kLanes < it.rows)
      finish_row<D, F16, 4>(a, it.first + (it.row0 + r) / a.G, it.kvh * a.G + (it.row0 + r) % a.G, d, acc, top, l);
  }
}

// Launches the joining of `ctas` runs, behind the kernel that wrote their pieces.
template <int D, int R, bool F16>
cudaError_t launch_join(const PagedArgs& a, int ctas, cudaStream_t s) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  constexpr int kRowsAtOnce = kJoinThreads / 32 * (128 / D);
  cfg.gridDim = dim3((unsigned)ctas, (unsigned)((R + 2 * kRowsAtOnce - 1) / (2 * kRowsAtOnce)), 1);
  cfg.blockDim = dim3(kJoinThreads, 1, 1);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<D, R, F16>, a);
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
