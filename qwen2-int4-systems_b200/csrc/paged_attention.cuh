// Work split and partial-result merging of the paged attention kernels.
//
// A batch is cut into items - one row tile (up to R consecutive rows of one
// sequence's tokens x the G query heads of one KV head, row = token * G + head)
// of one KV head - and every item into units of kBlockKeys keys that its rows
// see. The units of all items, in one line, are dealt to the CTAs in equal
// runs, so sequences of any mixture of lengths keep all SMs equally busy; a
// CTA's run may end inside an item. An item wholly inside one run is finished
// there; the pieces of another go to a workspace as (weighted sums, max, sum of
// weights), and a second, small launch joins them in the order of the runs, so
// no result depends on timing. (Counting the pieces in the kernel instead, the
// last CTA of an item joining them, cost 25 us where 74 CTAs met at one counter
// and one of them read all their pieces: 65 us for one sequence of 131,002 keys
// against 32 then with the second launch.) The second launch is 3 us of a small
// call, so where tables are short no item is split (`unsplit`), and few items of
// the mma.sync kernel are shared out within clusters (`share`) if their tables
// are not long.
#pragma once

#include "paged.cuh"
#include "tma_util.cuh"

namespace qi4 {

constexpr int kBlockKeys = 128;  // keys of a unit
constexpr int kMaxCtas = 256;    // CTAs of a launch at most

struct PagedArgs {
  const uint16_t* q;
  int64_t q_tok, q_head;  // strides, elements
  uint16_t* out;          // [T, Hq, D] contiguous
  const int32_t* table;
  int64_t table_stride;
  int table_width, pages, page_shift, box_shift;  // box: rows of one copy, min(page_size, kBlockKeys)
  const uint16_t* v;  // the values' pool, for add_odd
  int64_t v_page, v_head, v_slot;
  Ragged r;
  int fixed_len;  // >= 0: every sequence has this many keys (lengths is not read)
  int Hkv, G, cap;
  int causal;
  int unsplit;                 // an item is all done by the CTA that owns its first unit: nothing is joined
  int one_tile;                // no sequence has more rows than a tile (decode steps, drafts): the split is shorter
  int tile_rows, tile_tokens;  // R rows, or the most whole tokens that R rows hold (0 tokens: a token has more rows)
  FastDiv by_tile_rows, by_G, by_ctas;  // by_ctas: the launch's CTAs
  float scale_log2;  // scale * log2(e)
  float* ws;         // pieces: two slots per CTA, each R x D sums then R x (max, sum)
  struct SplitItem* splits;  // one per CTA: the item that begins in its run and ends beyond it
  // What another launch found for every row: per row t * Hq + h the D weighted
  // sums, and (max, sum of weights); or null. `late`: that launch is the one
  // before this, which waits for it only before it reads the state (all else it
  // reads is older than the launch before that one).
  const float* prior_acc;
  const float* prior_ml;
  int late;
  // Non-null: the rows' state is written here instead of `out`.
  float* state_acc;
  float* state_ml;
};

// An item whose pieces are joined: `pieces` of them (0: none), the first in
// slot `slot`, piece p > 0 in slot 2 (cta + p). Row r of its tile is query row
// row0 + r of the sequence whose first token is `first`.
struct alignas(8) SplitItem {
  int pieces, rows, slot, first, row0, kvh;
};

// The dealing of U units to C CTAs: CTA c owns [start(c), start(c + 1)),
// start(c) = floor(c U / C). U below 2^31 (checked on the host), so that
// nothing needs a 64-bit division.
struct Runs {
  int U, C, quot, rest;
  FastDiv by_C;
  __device__ __forceinline__ Runs() {}
  __device__ __forceinline__ Runs(const PagedArgs& a, int units, int ctas) : U(units), C(min(ctas, units)) {
    if (units < ctas) {
      quot = 1, rest = 0;  // one unit each
      by_C = {0u, 0u};
    } else {
      by_C = a.by_ctas;
      quot = by_C(units);
      rest = units - quot * ctas;
    }
  }
  __device__ __forceinline__ int start(int c) const { return c * quot + by_C(c * rest); }
  __device__ __forceinline__ int holder(int u) const {  // the CTA that owns unit u
    int c = min(C - 1, (int)(__fdividef((float)u, (float)U) * (float)C));
    while (start(c) > u) --c;
    while (c + 1 < C && start(c + 1) <= u) ++c;
    return c;
  }
};

// One CTA's walk over its units, item by item; every warp keeps its own copy
// (all lanes alike). A tile has R rows, or the most whole tokens that R rows
// hold; an item has one unit per kBlockKeys keys that its last row sees, and
// one more in front that stands for its fixed cost (queries, sums, output) in
// the dealing and is no work: where a run ends behind it, the item begins
// with the next CTA.
template <int R>
struct Walk {
  Runs runs;
  int u, end, item0;  // u: next unit; item0: the current item's first (fixed-cost) unit
  int b, first, n, len, tiles;       // sequence b: first token, tokens, keys, row tiles
  int tile, kvh, blocks, at;         // item; at: next of its 1 + blocks units
  int blk, nblk;                     // this piece: blocks [blk, blk + nblk) of the item

  __device__ __forceinline__ void load(const PagedArgs& a, int seq) {
    set(a, seq, seq_tokens(a.r, seq), a.fixed_len >= 0 ? a.fixed_len : __ldg(a.r.lengths + seq));
  }
  __device__ __forceinline__ void set(const PagedArgs& a, int seq, Tokens t, int length) {
    b = seq;
    first = t.first;
    n = t.count;
    len = min(max(length, 0), a.cap);
    tiles = a.one_tile ? n > 0 : a.by_tile_rows(n * a.G + a.tile_rows - 1);
  }
  // Keys that tile t's last row sees: none beyond is loaded.
  __device__ __forceinline__ int tile_visible(const PagedArgs& a, int t) const {
    if (!a.causal || a.one_tile) return len;
    const int last = a.G <= R ? min(n, (t + 1) * a.tile_tokens) - 1 : a.by_G(min(n * a.G, (t + 1) * a.tile_rows) - 1);
    return max(0, min(len, len - n + last + 1));
  }
  __device__ __forceinline__ int tile_visible(const PagedArgs& a) const { return tile_visible(a, tile); }
  __device__ __forceinline__ int blocks_of(const PagedArgs& a, int t) const {
    return max(1, (tile_visible(a, t) + kBlockKeys - 1) / kBlockKeys);
  }
  // Units of the loaded sequence, the tiles from `sub` on in steps of `step`.
  __device__ __forceinline__ int seq_units(const PagedArgs& a, int sub, int step) const {
    if (!a.causal || a.one_tile) return sub == 0 ? a.Hkv * tiles * (1 + blocks_of(a, 0)) : 0;
    int sum = 0;
    for (int t = sub; t < tiles; t += step) sum += 1 + blocks_of(a, t);
    return a.Hkv * sum;
  }
  // Units of sequences b0 .. b0 + 3, all their loads before the first use.
  __device__ __forceinline__ void quad_units(const PagedArgs& a, int b0, int (&w)[4]) {
    Tokens t[4];
    int l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int seq = min(b0 + i, a.r.B - 1);
      t[i] = seq_tokens(a.r, seq);
      l[i] = a.fixed_len >= 0 ? a.fixed_len : __ldg(a.r.lengths + seq);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      set(a, b0 + i, t[i], l[i]);
      w[i] = b0 + i < a.r.B ? seq_units(a, 0, 1) : 0;
    }
  }
  static __device__ __forceinline__ int scan(int x, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += v;
    }
    return x;
  }
  // False if the CTA has no units.
  __device__ __forceinline__ bool begin(const PagedArgs& a, int lane) {
    int U = 0, before = 0, seq = 0;
    if (a.r.B <= 32) {
      // A sequence for each group of lanes, which share its tiles.
      int lanes = 32;
      while (lanes > 1 && 32 / lanes < a.r.B) lanes >>= 1;
      int mine = 0;
      if (lane / lanes < a.r.B) {
        load(a, lane / lanes);
        mine = seq_units(a, lane & (lanes - 1), lanes);
      }
      for (int o = lanes / 2; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
      if (lane & (lanes - 1)) mine = 0;
      const int incl = scan(mine, lane);
      U = __shfl_sync(0xffffffffu, incl, 31);
      if (!deal(a, U)) return false;
      const unsigned hit = __ballot_sync(0xffffffffu, incl > u);
      const int src = __ffs(hit) - 1;
      seq = src / lanes;
      before = __shfl_sync(0xffffffffu, incl - mine, src);
    } else {
      // 128 at a time, four in a row for each lane; the first 128 stay at hand for the second pass.
      int kept[4];
      quad_units(a, 4 * lane, kept);
      U = __reduce_add_sync(0xffffffffu, kept[0] + kept[1] + kept[2] + kept[3]);
      for (int b0 = 128; b0 < a.r.B; b0 += 128) {
        int more[4];
        quad_units(a, b0 + 4 * lane, more);
        U += __reduce_add_sync(0xffffffffu, more[0] + more[1] + more[2] + more[3]);
      }
      if (!deal(a, U)) return false;
      for (int b0 = 0; b0 < a.r.B; b0 += 128) {
        if (b0) quad_units(a, b0 + 4 * lane, kept);
        const int mine = kept[0] + kept[1] + kept[2] + kept[3], incl = scan(mine, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, before + incl > u);
        if (hit) {
          int at0 = before + incl - mine, i = 0;
#pragma unroll
          for (int k = 0; k < 3; ++k)
            if (i == k && at0 + kept[k] <= u) {
              at0 += kept[k];
              ++i;
            }
          const int src = __ffs(hit) - 1;
          seq = __shfl_sync(0xffffffffu, b0 + 4 * lane + i, src);
          before = __shfl_sync(0xffffffffu, at0, src);
          break;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
    load(a, seq);
    for (tile = 0; tile + 1 < tiles; tile += 32) {
      const int units = tile + lane < tiles ? (1 + blocks_of(a, tile + lane)) * a.Hkv : 0;
      const int incl = scan(units, lane);
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
    at = u - before;
    kvh = min(a.Hkv - 1, (int)__fdividef((float)at, (float)(1 + blocks)));
    while (kvh * (1 + blocks) > at) --kvh;
    while ((kvh + 1) * (1 + blocks) <= at) ++kvh;
    at -= kvh * (1 + blocks);
    return true;
  }
  // Instead of a run: part `rank` of `parts` of item `item`, which is a sequence and KV head (one_tile). False if the
  // sequence has no tokens.
  __device__ __forceinline__ bool share(const PagedArgs& a, int item, int rank, int parts) {
    const int seq = item / a.Hkv;
    load(a, seq);
    kvh = item - seq * a.Hkv;
    tile = 0;
    blocks = blocks_of(a, 0);
    blk = blocks * rank / parts;
    nblk = blocks * (rank + 1) / parts - blk;
    return tiles > 0;
  }
  // This CTA's run of U units.
  __device__ __forceinline__ bool deal(const PagedArgs& a, int U) {
    if ((int)blockIdx.x >= min((int)gridDim.x, U)) return false;
    runs = Runs(a, U, gridDim.x);
    u = runs.start(blockIdx.x);
    end = runs.start(blockIdx.x + 1);
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
      int take = 1 + blocks - at;
      if (!a.unsplit) {
        take = min(take, end - u);
      } else if (at > 0) {  // the item belongs to an earlier CTA
        u += take;
        at += take;
        continue;
      }
      item0 = u - at;
      blk = max(at - 1, 0);
      nblk = at + take - 1 - blk;
      u += take;
      at += take;
      if (nblk > 0) return true;
    }
  }
  __device__ __forceinline__ bool whole() const { return nblk == blocks; }
  __device__ __forceinline__ int rows(const PagedArgs& a) const { return min(a.tile_rows, n * a.G - tile * a.tile_rows); }
  __device__ __forceinline__ int row0(const PagedArgs& a) const { return tile * a.tile_rows; }
  // Token and query head of row r of the tile.
  __device__ __forceinline__ void place(const PagedArgs& a, int r, int& token, int& head) const {
    const int row = row0(a) + r, t = a.by_G(row);
    token = first + t;
    head = kvh * a.G + row - t * a.G;
  }
  __device__ __forceinline__ int row_visible(const PagedArgs& a, int r) const {
    return a.causal ? max(0, min(len, len - n + a.by_G(row0(a) + r) + 1)) : len;
  }
  // Blocks of this piece that hold visible keys: all, but for an item of one empty block.
  __device__ __forceinline__ int loaded(int vis) const { return vis > 0 ? nblk : 0; }
  // The CTAs that hold the item's blocks, and where CTA p's piece lies: its first or its second slot.
  __device__ __forceinline__ int pieces() const { return runs.holder(item0 + blocks) - runs.holder(item0 + 1) + 1; }
  __device__ __forceinline__ int slot(int p) const { return 2 * p + (runs.start(p) >= item0 ? 0 : 1); }
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool F16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// Weights are taken relative to 2^(max - kLift), sums of weights and of values alike. Against a row's maximum that lags
// by up to 2^8 they reach 2^15 in FP16, which goes to 2^16, and not 2^8: FP16's steps end at 2^-24, so that a weight is
// off by up to 2^-25 however small it is, 2^-32 of the largest one at least (it would be 2^-25 without the lift).
// BF16 has FP32's exponents and needs none.
template <bool F16>
constexpr float kLift = F16 ? 7.f : 0.f;

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

// Values that are not finite (odd ones) at keys that only some rows of a tile
// see: the product would make 0 x inf = NaN of them in the rows that do not. The
// units that hold such keys (the last ones of a causal tile with several tokens)
// have their odd values cleared before the product, and at the item's end the
// rows that see them take them up from the pool: a positive weight times an
// infinity or NaN is it, whatever the weight. Looking costs what these units'
// batches take longer by: drafts (24 sequences, 20 rows each) 36.4 -> 38.1 us,
// ragged chunks 112 -> 116, a prompt of 8192 tokens 249 -> 251.

// Bits 15 and 31: that half of w is infinite or NaN.
template <bool F16>
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
  return ((w & (F16 ? 0x7C007C00u : 0x7F807F80u)) + (F16 ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}
// Clears the odd ones of eight values in shared memory; whether there were any.
template <bool F16>
__device__ __forceinline__ bool clear_odd(uint32_t saddr) {
  uint4 v = lds128(saddr);
  const uint32_t x = odd_halves<F16>(v.x), y = odd_halves<F16>(v.y), z = odd_halves<F16>(v.z), w = odd_halves<F16>(v.w);
  if (!(x | y | z | w)) return false;
  v.x &= ~((x >> 15) * 0xFFFFu);
  v.y &= ~((y >> 15) * 0xFFFFu);
  v.z &= ~((z >> 15) * 0xFFFFu);
  v.w &= ~((w >> 15) * 0xFFFFu);
  sts128(saddr, v);
  return true;
}
// Adds the odd values of keys from .. to - 1 of sequence b to what this thread has written for a row: its dims
// d .. d + n - 1, FP32 at sums[dim * step], or the output where sums is null.
template <bool F16>
__device__ __forceinline__ void add_odd(const PagedArgs& a, int b, int kvh, int from, int to, int d, int n,
                                        uint16_t* out, float* sums, int step) {
#pragma unroll 1
  for (int key = from; key < to; ++key) {
    const int page = __ldg(a.table + b * a.table_stride + (key >> a.page_shift));
    if (page < 0 || page >= a.pages) continue;  // (reads as zeros)
    const uint16_t* v = a.v + page * a.v_page + kvh * a.v_head + (key & ((1 << a.page_shift) - 1)) * a.v_slot;
#pragma unroll 1
    for (int i = d; i < d + n; ++i) {
      const uint32_t w = __ldg(v + i);
      if (!odd_halves<F16>(w)) continue;
      const float x = unpack2<F16>(w).x;
      if (sums)
        sums[i * step] += x;
      else
        out[i] = (uint16_t)pack2<F16>(unpack2<F16>(out[i]).x + x, 0.f);
    }
  }
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
  if (a.unsplit) return;
  SplitItem it = {0, 0, 0, 0, 0, 0};
  if (any && w.blk == 0 && w.nblk > 0 && !w.whole())
    it = {w.pieces(), w.rows(a), w.slot(blockIdx.x), w.first, w.row0(a), w.kvh};
  a.splits[blockIdx.x] = it;
}

// The joining launches: every block learns of all split items (one entry per
// CTA of the launch before) and takes every gridDim.x-th of their shares.
// Blocks that own (CTA, rows) places instead, most of them empty, took two to
// three times as long: thousands of blocks, each a round trip to memory. (Two
// blocks per SM in place of four were slower, eight gained 1 us of 230 at most.)
constexpr int kJoinThreads = 256;
constexpr int kJoinBlocksPerSm = 4;

// ends[c]: shares of the items noted by CTAs 0 .. c; `shares` of an item as given. All threads of the block take part.
template <class Shares>
__device__ __forceinline__ int count_shares(const SplitItem* splits, int ctas, int* ends, const Shares& shares) {
  __shared__ int warp_sum[kJoinThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int before = 0;
  for (int c0 = 0; c0 < ctas; c0 += kJoinThreads) {
    const int c = c0 + threadIdx.x;
    int x = 0;
    if (c < ctas) {
      const int2 head = *reinterpret_cast<const int2*>(&splits[c].pieces);
      x = head.x ? shares(head.x, head.y) : 0;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) {
      if (i == warp) x += before + all;
      all += warp_sum[i];
    }
    if (c < ctas) ends[c] = x;
    before += all;
    __syncthreads();
  }
  return before;
}
// The CTA whose item has share u, and the share's number within the item.
__device__ __forceinline__ int share_owner(const int* ends, int ctas, int u, int& within) {
  int lo = 0, hi = ctas - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] <= u)
      lo = mid + 1;
    else
      hi = mid;
  }
  within = u - (lo ? ends[lo - 1] : 0);
  return lo;
}

// Launch of the tcgen05 kernel (paged_prefill.cu): tiles of kTcRows rows.
constexpr int kTcRows = 256;
// q: the queries as (dims, heads, tokens), box {64, G, kTcRows / G}.
cudaError_t launch_paged_tc(int D, bool f16, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                            const PagedArgs& a, int ctas, cudaStream_t s);

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
