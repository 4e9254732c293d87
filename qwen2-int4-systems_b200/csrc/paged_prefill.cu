// Paged attention for many rows per key (prompts, prompt chunks, the rows of a
// whole batch over a shared prefix) on the 5th-generation tensor cores.
//
// The sums of paged_attention.cu, on tiles of whole tokens: kTcRows / G tokens
// x the G query heads of a KV head, at most 256 rows, as two tensor-memory
// tiles of 128. Bound by the two products (4 D flops per row and key) and by
// the exponentials: a unit of 256 rows x 128 keys takes 2048 cycles of
// tcgen05.mma and 2048 cycles of the SM's 16 exponentials per clock, so the
// two tiles take turns: while one is in its softmax the tensor cores work for
// the other. Units are dealt to the CTAs as in paged_attention.cuh, each item
// with the units its rows can see (causal tiles near the start are short).
//
// Warps of a CTA (one per SM):
//   0-3, 4-7  softmax of tile 0, 1: a thread per row. Scores from tensor memory
//             (tcgen05.ld), the weights back into it over the scores, rounded
//             to the cache's type (the operand type of the second product; the
//             sum of the weights stays FP32 and unrounded). The weights are
//             taken relative to a row maximum that is moved only when a score
//             exceeds it by more than 2^8 (exponents leave room): the sums in
//             tensor memory are then rescaled, rarely. Also the queries (plain
//             loads, swizzled stores) and the epilogue.
//   8         issues the products: S = Q K^T (both operands from shared
//             memory), O += P V (P from tensor memory, V as it lies in the
//             page: key-major, the descriptor's transposed form). Products
//             execute in the order of issue, so "scores of unit i are there"
//             also says that the sums of unit i - 1 are.
//   9         fetches keys and values page by page (TMA, 128-byte swizzle) into
//             a ring of 128-key slots, keys and values by turns.
// Tensor memory: scores 2 x 128 columns, sums 2 x D. All waits are bounded.
#include <algorithm>
#include <atomic>

#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace qi4 {

__device__ int g_paged_tc_error;

namespace {

constexpr int kThreads = 384;
constexpr int kSoftmaxWarps = 8;
constexpr int kMergeRowBlocks = 16;
constexpr int slot_bytes(int D) { return kBlockKeys * D * 2; }
constexpr int ring_slots(int D) { return D == 128 ? 5 : 10; }
constexpr size_t smem_of(int D) {
  return 1024 + (size_t)kTcRows * D * 2 + (size_t)ring_slots(D) * slot_bytes(D) +
         (8 + 2 * ring_slots(D)) * sizeof(uint64_t) + 16;
}

// The walk of paged_attention.cuh over tiles of whole tokens, each item with
// as many units as its last token sees.
struct TileWalk {
  long long U, u, end, item0;
  int C, c, b, tile_tokens;
  int first, n, len, tiles;          // sequence b
  int tile, kvh, blocks, blk, nblk;  // this piece

  __device__ __forceinline__ void load(const PagedArgs& a, int seq) {
    b = seq;
    const Tokens t = seq_tokens(a.r, seq);
    first = t.first;
    n = t.count;
    len = a.fixed_len >= 0 ? a.fixed_len : __ldg(a.r.lengths + seq);
    len = min(max(len, 0), a.cap);
    tiles = (n + tile_tokens - 1) / tile_tokens;
  }
  __device__ __forceinline__ int visible(const PagedArgs& a, int token) const {
    return a.causal ? max(0, min(len, len - n + token + 1)) : len;
  }
  __device__ __forceinline__ int blocks_of(const PagedArgs& a, int t) const {
    return max(1, (visible(a, min(n, (t + 1) * tile_tokens) - 1) + kBlockKeys - 1) / kBlockKeys);
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
        if (sub == 0) sum = (long long)tiles * blocks_of(a, 0);
      } else {
        for (int t = sub; t < tiles; t += lanes) sum += blocks_of(a, t);
      }
    }
    for (int o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sub == 0 ? sum * a.Hkv : 0;
  }
  __device__ __forceinline__ bool begin(const PagedArgs& a, int lane) {
    tile_tokens = kTcRows / a.G;
    int per = 32;
    while (per > 1 && per / 2 >= a.r.B) per >>= 1;
    U = 0;
    for (int b0 = 0; b0 < a.r.B; b0 += per) {
      long long x = group_units(a, b0, per, lane);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      U += x;
    }
    C = (int)min((long long)gridDim.x, U);
    c = blockIdx.x;
    if (c >= C) return false;
    u = run_start(c, U, C);
    end = run_start(c + 1, U, C);
    // The sequence that holds unit u, then the tile.
    long long before = 0;
    int seq = 0;
    for (int b0 = 0; b0 < a.r.B; b0 += per) {
      const long long mine = group_units(a, b0, per, lane);
      long long incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
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
    for (int t0 = 0;; t0 += 32) {
      const long long mine = t0 + lane < tiles ? (long long)blocks_of(a, t0 + lane) * a.Hkv : 0;
      long long incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + incl > u);
      if (hit || t0 + 32 >= tiles) {
        const int src = hit ? __ffs(hit) - 1 : 31;
        tile = t0 + src;
        before += __shfl_sync(0xffffffffu, incl - mine, src);
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    blocks = blocks_of(a, tile);
    const int rem = (int)(u - before);
    kvh = rem / blocks;
    blk = rem - kvh * blocks;
    nblk = 0;
    return true;
  }
  __device__ __forceinline__ bool next(const PagedArgs& a) {
    if (u >= end) return false;
    blk += nblk;
    if (blk >= blocks) {  // the next KV head, tile or sequence with tokens
      blk = 0;
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
    nblk = (int)min((long long)(blocks - blk), end - u);
    item0 = u - blk;
    u += nblk;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return blk == 0 && nblk == blocks; }
  __device__ __forceinline__ int rows(const PagedArgs& a) const {
    return min(tile_tokens, n - tile * tile_tokens) * a.G;
  }
  __device__ __forceinline__ int64_t token(const PagedArgs& a, int r) const {
    return first + tile * tile_tokens + r / a.G;
  }
  __device__ __forceinline__ int head(const PagedArgs& a, int r) const { return kvh * a.G + r % a.G; }
  __device__ __forceinline__ int row_visible(const PagedArgs& a, int r) const {
    return visible(a, tile * tile_tokens + r / a.G);
  }
  __device__ __forceinline__ int tile_visible(const PagedArgs& a) const {
    return visible(a, min(n, (tile + 1) * tile_tokens) - 1);
  }
  __device__ __forceinline__ int first_cta() const { return run_of(item0, U, C); }
  __device__ __forceinline__ int pieces() const { return run_of(item0 + blocks - 1, U, C) - first_cta() + 1; }
  __device__ __forceinline__ int slot(int p) const { return 2 * p + (run_start(p, U, C) >= item0 ? 0 : 1); }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// (x, y) * s - b, and sums of pairs, as packed FP32 operations.
__device__ __forceinline__ void fma_pair(float& x, float& y, float s, float nb) {
  asm("{\n\t.reg .b64 p, m, d;\n\t"
      "mov.b64 p, {%0, %1};\n\t"
      "mov.b64 m, {%2, %2};\n\t"
      "mov.b64 d, {%3, %3};\n\t"
      "fma.rn.f32x2 p, p, m, d;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(s), "f"(nb));
}
__device__ __forceinline__ void add_pair(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 p, q;\n\t"
      "mov.b64 p, {%0, %1};\n\t"
      "mov.b64 q, {%2, %3};\n\t"
      "add.rn.f32x2 p, p, q;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}

// 32 columns of this warp's 32 lanes; the values are there after tmem_ld_wait.
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}
// Waits for the loads, and keeps every use of the N values behind the wait.
template <int N>
__device__ __forceinline__ void tmem_ld_wait(float* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(r[i]));
}
// 16 or 32 columns of 32-bit words.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Descriptor of V as the second product's B operand: rows are keys (the
// contraction), 64 dims (128 bytes, swizzled) each; 8-key groups 1024 bytes
// apart, the next 64 dims one half-slot on.
template <int D>
__device__ __forceinline__ uint64_t v_desc(uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)((kBlockKeys * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// kind::f16 instruction: M = 128, N columns; `v`: B with keys as rows.
__host__ __device__ constexpr uint32_t idesc(bool f16, int N, bool v) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | (v ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const PagedArgs a) {
  constexpr int kSlots = ring_slots(D), kSlotBytes = slot_bytes(D), kHalf = kBlockKeys * 128;
  constexpr int kTileBytes = 128 * D * 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_s = smem;                      // 2 tiles [D / 64][128 rows][128 B]
  uint8_t* ring = smem + 2 * kTileBytes;    // slots [D / 64][128 keys][128 B]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(ring + kSlots * kSlotBytes);  // [2] 4 warps
  uint64_t* s_full = q_full + 2;                                               // [2] commit
  uint64_t* p_full = s_full + 2;                                               // [2] 4 warps
  uint64_t* o_full = p_full + 2;                                               // [2] commit
  uint64_t* kv_full = o_full + 2;                                              // [kSlots] TMA
  uint64_t* kv_empty = kv_full + kSlots;                                       // [kSlots] commit
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kv_empty + kSlots);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    fence_barrier_init();
    prefetch_tensor_map(&kmap);
    prefetch_tensor_map(&vmap);
  }
  if (warp == kSoftmaxWarps) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // S0, S1 at 0, 128; O0, O1 at 256, 256 + D
  pdl_wait();
  pdl_launch_dependents();

  TileWalk w;
  const bool any = w.begin(a, lane);
  if (any && warp == kSoftmaxWarps + 1) {
    // ---- producer ----
    const int box_rows = 1 << a.box_shift;
    int pos = 0;  // ring position
    while (w.next(a)) {
      const int vis = w.tile_visible(a);
      if (lane == 0 && a.fixed_len < 0 && __ldg(a.r.lengths + w.b) > a.cap)
        atomicOr(&g_paged_tc_error, kErrCacheFull);
      int win0 = -1, win = -1;
      for (int i = 0; i < w.nblk; ++i) {
        const int key0 = (w.blk + i) * kBlockKeys;
        if (key0 >= vis) break;
        const int nb = (min(kBlockKeys, vis - key0) + box_rows - 1) >> a.box_shift;
        const int pj = key0 >> a.page_shift, slot = key0 & ((1 << a.page_shift) - 1);
        if ((pj & ~31) != win0) {
          win0 = pj & ~31;
          const int j = win0 + lane;
          win = j < a.table_width ? __ldg(a.table + w.b * a.table_stride + j) : -1;
        }
        const int boxes = (D / 64) * nb;
        const int bx = lane / (D / 64), half = lane % (D / 64);
        const int page = __shfl_sync(0xffffffffu, win, (pj + min(bx, nb - 1)) & 31);
        if (lane < boxes && (page < 0 || page >= a.pages)) atomicOr(&g_paged_tc_error, kErrBadPage);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++pos) {
          const int st = pos % kSlots;
          mbar_wait(&kv_empty[st], ((uint32_t)(pos / kSlots) & 1u) ^ 1u, &g_paged_tc_error);
          if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], (uint32_t)(boxes * box_rows * 128));
          __syncwarp();
          if (lane < boxes)  // at most 2 x 128 / 8 = 32 boxes
            load_box(smem_addr(ring + st * kSlotBytes) + half * kHalf + (bx << a.box_shift) * 128, kv ? &vmap : &kmap,
                     half * 64, slot, w.kvh, page, &kv_full[st]);
        }
      }
    }
  } else if (any && warp == kSoftmaxWarps) {
    // ---- products ----
    if (lane == 0) {
      constexpr uint32_t s_id = idesc(F16, kBlockKeys, false), o_id = idesc(F16, D, true);
      int pos = 0;
      uint32_t nq[2] = {0, 0}, np[2] = {0, 0};
      auto scores = [&](int t, int st) {
        const uint32_t qa = smem_addr(q_s + t * kTileBytes), ka = smem_addr(ring + st * kSlotBytes);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc_mma(tmem + 128 * t, sw128_desc(qa + (k / 4) * kHalf + (k % 4) * 32),
                 sw128_desc(ka + (k / 4) * kHalf + (k % 4) * 32), s_id, k > 0);
        tc_commit(&s_full[t]);
      };
      while (w.next(a)) {
        const int vis = w.tile_visible(a);
        const int nload = max(0, min(w.nblk, (vis + kBlockKeys - 1) / kBlockKeys - w.blk));
        if (nload == 0) continue;
        const int nt = w.rows(a) > 128 ? 2 : 1;
        int st = pos % kSlots;
        mbar_wait(&kv_full[st], (uint32_t)(pos / kSlots) & 1u, &g_paged_tc_error);
        for (int t = 0; t < nt; ++t) {
          mbar_wait(&q_full[t], nq[t]++ & 1u, &g_paged_tc_error);
          tc_fence_after();
          scores(t, st);
        }
        tc_commit(&kv_empty[st]);
        ++pos;
        for (int i = 0; i < nload; ++i) {
          const int vs = pos % kSlots, ks = (pos + 1) % kSlots;
          for (int t = 0; t < nt; ++t) {
            mbar_wait(&p_full[t], np[t]++ & 1u, &g_paged_tc_error);
            if (t == 0) mbar_wait(&kv_full[vs], (uint32_t)(pos / kSlots) & 1u, &g_paged_tc_error);
            tc_fence_after();
            const uint32_t va = smem_addr(ring + vs * kSlotBytes);
#pragma unroll
            for (int k = 0; k < kBlockKeys / 16; ++k)
              tc_mma_ta(tmem + 256 + D * t, tmem + 128 * t + 8 * k, v_desc<D>(va + k * 2048), o_id, i > 0 || k > 0);
            if (t == nt - 1) tc_commit(&kv_empty[vs]);
            if (i + 1 < nload) {
              if (t == 0) mbar_wait(&kv_full[ks], (uint32_t)((pos + 1) / kSlots) & 1u, &g_paged_tc_error);
              tc_fence_after();
              scores(t, ks);
              if (t == nt - 1) tc_commit(&kv_empty[ks]);
            } else {
              tc_commit(&o_full[t]);
            }
          }
          pos += i + 1 < nload ? 2 : 1;
        }
      }
    }
  } else if (any && warp < kSoftmaxWarps) {
    // ---- softmax, queries, epilogue ----
    const int t = warp >> 2, r = (warp & 3) * 32 + lane;  // row r of tile t
    const int row = t * 128 + r;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_tm = tmem + 128 * t + lanes, o_tm = tmem + 256 + D * t + lanes;
    // The row maximum is taken of the raw scores: a negative scale turns the queries' signs.
    const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    const float scale = fmaxf(fabsf(a.scale_log2), 1e-30f);
    int pos = 0;
    uint32_t ns = 0, no = 0;
    while (w.next(a)) {
      const int rows = w.rows(a), vis = w.tile_visible(a);
      const int nload = max(0, min(w.nblk, (vis + kBlockKeys - 1) / kBlockKeys - w.blk));
      const int base_pos = pos;
      pos += 2 * nload;
      if (t * 128 >= rows) continue;
      const bool whole = w.whole();
      float* slot = whole ? nullptr : a.ws + (int64_t)w.slot(w.c) * (kTcRows * (D + 2));
      float m = -INFINITY, l = 0.f;
      if (nload > 0) {
        // The queries of this tile: 16-byte chunks, rows past the last zero.
        for (int i = (warp & 3) * 32 + lane; i < 128 * (D / 8); i += 128) {
          const int qr = i / (D / 8), ch = i - qr * (D / 8), x = t * 128 + qr;
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (x < rows) {
            v = *reinterpret_cast<const uint4*>(a.q + w.token(a, x) * a.q_tok + w.head(a, x) * a.q_head + ch * 8);
            v.x ^= sign, v.y ^= sign, v.z ^= sign, v.w ^= sign;
          }
          sts128(smem_addr(q_s + t * kTileBytes) + (ch >> 3) * kHalf + qr * 128 + (((ch & 7) ^ (qr & 7)) << 4), v);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[t]);
        const int lim = row < rows ? w.row_visible(a, row) : 0;
        for (int i = 0; i < nload; ++i) {
          const int key0 = (w.blk + i) * kBlockKeys;
          mbar_wait(&s_full[t], ns++ & 1u, &g_paged_tc_error);
          tc_fence_after();
          float s[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld(s_tm + 32 * c, s + 32 * c);
          tmem_ld_wait<128>(s);
          if (__any_sync(0xffffffffu, lim < key0 + kBlockKeys)) {
#pragma unroll
            for (int k = 0; k < 128; ++k) s[k] = key0 + k < lim ? s[k] : -INFINITY;
          }
          float mx[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = s[k];
#pragma unroll
          for (int k = 4; k < 128; k += 8) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              mx[j] = k + 4 + j < 128 ? max3(mx[j], s[k + j], s[k + 4 + j]) : fmaxf(mx[j], s[k + j]);
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
          const bool move = top > m + 8.f || (m == -INFINITY && top > m);
          if (__any_sync(0xffffffffu, move)) {
            const float to = move ? top : m;
            if (i > 0) {
              const float f = move ? exp2_approx(m - to) : 1.f;
              l *= f;
#pragma unroll
              for (int c = 0; c < D / 32; ++c) {
                float o[32];
                tmem_ld(o_tm + 32 * c, o);
                tmem_ld_wait<32>(o);
                uint32_t x[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(o[k] * f);
                tmem_st32(o_tm + 32 * c, x);
              }
              tmem_st_wait();
            }
            m = to;
          }
          const float nb = m == -INFINITY ? 0.f : -m;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t p[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              float& x = s[64 * c + 2 * k];
              float& y = s[64 * c + 2 * k + 1];
              fma_pair(x, y, scale, nb);
              x = exp2_approx(x);
              y = exp2_approx(y);
              add_pair(sum[(k & 1) * 2], sum[(k & 1) * 2 + 1], x, y);
              p[k] = pack2<F16>(x, y);
            }
            tmem_st32(s_tm + 32 * c, p);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          if (t == 0 && key0 + kBlockKeys > vis) {
            // Slots past the last key may hold anything: their values are zeroed, as a weight of zero times a NaN
            // is not zero.
            const int vp = base_pos + 2 * i + 1, st = vp % kSlots;
            mbar_wait(&kv_full[st], (uint32_t)(vp / kSlots) & 1u, &g_paged_tc_error);
            if (key0 + r >= vis) {
              const uint32_t at = smem_addr(ring + st * kSlotBytes) + r * 128;
#pragma unroll
              for (int x = 0; x < D / 8; ++x) sts128(at + (x >> 3) * kHalf + (x & 7) * 16, make_uint4(0u, 0u, 0u, 0u));
            }
            fence_proxy_async_smem();
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[t]);
        }
        mbar_wait(&o_full[t], no++ & 1u, &g_paged_tc_error);
        tc_fence_after();
      }
      // ---- the rows' sums: out, or a piece ----
      const bool live = row < rows;
      const int64_t token = live ? w.token(a, row) : 0;
      const int head = live ? w.head(a, row) : 0;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        if (nload > 0) {
          tmem_ld(o_tm + 32 * c, o);
          tmem_ld_wait<32>(o);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0.f;
        }
        if (live) {
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = o[k + j];
            if (whole) {
              finish_row<D, F16, 8>(a, token, head, 32 * c + k, x, m, l);
            } else {
              float4* at = reinterpret_cast<float4*>(slot + row * D + 32 * c + k);
              at[0] = make_float4(x[0], x[1], x[2], x[3]);
              at[1] = make_float4(x[4], x[5], x[6], x[7]);
            }
          }
        }
      }
      if (live && !whole) *reinterpret_cast<float2*>(slot + kTcRows * D + 2 * row) = make_float2(m, l);
      tc_fence_before();  // the sums are read before the next item's first product (behind q_full and p_full)
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftmaxWarps) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of split items: block (c, y) takes every 16th group of rows
// of the item that begins in CTA c's run and ends beyond it, if there is one.
template <int D, bool F16>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  TileWalk w;
  if (!w.begin(a, lane)) return;
  bool found = false;
  while (w.next(a)) found = w.blk == 0 && w.nblk < w.blocks;
  if (found) merge_pieces<D, kTcRows, F16>(a, w, warp + 8 * blockIdx.y, 8 * gridDim.y, lane);
}

template <int D, bool F16>
cudaError_t launch(const CUtensorMap& k, const CUtensorMap& v, const PagedArgs& a, int ctas, cudaStream_t s) {
  auto kernel = paged_tc_kernel<D, F16>;
  static std::atomic<unsigned long long> configured{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured.load(std::memory_order_relaxed) & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_of(D));
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem_of(D);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, k, v, a);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3((unsigned)ctas, kMergeRowBlocks, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_merge_kernel<D, F16>, a);
}

}  // namespace

int read_paged_tc_error(cudaStream_t stream) { return read_error_word(&g_paged_tc_error, stream); }

cudaError_t launch_paged_tc(int D, bool f16, const CUtensorMap& k, const CUtensorMap& v, const PagedArgs& a, int ctas,
                            cudaStream_t s) {
  if (D == 128) return f16 ? launch<128, true>(k, v, a, ctas, s) : launch<128, false>(k, v, a, ctas, s);
  return f16 ? launch<64, true>(k, v, a, ctas, s) : launch<64, false>(k, v, a, ctas, s);
}

}  // namespace qi4
