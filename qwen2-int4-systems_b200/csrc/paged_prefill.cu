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
//             tensor memory are then rescaled, rarely. Also the epilogue.
//   8         issues the products: S = Q K^T (both operands from shared
//             memory), O += P V (P from tensor memory, V as it lies in the
//             page: key-major, the descriptor's transposed form). Products
//             execute in the order of issue, so "scores of unit i are there"
//             also says that the sums of unit i - 1 are.
//   9         fetches the queries (one TMA box of whole tokens per 64 dims) and,
//             page by page, keys and values into a ring of 128-key slots, keys
//             and values by turns (128-byte swizzle throughout).
// The weights of a unit are announced in two halves of 64 keys, so that the
// first half's product runs under the second half's exponentials. (Scores in
// halves of 64 columns as well, to have one half's always ready, took longer
// with one warp for the products: they are twice as many, and with N = 64 and
// both operands in shared memory each takes 48 cycles against 64 with N = 128.)
// Tensor memory: scores 2 x 128 columns, sums 2 x D. All waits are bounded.
//
// Measured (device time, BF16, 12 query heads on 2 KV heads of 128 dims): a
// prompt of 8192 tokens 251 us in calls back to back, 820 TFLOP/s; six ragged
// chunks of up to 2047 tokens 116 us. A unit takes some 4000 cycles: the tensor
// cores are active for 46% of them and the exponentials' pipe as long. Neither
// alone is the bound (the 230 us of a short burst, at higher clocks, which the
// figures below go by, become 198 without the exponentials, 213 with an eighth
// of the products): it is the chain scores - maximum - weights - product of a tile,
// which one tile alone takes as long for. Slower were: the maximum and the
// weights of a whole unit at once (288 us; 276 with registers moved from the
// other warps), 16 softmax warps of half a row each (313), a warp for the
// products of either tile (248; with scores in halves of 64 keys, always one
// ready, 230, and a quarter of the exponentials as polynomials then 225),
// products issued by the softmax warps (266 to 248 then), weights under the old
// maximum beside the search for the new (241).
#include <atomic>

#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace qi4 {

__device__ int g_paged_tc_error;

namespace {

constexpr int kThreads = 320;
constexpr int kSoftmaxWarps = 8;
constexpr int slot_bytes(int D) { return kBlockKeys * D * 2; }
constexpr int ring_slots(int D) { return D == 128 ? 5 : 10; }
constexpr size_t smem_of(int D) {
  return 1024 + (size_t)kTcRows * D * 2 + (size_t)ring_slots(D) * slot_bytes(D) +
         (12 + 2 * ring_slots(D)) * sizeof(uint64_t) + 16;
}

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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(taddr));
}
// Waits for the loads, and keeps every use of the N values behind the wait.
template <int N>
__device__ __forceinline__ void tmem_ld_wait(float* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(r[i]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
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

// Clears the odd values of a key's row (chunks in an order by which neighbouring rows r meet in no bank).
template <int D, bool F16>
__device__ __forceinline__ bool clear_row(uint32_t row, int half_bytes, int r) {
  uint32_t any = 0;
#pragma unroll
  for (int k = 0; k < D / 8; ++k) {
    const uint4 v = lds128(row + (k >> 3) * half_bytes + ((k ^ r) & 7) * 16);
    any |= odd_halves<F16>(v.x) | odd_halves<F16>(v.y) | odd_halves<F16>(v.z) | odd_halves<F16>(v.w);
  }
  if (!any) return false;
#pragma unroll 1
  for (int k = 0; k < D / 8; ++k) clear_odd<F16>(row + (k >> 3) * half_bytes + (k & 7) * 16);
  return true;
}

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap, const PagedArgs a) {
  constexpr int kSlots = ring_slots(D), kSlotBytes = slot_bytes(D), kHalf = kBlockKeys * 128;
  constexpr int kTileBytes = 128 * 128, kQHalf = kTcRows * 128;  // 128 rows, and 256 rows, of 64 dims
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_s = smem;                      // [D / 64][256 rows][128 B]: the tiles are its row halves
  uint8_t* ring = smem + kTcRows * D * 2;   // slots [D / 64][128 keys][128 B]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(ring + kSlots * kSlotBytes);  // TMA
  uint64_t* q_empty = q_full + 1;                                              // commit
  uint64_t* s_full = q_empty + 1;                                              // [2 tiles] commit
  uint64_t* p_full = s_full + 2;                                               // [2][2 halves] 4 warps
  uint64_t* o_done = p_full + 4;                                               // [2] commit, per half
  uint64_t* o_full = o_done + 2;                                               // [2] commit, per item
  uint64_t* kv_full = o_full + 2;                                              // [kSlots] TMA
  uint64_t* kv_empty = kv_full + kSlots;                                       // [kSlots] commit
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kv_empty + kSlots);
  int* odd = reinterpret_cast<int*>(tmem_slot + 1);  // the last piece with odd values to add

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&p_full[i], 4);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    *odd = 0;
    fence_barrier_init();
    prefetch_tensor_map(&qmap);
    prefetch_tensor_map(&kmap);
    prefetch_tensor_map(&vmap);
  }
  if (warp == kSoftmaxWarps) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // S0, S1 at 0, 128; O0, O1 at 256, 256 + D
  if (!a.late) pdl_wait();
  pdl_launch_dependents();

  Walk<kTcRows> w;
  const bool any = w.begin(a, lane);
  if (any && warp == kSoftmaxWarps + 1) {
    // ---- producer ----
    const int box_rows = 1 << a.box_shift;
    int pos = 0;  // ring position
    uint32_t nq = 0;
    while (w.next(a)) {
      const int vis = w.tile_visible(a);
      if (w.loaded(vis) > 0) {
        // The tile's queries: whole tokens of the KV head's G query heads are its rows in order. Tokens of the next
        // sequence that come with a sequence's last tile, and rows past the box, only make rows that nobody reads.
        mbar_wait(q_empty, (nq++ & 1u) ^ 1u, &g_paged_tc_error);
        if (lane == 0) {
          mbar_arrive_expect_tx(q_full, (uint32_t)(a.tile_rows * D * 2));
#pragma unroll
          for (int h = 0; h < D / 64; ++h)
            tma_load_3d(q_s + h * kQHalf, &qmap, 64 * h, w.kvh * a.G, w.first + w.tile * a.tile_tokens, q_full);
        }
        __syncwarp();
      }
      if (lane == 0 && a.fixed_len < 0 && __ldg(a.r.lengths + w.b) > a.cap)
        atomicOr(&g_paged_tc_error, kErrCacheFull);
      if (lane == 0 && a.one_tile && w.n * a.G > a.tile_rows)
        atomicOr(&g_paged_tc_error, QI4_DEVICE_TOO_MANY_TOKENS);
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
    if (lane == 0) note_split(a, w, true);
  } else if (any && warp == kSoftmaxWarps) {
    // ---- products ----
    // The whole warp runs the loops and the waits; one lane issues.
    constexpr uint32_t s_id = idesc(F16, kBlockKeys, false), o_id = idesc(F16, D, true);
    const uint64_t q_desc = sw128_desc(smem_addr(q_s)), k_desc = sw128_desc(smem_addr(ring)),
                   v_desc0 = v_desc<D>(smem_addr(ring));  // (descriptors count addresses in 16 bytes)
    int pos = 0;
    uint32_t nq = 0, np[2] = {0, 0};  // uses of q_full, and of p_full of either half
    // Scores of tile t and the keys of slot st; `last`: frees the slot, and `done` the queries.
    auto scores = [&](int t, int st, bool last, bool done) {
      tc_fence_after();
      if (elect_one()) {
        const uint64_t qd = q_desc + t * (kTileBytes >> 4), kd = k_desc + st * (kSlotBytes >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc_mma(tmem + 128 * t, qd + (((k / 4) * kQHalf + (k % 4) * 32) >> 4),
                 kd + (((k / 4) * kHalf + (k % 4) * 32) >> 4), s_id, k > 0);
        tc_commit(&s_full[t]);
        if (last) tc_commit(&kv_empty[st]);
        if (done) tc_commit(q_empty);
      }
      __syncwarp();
    };
    while (w.next(a)) {
      const int nload = w.loaded(w.tile_visible(a));
      if (nload == 0) continue;
      const int nt = w.rows(a) > 128 ? 2 : 1;
      const int k0 = pos % kSlots;
      mbar_wait(&kv_full[k0], (uint32_t)(pos / kSlots) & 1u, &g_paged_tc_error);
      mbar_wait(q_full, nq++ & 1u, &g_paged_tc_error);
      for (int t = 0; t < nt; ++t) scores(t, k0, t == nt - 1, t == nt - 1 && nload == 1);
      ++pos;
      for (int i = 0; i < nload; ++i) {
        const bool more = i + 1 < nload;
        const int vs = pos % kSlots, ks = (pos + 1) % kSlots;
        const uint64_t vd = v_desc0 + vs * (kSlotBytes >> 4);
        for (int t = 0; t < nt; ++t) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mbar_wait(&p_full[2 * t + x], np[t] & 1u, &g_paged_tc_error);
            if (x == 0 && t == 0) mbar_wait(&kv_full[vs], (uint32_t)(pos / kSlots) & 1u, &g_paged_tc_error);
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                tc_mma_ta(tmem + 256 + D * t, tmem + 128 * t + 64 * x + 8 * k, vd + (4 * x + k) * (2048 >> 4), o_id,
                          i > 0 || x > 0 || k > 0);
              tc_commit(&o_done[t]);
              if (x == 1 && !more) tc_commit(&o_full[t]);
              if (x == 1 && t == nt - 1) tc_commit(&kv_empty[vs]);
            }
            __syncwarp();
          }
          ++np[t];
          if (more) {
            if (t == 0) mbar_wait(&kv_full[ks], (uint32_t)((pos + 1) / kSlots) & 1u, &g_paged_tc_error);
            scores(t, ks, t == nt - 1, t == nt - 1 && i + 2 == nload);
          }
        }
        pos += more ? 2 : 1;
      }
    }
  } else if (warp < kSoftmaxWarps) {
    // ---- softmax, queries, epilogue ----
    const int t = warp >> 2, r = (warp & 3) * 32 + lane;  // row r of tile t
    const int row = t * 128 + r;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_tm = tmem + 128 * t + lanes, o_tm = tmem + 256 + D * t + lanes;
    // The row maximum is taken of the raw scores (the scale is not negative here; never zero, which would make
    // a hidden key's -inf a NaN).
    const float scale = fmaxf(a.scale_log2, 1e-30f);
    int pos = 0, item = 0;
    uint32_t ns = 0, no = 0, done = 0;  // uses of s_full, o_full, and o_done
    bool have = any && w.next(a);
    while (have) {
      ++item;
      const int rows = w.rows(a), vis = w.tile_visible(a), nload = w.loaded(vis);
      const int base_pos = pos;
      pos += 2 * nload;
      if (t * 128 >= rows) {
        have = w.next(a);
        continue;
      }
      const bool whole = w.whole(), live = row < rows;
      float* slot = whole ? nullptr : a.ws + (int64_t)w.slot(blockIdx.x) * (kTcRows * (D + 2));
      int token = 0, head = 0;
      if (live) w.place(a, row, token, head);
      const int lim = live ? w.row_visible(a, row) : 0, blk0 = w.blk;
      const int lim_min = min(vis, w.row_visible(a, 0));  // the tile's first token sees the fewest keys
      const int seq = w.b, kvh = w.kvh;
      float m = -INFINITY, l = 0.f;
      for (int h = 0; h < 2 * nload; ++h) {  // halves of 64 keys
        const int x = h & 1, key0 = (blk0 + (h >> 1)) * kBlockKeys + 64 * x;
        const uint32_t s_at = s_tm + 64 * x;
        if (t == 0 && x == 0 && key0 + kBlockKeys > lim_min) {
          // Slots past the last key may hold anything: their values are zeroed, as a weight of zero times a NaN is
          // not zero. So are the odd ones of keys that not every row sees. (Here, while the scores are on their way:
          // behind the weights it is on the path from one unit to the next: 8192 tokens 257 us against 250.)
          const int vp = base_pos + h + 1, st = vp % kSlots;
          mbar_wait(&kv_full[st], (uint32_t)(vp / kSlots) & 1u, &g_paged_tc_error);
          const uint32_t at = smem_addr(ring + st * kSlotBytes) + r * 128;
          if (key0 + r >= vis) {
#pragma unroll
            for (int k = 0; k < D / 8; ++k) sts128(at + (k >> 3) * kHalf + (k & 7) * 16, make_uint4(0u, 0u, 0u, 0u));
          } else if (key0 + r >= lim_min && clear_row<D, F16>(at, kHalf, r)) {
            atomicMax(odd, item);
          }
          fence_proxy_async_smem();
        }
        if (x == 0) mbar_wait(&s_full[t], ns++ & 1u, &g_paged_tc_error);
        tc_fence_after();
        float s[64];
        tmem_ld(s_at, s);
        tmem_ld(s_at + 32, s + 32);
        tmem_ld_wait<64>(s);
        if (__any_sync(0xffffffffu, lim < key0 + 64)) {
#pragma unroll
          for (int k = 0; k < 64; ++k) s[k] = key0 + k < lim ? s[k] : -INFINITY;
        }
        float mx[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) mx[j] = fmaxf(s[j], s[j + 4]);
#pragma unroll
        for (int k = 8; k < 64; k += 8)
#pragma unroll
          for (int j = 0; j < 4; ++j) mx[j] = max3(mx[j], s[k + j], s[k + 4 + j]);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
        const bool move = top > m + 8.f;
        if (__any_sync(0xffffffffu, move)) {
          const float to = move ? top : m;
          if (h > 0) {
            // The sums of the half before must be complete (phase done + h - 1). Those of the unit before are, as
            // this unit's scores were issued behind them, so the parity says which phase it is.
            mbar_wait(&o_done[t], (done + h - 1) & 1u, &g_paged_tc_error);
            tc_fence_after();
            const float f = move ? exp2_approx(m - to) : 1.f;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              float o[16];
              tmem_ld16(o_tm + 16 * c, o);
              tmem_ld_wait<16>(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] *= f;
              tmem_st16(o_tm + 16 * c, reinterpret_cast<uint32_t*>(o));
            }
          }
          m = to;
        }
        const float nb = m == -INFINITY ? 0.f : kLift<F16> - m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float &u = s[32 * c + 2 * k], &v = s[32 * c + 2 * k + 1];
            fma_pair(u, v, scale, nb);
            u = exp2_approx(u);
            v = exp2_approx(v);
            add_pair(sum[(k & 1) * 2], sum[(k & 1) * 2 + 1], u, v);
            p[k] = pack2<F16>(u, v);
          }
          tmem_st16(s_at + 16 * c, p);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + x]);
      }
      have = w.next(a);
      if (a.late) pdl_wait();
      if (nload > 0) {
        done += 2 * nload;
        mbar_wait(&o_full[t], no++ & 1u, &g_paged_tc_error);
        tc_fence_after();
      }
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        float o[16];
        if (nload > 0) {
          tmem_ld16(o_tm + 16 * c, o);
          tmem_ld_wait<16>(o);
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = 0.f;
        }
        if (live) {
          if (whole) {
            finish_row<D, F16, 16>(a, token, head, 16 * c, o, m, l);
          } else {
            // (dims major: a warp's 32 rows side by side)
#pragma unroll
            for (int k = 0; k < 16; ++k) slot[(16 * c + k) * kTcRows + row] = o[k];
          }
        }
      }
      if (live && !whole) *reinterpret_cast<float2*>(slot + kTcRows * D + 2 * row) = make_float2(m, l);
      // (Tile 1 sees the word too: the products behind its sums were issued after tile 0 had announced its weights.)
      if (live && *static_cast<volatile int*>(odd) >= item) {
        const int64_t at = (int64_t)token * (a.Hkv * a.G) + head;
        add_odd<F16>(a, seq, kvh, max(lim_min, blk0 * kBlockKeys), min(lim, (blk0 + nload) * kBlockKeys), 0, D,
                     a.out + at * D, !whole ? slot + row : a.state_acc ? a.state_acc + at * D : nullptr,
                     whole ? 1 : kTcRows);
      }
      tc_fence_before();  // the sums are read before the next item's first weights are announced
    }
  }
  if (!any && threadIdx.x == 0) note_split(a, w, false);
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftmaxWarps) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of the split items. A piece is [D][kTcRows] sums, then
// [kTcRows] (max, sum): lanes are rows. A share is 32 rows: all dims of an item
// of few pieces, 32 dims of one of many, each warp an eighth of them, with 32
// loads under way in every thread.
template <int D, int kPieces, int kDims>
__device__ __forceinline__ void join_rows(const float* first, const float* later, int np, int d, int r, float (&acc)[kDims],
                                          float& top, float& l) {
  constexpr int64_t kSlot = (int64_t)kTcRows * (D + 2);
#pragma unroll
  for (int k = 0; k < kDims; ++k) acc[k] = 0.f;
  top = -INFINITY, l = 0.f;
  for (int p0 = 0; p0 < np; p0 += kPieces) {
    float v[kPieces][kDims];
    float2 ml[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int p = p0 + i;
      ml[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < kDims; ++k) v[i][k] = 0.f;
      if (p < np) {
        const float* src = p ? later + 2 * p * kSlot : first;
        ml[i] = *reinterpret_cast<const float2*>(src + (int64_t)kTcRows * D + 2 * r);
#pragma unroll
        for (int k = 0; k < kDims; ++k) v[i][k] = src[(d + k) * kTcRows + r];
      }
    }
    float to = top;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) to = fmaxf(to, ml[i].x);
    const float base = to == -INFINITY ? 0.f : to, back = exp2_approx(top - base);
    top = to;
    l *= back;
#pragma unroll
    for (int k = 0; k < kDims; ++k) acc[k] *= back;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const float f = exp2_approx(ml[i].x - base);
      l += ml[i].y * f;
#pragma unroll
      for (int k = 0; k < kDims; ++k) acc[k] += v[i][k] * f;
    }
  }
}

template <int D, bool F16>
__global__ void __launch_bounds__(kJoinThreads) paged_tc_join_kernel(const PagedArgs a, int ctas) {
  constexpr int64_t kSlot = (int64_t)kTcRows * (D + 2);
  constexpr int kFew = 4;
  __shared__ float out_s[32][D + 1], top_s[32], l_s[32];
  __shared__ int ends[kMaxCtas];
  pdl_launch_dependents();
  pdl_wait();
  const int total = count_shares(a.splits, ctas, ends, [](int pieces, int rows) {
    return (rows + 31) / 32 * (pieces <= kFew ? 1 : D / 32);
  });
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int u = blockIdx.x; u < total; u += gridDim.x) {
    int part;
    const int c = share_owner(ends, ctas, u, part);
    const SplitItem it = a.splits[c];
    const bool few = it.pieces <= kFew;
    const int z = few ? 0 : part % (D / 32), r0 = 32 * (few ? part : part / (D / 32));
    const int r = min(r0 + lane, kTcRows - 1), dims = few ? D : 32;
    const float* first = a.ws + it.slot * kSlot;
    const float* later = a.ws + 2 * (int64_t)c * kSlot;
    float top, l;
    if (few) {
      constexpr int kEach = D / 8;
      float acc[kEach];
      join_rows<D, 2, kEach>(first, later, it.pieces, kEach * warp, r, acc, top, l);
#pragma unroll
      for (int k = 0; k < kEach; ++k) out_s[lane][kEach * warp + k] = acc[k];
    } else {
      float acc[4];
      join_rows<D, 8, 4>(first, later, it.pieces, 32 * z + 4 * warp, r, acc, top, l);
#pragma unroll
      for (int k = 0; k < 4; ++k) out_s[lane][4 * warp + k] = acc[k];
    }
    if (warp == 0) top_s[lane] = top, l_s[lane] = l;
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * dims / 4; i += kJoinThreads) {
      const int orow = i / (dims / 4), od = (i - orow * (dims / 4)) * 4;
      if (r0 + orow < it.rows) {
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = out_s[orow][od + k];
        const int row = it.row0 + r0 + orow, token = a.by_G(row);
        finish_row<D, F16, 4>(a, it.first + token, it.kvh * a.G + row - token * a.G, 32 * z + od, x, top_s[orow],
                              l_s[orow]);
      }
    }
    __syncthreads();  // the next share's sums replace these
  }
}

template <int D, bool F16>
cudaError_t launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const PagedArgs& a, int ctas,
                   cudaStream_t s) {
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, q, k, v, a);
  if (e != cudaSuccess || a.unsplit) return e;
  cfg.gridDim = dim3((unsigned)(kJoinBlocksPerSm * ctas), 1, 1);
  cfg.blockDim = dim3(kJoinThreads, 1, 1);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_tc_join_kernel<D, F16>, a, ctas);
}

}  // namespace

int read_paged_tc_error(cudaStream_t stream) { return read_error_word(&g_paged_tc_error, stream); }

cudaError_t launch_paged_tc(int D, bool f16, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                            const PagedArgs& a, int ctas, cudaStream_t s) {
  if (D == 128) return f16 ? launch<128, true>(q, k, v, a, ctas, s) : launch<128, false>(q, k, v, a, ctas, s);
  return f16 ? launch<64, true>(q, k, v, a, ctas, s) : launch<64, false>(q, k, v, a, ctas, s);
}

}  // namespace qi4
