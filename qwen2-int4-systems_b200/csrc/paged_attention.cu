// Attention of a ragged batch's new tokens over a paged KV cache (sm_100a):
//   out[t, h] = sum_j w_j V[j] / sum_j w_j,   w_j = exp(scale q[t, h] . K[j])
// over the keys j the token sees (causal: token i of n sees keys up to
// length - n + i). Work split and merging: paged_attention.cuh.
//
// This kernel serves rows that are few per key (decode steps, drafts; larger
// counts go to paged_prefill.cu): it is
// bound by the one pass over the keys and values. One CTA per SM; a producer
// warp fetches units of 128 keys page by page (one TMA box per page and 64
// dimensions, 128-byte swizzle) into a ring of 64 KB (D = 128) stages, three
// of them: 192 KB in flight per SM, four times what the HBM latency asks for.
// Eight warps take 16 keys each on mma.sync, keys as the 16 rows and the query
// rows as columns of 8, so 6 query heads of a KV head waste 2 columns and not
// 10. Scores S^T = K Q^T, a softmax on the score registers with a maximum per
// warp that moves only when a score exceeds it by more than 2^8, O^T += V^T P^T
// with P split into a 16-bit value and its 16-bit remainder (the products keep
// 16 bits of each weight in BF16, 22 in FP16 down to steps of 2^-32 of the
// largest weight; the second product is hidden behind the loads). The warps' sums meet in the stage of the item's last unit, which is
// released afterwards.
//
// Measured (device time, BF16, 12 query heads on 2 KV heads of 128 dims): one
// sequence of 131,002 keys 30 us, 64 sequences of 1151 keys 22.7 us; per
// further unit 6 to 7 TB/s, so what bounds them is the 9 to 11 us of a call
// that do not grow with the keys: the launch, each warp's way to its first unit
// (boundaries, lengths and page table, one after the other), the warps' sums,
// the joining launch. Items that leave two CTAs or more for each, of tables that
// are not long, are a cluster's work, without a joining launch: one sequence of
// 641 keys 6.5 us, 16 of 450 keys 6.7.
// Sixteen consumer warps in two groups that take the units
// by turns had 96 registers each and were slower (25.1 us for the 64).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "paged_attention.cuh"

namespace cg = cooperative_groups;

namespace qi4 {

__device__ int g_paged_error;

namespace {

constexpr int kWarps = 8;                        // consumer warps
constexpr int kThreads = 32 * (kWarps + 1);      // and the producer
constexpr int stages_of(int D) { return D == 128 ? 3 : 6; }
constexpr int stage_bytes(int D) { return 2 * kBlockKeys * D * 2; }
constexpr size_t smem_of(int D, int NT, bool clusters) {
  return 1024 + (size_t)stages_of(D) * stage_bytes(D) + (size_t)8 * NT * (2 * D + 16) +
         2 * 2 * kWarps * 8 * NT * sizeof(float) + 2 * stages_of(D) * sizeof(uint64_t) +
         (clusters ? 8 * NT * (D + 2) * sizeof(float) : 0) + sizeof(int);
}

template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
// kClusters: an item is the work of one cluster, whose CTAs share its units out
// in order and exchange their sums over distributed shared memory; else the
// units are dealt to all CTAs (paged_attention.cuh).
template <int D, int NT, bool F16, bool kClusters>
__global__ void __launch_bounds__(kThreads, 1)
    paged_decode_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                        const PagedArgs a) {
  constexpr int R = 8 * NT;
  constexpr int kStages = stages_of(D), kStageBytes = stage_bytes(D), kHalfBytes = kBlockKeys * 128;
  constexpr int kQRow = 2 * D + 16;  // bytes of a staged query row (padded: conflict-free)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_s = smem + kStages * kStageBytes;
  float* red_m = reinterpret_cast<float*>(q_s + R * kQRow);  // [2][kWarps][R]
  float* red_l = red_m + 2 * kWarps * R;
  uint64_t* full = reinterpret_cast<uint64_t*>(red_l + 2 * kWarps * R);
  uint64_t* empty = full + kStages;
  float* part = reinterpret_cast<float*>(empty + kStages);  // kClusters: [R][D] sums, [R] (max, sum)
  int* odd = reinterpret_cast<int*>(part + (kClusters ? R * (D + 2) : 0));  // the last item with odd values to add

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    *odd = 0;
    fence_barrier_init();
    prefetch_tensor_map(&kmap);
    prefetch_tensor_map(&vmap);
  }
  __syncthreads();
  // The next launch may be scheduled once every CTA has passed its own wait:
  // what it reads before its wait is then older than this launch.
  if (!a.late) pdl_wait();
  pdl_launch_dependents();

  Walk<R> w;
  if constexpr (kClusters) {
    const int C = (int)cg::this_cluster().num_blocks(), item = (int)blockIdx.x / C;
    if (!w.share(a, item, (int)blockIdx.x - item * C, C)) return;  // (no tokens: the whole cluster)
  } else if (!w.begin(a, lane)) {
    if (threadIdx.x == 0) note_split(a, w, false);
    return;
  }
  int stage = 0;
  uint32_t phase = 0;

  if (warp == kWarps) {
    // ---- producer: pages -> ring ----
    const int box_rows = 1 << a.box_shift;
    for (bool one = true; kClusters ? one : w.next(a); one = false) {
      const int vis = w.tile_visible(a);
      const int nload = w.loaded(vis);
      if (lane == 0 && a.fixed_len < 0 && __ldg(a.r.lengths + w.b) > a.cap) atomicOr(&g_paged_error, kErrCacheFull);
      if (lane == 0 && a.one_tile && w.n * a.G > a.tile_rows) atomicOr(&g_paged_error, QI4_DEVICE_TOO_MANY_TOKENS);
      int win0 = -1, win = -1;  // table entries win0 .. win0 + 31, one per lane
      for (int i = 0; i < nload; ++i) {
        const int key0 = (w.blk + i) * kBlockKeys;
        const int nb = (min(kBlockKeys, vis - key0) + box_rows - 1) >> a.box_shift;  // boxes per 64 dims
        const int pj = key0 >> a.page_shift, slot = key0 & ((1 << a.page_shift) - 1);
        if ((pj & ~31) != win0) {
          win0 = pj & ~31;
          const int j = win0 + lane;
          win = j < a.table_width ? __ldg(a.table + w.b * a.table_stride + j) : -1;
        }
        mbar_wait(&empty[stage], phase ^ 1u, &g_paged_error);
        const int boxes = 2 * (D / 64) * nb;
        if (lane == 0) mbar_arrive_expect_tx(&full[stage], (uint32_t)(boxes * box_rows * 128));
        __syncwarp();
        const uint32_t base = smem_addr(smem + stage * kStageBytes);
        for (int j0 = 0; j0 < boxes; j0 += 32) {
          const int j = j0 + lane;
          const int bx = j / (2 * (D / 64)), part = j - bx * (2 * (D / 64));  // part: K or V, 64-dim half
          const int page = __shfl_sync(0xffffffffu, win, (pj + min(bx, nb - 1)) & 31);
          if (j < boxes) {
            // A page outside the pool reads as zeros (the copy's own bounds), and is reported.
            if (part == 0 && (page < 0 || page >= a.pages)) atomicOr(&g_paged_error, kErrBadPage);
            load_box(base + part * kHalfBytes + (bx << a.box_shift) * 128, part < D / 64 ? &kmap : &vmap,
                     (part % (D / 64)) * 64, slot, w.kvh, page, &full[stage]);
          }
        }
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if constexpr (!kClusters) {
      if (lane == 0) note_split(a, w, true);
      return;
    }
  }

  // ---- consumers ----
  const int gq = lane >> 2, tq = lane & 3;
  const int r0 = warp * 16;  // this warp's keys of every unit
  const int lrow = r0 + (lane & 7) + (((lane >> 3) & 1) << 3), lchunk = lane >> 4, lx = lane & 7;
  int par = 0, item = 0;
  for (bool one = warp < kWarps; kClusters ? one : w.next(a); one = false) {
    ++item;
    const int rows = w.rows(a), vis = w.tile_visible(a), nload = w.loaded(vis);
    if (kClusters && nload == 0) {
      if (threadIdx.x < R) *reinterpret_cast<float2*>(part + R * D + 2 * threadIdx.x) = make_float2(-INFINITY, 0.f);
    } else if (nload == 0) {  // no row sees a key
      if (a.late) pdl_wait();
      for (int i = threadIdx.x; i < rows * (D / 4); i += 32 * kWarps) {
        const int r = i / (D / 4);
        float none[4] = {0.f, 0.f, 0.f, 0.f};
        int token, head;
        w.place(a, r, token, head);
        finish_row<D, F16, 4>(a, token, head, (i - r * (D / 4)) * 4, none, -INFINITY, 0.f);
      }
    } else {
      // The tile's queries (rows past the last are zero).
      for (int i = threadIdx.x; i < R * (D / 8); i += 32 * kWarps) {
        const int r = i / (D / 8), ch = i - r * (D / 8);
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows) {
          int token, head;
          w.place(a, r, token, head);
          v = *reinterpret_cast<const uint4*>(a.q + token * a.q_tok + head * a.q_head + ch * 8);
        }
        sts128(smem_addr(q_s) + r * kQRow + ch * 16, v);
      }
      named_barrier(1, 32 * kWarps);
      uint32_t qf[NT == 1 ? D / 16 : 1][2];
      const uint32_t q_addr = smem_addr(q_s) + (lane & 7) * kQRow + (lane >> 3) * 16;
      if constexpr (NT == 1) {
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
          ldsm4(q_addr + ks * 64, qf[2 * ks][0], qf[2 * ks][1], qf[2 * ks + 1][0], qf[2 * ks + 1][1]);
        }
      }
      int lim[NT][2];  // keys that query row nt * 8 + 2 tq + e sees
      int lim_min = vis;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + 2 * tq + e;
          lim[nt][e] = r < rows ? w.row_visible(a, r) : 0;
          if (r < rows) lim_min = min(lim_min, lim[nt][e]);
        }
      lim_min = __reduce_min_sync(0xffffffffu, lim_min);
      float m[NT][2], l[NT][2], o[D / 16][NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) o[mt][nt][0] = o[mt][nt][1] = o[mt][nt][2] = o[mt][nt][3] = 0.f;
      }
      int held = 0;
      for (int i = 0; i < nload; ++i) {
        const int key0 = (w.blk + i) * kBlockKeys + r0;
        mbar_wait(&full[stage], phase, &g_paged_error);
        const uint32_t kb = smem_addr(smem + stage * kStageBytes) + lrow * 128;
        const uint32_t vb = kb + (D / 64) * kHalfBytes;
        if (key0 < vis) {
          if (key0 + 16 > lim_min) {
            // Slots past the last key may hold anything: their values are
            // zeroed, as a weight of zero times a NaN is not zero. So are the
            // odd ones of keys that not every row sees.
            for (int j = lane; j < 16 * (D / 8); j += 32) {
              const int r = j / (D / 8), ch = j - r * (D / 8);
              if (key0 + r >= vis)
                sts128(smem_addr(smem + stage * kStageBytes) + (D / 64 + (ch >> 3)) * kHalfBytes + (r0 + r) * 128 +
                           ((ch & 7) << 4), make_uint4(0u, 0u, 0u, 0u));
            }
            const int some = min(16, vis - key0) * (D / 8);
#pragma unroll 1
            for (int j = max(0, lim_min - key0) * (D / 8) + lane; j < some; j += 32) {
              const int r = j / (D / 8), ch = j - r * (D / 8);
              if (clear_odd<F16>(smem_addr(smem + stage * kStageBytes) + (D / 64 + (ch >> 3)) * kHalfBytes +
                                 (r0 + r) * 128 + ((ch & 7) << 4)))
                atomicMax(odd, item);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          float sc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
          for (int k2 = 0; k2 < D / 32; ++k2) {
            uint32_t ka[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int ch = (2 * k2 + h) * 2 + lchunk;
              ldsm4(kb + (ch >> 3) * kHalfBytes + (((ch & 7) ^ lx) << 4), ka[h][0], ka[h][1], ka[h][2], ka[h][3]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint32_t q0, q1, q2, q3;
              if constexpr (NT == 1) {
                q0 = qf[2 * k2][0], q1 = qf[2 * k2][1], q2 = qf[2 * k2 + 1][0], q3 = qf[2 * k2 + 1][1];
              } else {
                ldsm4(q_addr + nt * 8 * kQRow + k2 * 64, q0, q1, q2, q3);
              }
              mma16816<F16>(sc[nt], ka[0], q0, q1);
              mma16816<F16>(sc[nt], ka[1], q2, q3);
            }
          }
          // Hidden keys, and whether a score leaves its row's maximum more than 2^8 behind.
          const bool masked = key0 + 16 > lim_min;
          bool move = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float &x0 = sc[nt][e], &x1 = sc[nt][2 + e];
              x0 *= a.scale_log2, x1 *= a.scale_log2;
              if (masked || lim[nt][e] == 0) {
                x0 = key0 + gq < lim[nt][e] ? x0 : -INFINITY;
                x1 = key0 + gq + 8 < lim[nt][e] ? x1 : -INFINITY;
              }
              move |= fmaxf(x0, x1) > m[nt][e] + 8.f;
            }
          if (__any_sync(0xffffffffu, move)) {
            // The maxima move (in the first unit, and rarely after it): the sums so far are rescaled.
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float t = fmaxf(sc[nt][e], sc[nt][2 + e]);
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                const float mn = fmaxf(m[nt][e], t), alpha = mn == -INFINITY ? 1.f : exp2_approx(m[nt][e] - mn);
                m[nt][e] = mn;
                l[nt][e] *= alpha;
#pragma unroll
                for (int mt = 0; mt < D / 16; ++mt) {
                  o[mt][nt][e] *= alpha;
                  o[mt][nt][2 + e] *= alpha;
                }
              }
          }
          uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float base = m[nt][e] == -INFINITY ? 0.f : m[nt][e] - kLift<F16>;
              p[e] = exp2_approx(sc[nt][e] - base);
              p[2 + e] = exp2_approx(sc[nt][2 + e] - base);
              l[nt][e] += p[e] + p[2 + e];  // this lane's keys; summed over gq at the end
            }
            const uint32_t h0 = pack2<F16>(p[0], p[1]), h1 = pack2<F16>(p[2], p[3]);
            const float2 f0 = unpack2<F16>(h0), f1 = unpack2<F16>(h1);
            ph[nt][0] = transpose8x8(h0);
            ph[nt][1] = transpose8x8(h1);
            pl[nt][0] = transpose8x8(pack2<F16>(p[0] - f0.x, p[1] - f0.y));
            pl[nt][1] = transpose8x8(pack2<F16>(p[2] - f1.x, p[3] - f1.y));
          }
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt) {
            uint32_t va[4];
            const int ch = mt * 2 + lchunk;
            ldsm4_t(vb + (ch >> 3) * kHalfBytes + (((ch & 7) ^ lx) << 4), va[0], va[2], va[1], va[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<F16>(o[mt][nt], va, ph[nt][0], ph[nt][1]);
              mma16816<F16>(o[mt][nt], va, pl[nt][0], pl[nt][1]);
            }
          }
        }
        if (i + 1 < nload) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[stage]);
        } else {
          held = stage;  // the last unit's stage becomes the buffer of the reduction below
        }
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // ---- the warps' sums ----
      float* rm = red_m + par * kWarps * R;
      float* rl = red_l + par * kWarps * R;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float t = l[nt][e];
          t += __shfl_xor_sync(0xffffffffu, t, 4);
          t += __shfl_xor_sync(0xffffffffu, t, 8);
          t += __shfl_xor_sync(0xffffffffu, t, 16);
          if (gq == 0) {
            rm[warp * R + nt * 8 + 2 * tq + e] = m[nt][e];
            rl[warp * R + nt * 8 + 2 * tq + e] = t;
          }
        }
      named_barrier(1, 32 * kWarps);  // every warp is done with the held stage
      // Buffers [R][D], dims swizzled so that the fragments' stores spread over the banks: one per warp where they
      // fit the stage, else one for each of four warps, which add theirs to another's.
      constexpr int kBuffers = NT <= 2 ? kWarps : kWarps / 2;
      float* buf = reinterpret_cast<float*>(smem + held * kStageBytes);
      static_assert(kBuffers * R * D * sizeof(float) <= (size_t)stage_bytes(D), "the sums must fit one stage");
      float f[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = -INFINITY;
#pragma unroll
          for (int x = 0; x < kWarps; ++x) top = fmaxf(top, rm[x * R + nt * 8 + 2 * tq + e]);
          f[nt][e] = m[nt][e] == -INFINITY ? 0.f : exp2_approx(m[nt][e] - top);
        }
      float* mine = buf + (warp % kBuffers) * R * D;
#pragma unroll
      for (int round = 0; round < kWarps / kBuffers; ++round) {
        if (kBuffers == kWarps || (warp >= kBuffers) == (round == 0)) {
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const int r = nt * 8 + 2 * tq + (x & 1), d = mt * 16 + gq + (x >> 1) * 8;
                float* at = mine + r * D + (d ^ (tq << 3));
                const float v = o[mt][nt][x] * f[nt][x & 1];
                *at = round == 0 ? v : *at + v;
              }
        }
        named_barrier(1, 32 * kWarps);
      }
      constexpr int kLanes = D / 4;
      if (!kClusters && a.late) pdl_wait();
      const bool whole = !kClusters && w.whole();
      float* slot = kClusters ? part : whole ? nullptr : a.ws + (int64_t)w.slot(blockIdx.x) * (R * (D + 2));
      for (int i = threadIdx.x; i < rows * kLanes; i += 32 * kWarps) {
        const int r = i / kLanes, d = (i - r * kLanes) * 4;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int x = 0; x < kWarps; ++x) top = fmaxf(top, rm[x * R + r]);
#pragma unroll
        for (int x = 0; x < kWarps; ++x)  // (a warp without a maximum has a sum of 0, or of NaN where no score is a number)
          sum += rm[x * R + r] == -INFINITY ? rl[x * R + r] : rl[x * R + r] * exp2_approx(rm[x * R + r] - top);
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < kBuffers; ++x) {
          const float4 v = *reinterpret_cast<const float4*>(buf + (x * R + r) * D + (d ^ (((r >> 1) & 3) << 3)));
          acc[0] += v.x, acc[1] += v.y, acc[2] += v.z, acc[3] += v.w;
        }
        if (whole) {
          int token, head;
          w.place(a, r, token, head);
          finish_row<D, F16, 4>(a, token, head, d, acc, top, sum);
        } else {
          *reinterpret_cast<float4*>(slot + r * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
          if (d == 0) *reinterpret_cast<float2*>(slot + R * D + 2 * r) = make_float2(top, sum);
        }
      }
      if (*static_cast<volatile int*>(odd) >= item) {  // (written before the barriers above)
#pragma unroll 1
        for (int i = threadIdx.x; i < rows * kLanes; i += 32 * kWarps) {
          const int r = i / kLanes, d = (i - r * kLanes) * 4;
          int token, head;
          w.place(a, r, token, head);
          const int64_t row = (int64_t)token * (a.Hkv * a.G) + head;
          add_odd<F16>(a, w.b, w.kvh, max(lim_min, w.blk * kBlockKeys),
                       min(w.row_visible(a, r), (w.blk + nload) * kBlockKeys), d, 4, a.out + row * D,
                       !whole ? slot + r * D : a.state_acc ? a.state_acc + row * D : nullptr, 1);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[held]);
      par ^= 1;
    }
  }
  if constexpr (kClusters) {
    // The cluster's CTAs share out the rows' dims; the pieces are joined in their order.
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (a.late) pdl_wait();
    const int C = (int)cluster.num_blocks(), rows = w.rows(a);
    constexpr int kLanes = D / 4;
    for (int i = (int)cluster.block_rank() * kThreads + threadIdx.x; i < rows * kLanes; i += C * kThreads) {
      const int r = i / kLanes, d = (i - r * kLanes) * 4;
      float acc[4] = {0.f, 0.f, 0.f, 0.f}, top = -INFINITY, sum = 0.f;
      for (int p0 = 0; p0 < C; p0 += 8) {
        float2 ml[8];
        float4 v[8];
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          ml[p] = make_float2(-INFINITY, 0.f);
          if (p0 + p < C) {
            const float* there = cluster.map_shared_rank(part, p0 + p);
            ml[p] = *reinterpret_cast<const float2*>(there + R * D + 2 * r);
            v[p] = *reinterpret_cast<const float4*>(there + r * D + d);
          }
        }
        float to = top;
#pragma unroll
        for (int p = 0; p < 8; ++p) to = fmaxf(to, ml[p].x);
        const float base = to == -INFINITY ? 0.f : to, back = exp2_approx(top - base);
        top = to;
        sum *= back;
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] *= back;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          // A piece that saw no key has written no sums. (One whose scores are no numbers has: its sum of weights is NaN.)
          if (ml[p].x == -INFINITY && ml[p].y == 0.f) continue;
          const float f = exp2_approx(ml[p].x - base);
          sum += ml[p].y * f;
          acc[0] += v[p].x * f, acc[1] += v[p].y * f, acc[2] += v[p].z * f, acc[3] += v[p].w * f;
        }
      }
      int token, head;
      w.place(a, r, token, head);
      finish_row<D, F16, 4>(a, token, head, d, acc, top, sum);
    }
    cluster.sync();  // no CTA leaves while its sums are read
  }
}

// Joins the pieces of the split items. Groups of D / 4 lanes, eight pieces'
// loads under way in each: of an item of few pieces every group takes a row; of
// one of many the groups share a row's pieces, and their sums meet in shared
// memory in the groups' order.
template <int D, int R, bool F16>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedArgs a, int ctas) {
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes, kAtOnce = 8;
  constexpr int64_t kSlot = (int64_t)R * (D + 2);
  __shared__ float4 acc_s[kGroups][kLanes];
  __shared__ float2 ml_s[kGroups];
  __shared__ int ends[kMaxCtas];
  pdl_launch_dependents();  // (what follows waits for this launch, and it for the one before)
  pdl_wait();
  const int total = count_shares(a.splits, ctas, ends, [](int pieces, int rows) {
    return pieces <= kAtOnce ? (rows + kGroups - 1) / kGroups : rows;
  });
  const int group = threadIdx.x / kLanes, d = (threadIdx.x % kLanes) * 4;
  for (int u = blockIdx.x; u < total; u += gridDim.x) {
    int part;
    const int c = share_owner(ends, ctas, u, part);
    const SplitItem it = a.splits[c];
    const int np = it.pieces;
    const bool many = np > kAtOnce;
    const int r = many ? part : part * kGroups + group;
    const float* first = a.ws + it.slot * kSlot;
    const float* later = a.ws + 2 * (int64_t)c * kSlot;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, l = 0.f;
    if (r < it.rows) {
      const int step = many ? kGroups : 1;
      for (int q0 = many ? group : 0; q0 < np; q0 += step * kAtOnce) {
        float2 ml[kAtOnce];
        float4 v[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          const int p = q0 + j * step;
          ml[j] = make_float2(-INFINITY, 0.f);
          v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (p < np) {
            const float* src = p ? later + 2 * p * kSlot : first;
            ml[j] = *reinterpret_cast<const float2*>(src + R * D + 2 * r);
            v[j] = *reinterpret_cast<const float4*>(src + r * D + d);
          }
        }
        float to = top;
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) to = fmaxf(to, ml[j].x);
        const float base = to == -INFINITY ? 0.f : to, back = exp2_approx(top - base);
        top = to;
        l *= back;
        x[0] *= back, x[1] *= back, x[2] *= back, x[3] *= back;
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          const float f = exp2_approx(ml[j].x - base);
          l += ml[j].y * f;
          x[0] += v[j].x * f, x[1] += v[j].y * f, x[2] += v[j].z * f, x[3] += v[j].w * f;
        }
      }
    }
    if (many) {  // (the same for every thread of the block)
      acc_s[group][threadIdx.x % kLanes] = make_float4(x[0], x[1], x[2], x[3]);
      if (d == 0) ml_s[group] = make_float2(top, l);
      __syncthreads();
      if (group == 0) {
        top = -INFINITY, l = 0.f;
        x[0] = x[1] = x[2] = x[3] = 0.f;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) top = fmaxf(top, ml_s[g].x);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const float f = exp2_approx(ml_s[g].x - base);
          const float4 v = acc_s[g][threadIdx.x];
          l += ml_s[g].y * f;
          x[0] += v.x * f, x[1] += v.y * f, x[2] += v.z * f, x[3] += v.w * f;
        }
      }
    }
    if (r < it.rows && (!many || group == 0)) {
      const int row = it.row0 + r, token = a.by_G(row);
      finish_row<D, F16, 4>(a, it.first + token, it.kvh * a.G + row - token * a.G, d, x, top, l);
    }
    if (many) __syncthreads();  // the next share's sums replace these
  }
}

template <int D, int R, bool F16>
cudaError_t launch_join(const PagedArgs& a, int ctas, cudaStream_t s) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(kJoinBlocksPerSm * ctas), 1, 1);
  cfg.blockDim = dim3(kJoinThreads, 1, 1);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<D, R, F16>, a, ctas);
}

}  // namespace

int read_paged_error(cudaStream_t stream) { return read_error_word(&g_paged_error, stream); }

namespace {

// Where the tables cover at most this many keys, an item is one CTA's work and
// no joining launch follows; half as many for mma.sync items that leave two
// CTAs or more for each (clusters take those). Lengths are on the device: the
// tables' width is what the host knows. Split and whole, us: 64 sequences of 500
// keys, 12 query heads on 2 KV heads of 128 dims 15.7 and 12.3; 1 sequence of
// 250 keys 8.8 and 7.2, of 500 8.8 and 10.1; 16 prompts of 500 tokens 45.8 and
// 37.8, 1 prompt of 200 16.8 and 13.7, of 500 18.5 and 17.2. More keys are split
// although even batches would still gain (64 sequences of 1000 keys: 20.9 and
// 18.1), for the sake of ragged ones, whose longest sequence would be the bound
// (64 of up to 1000 keys: 15.7 and 18.4; one of 1000 alone 8.9 and 15.9). A
// shared prefix, few long items of one length, is always split (500 keys under
// 64 sequences: 22.7 and 27.7). Wider tables cost the same batch the difference:
// 64 sequences of 500 keys under tables of 8192 take 15.6 us.
constexpr int kWholeKeys = 512;

// Where no more items of one row tile are in a batch than clusters of 16, 8, 4
// or 2 CTAs are resident at once, an item is the work of one cluster, the
// largest such, if the tables cover at most kWholeKeys for each of its CTAs and
// kClusterKeys in all: one launch, no pieces in memory. Dealt to all SMs and in
// clusters, us (12 query heads on 2 KV heads of 128 dims): one sequence of 641
// keys 8.7 and 6.6, of 4000 9.2 and 8.3; four of 1000 9.2 and 6.8, of 4000 10.9
// and 10.8; 16 of 450 10.3 and 6.7, of 2000 14.4 and 11.7; 32 of 900 14.2 and
// 11.6; ragged, 8 of up to 4000 10.7 and 10.7, 32 of up to 1000 11.7 and 10.6.
// Clusters of 16 only where the tables cover more than 8 units (one sequence of
// 1000 keys took 6.1 in a cluster of 8 and 6.7 of 16 when the rule was made).
constexpr int kClusterKeys = 4096;

template <int D, int NT, bool F16, bool kClusters>
cudaError_t configure(int dev) {
  static std::atomic<unsigned long long> configured{0};
  const unsigned long long bit = 1ull << (dev & 63);
  if (configured.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  auto kernel = paged_decode_kernel<D, NT, F16, kClusters>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)smem_of(D, NT, kClusters));
  if (e == cudaSuccess && kClusters) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) configured.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <int D, int NT, bool F16>
cudaError_t launch_decode(const CUtensorMap& k, const CUtensorMap& v, const PagedArgs& a, int ctas, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int64_t items = (int64_t)a.r.B * a.Hkv;
  if (a.one_tile && !a.unsplit && a.cap <= kClusterKeys && items * 2 <= ctas) {
    auto kernel = paged_decode_kernel<D, NT, F16, true>;
    cudaError_t e = configure<D, NT, F16, true>(dev);
    if (e != cudaSuccess) return e;
    static std::atomic<int> resident[4][64];  // clusters of 16, 8, 4 and 2 on a device, plus one
    cfg.dynamicSmemBytes = smem_of(D, NT, true);
    cfg.numAttrs = 2;
    for (int i = a.cap > 8 * kBlockKeys ? 0 : 1; i < 4; ++i) {
      const int C = 16 >> i;
      if (a.cap > C * kWholeKeys) break;
      attr[1].val.clusterDim.x = (unsigned)C;
      cfg.gridDim = dim3((unsigned)(items * C), 1, 1);
      int fit = resident[i][dev & 63].load(std::memory_order_relaxed) - 1;
      if (fit < 0) {
        e = cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg);
        if (e != cudaSuccess) {
          cudaGetLastError();
          fit = 0;
        }
        resident[i][dev & 63].store(fit + 1, std::memory_order_relaxed);
      }
      if (items <= fit) return cudaLaunchKernelEx(&cfg, kernel, k, v, a);
    }
    cfg.numAttrs = 1;
  }
  cudaError_t e = configure<D, NT, F16, false>(dev);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3((unsigned)ctas, 1, 1);
  cfg.dynamicSmemBytes = smem_of(D, NT, false);
  e = cudaLaunchKernelEx(&cfg, paged_decode_kernel<D, NT, F16, false>, k, v, a);
  return e != cudaSuccess || a.unsplit ? e : launch_join<D, 8 * NT, F16>(a, ctas, s);
}

template <int D, bool F16>
cudaError_t launch_rows(int nt, const CUtensorMap& k, const CUtensorMap& v, const PagedArgs& a, int ctas,
                        cudaStream_t s) {
  if (nt == 1) return launch_decode<D, 1, F16>(k, v, a, ctas, s);
  if (nt == 2) return launch_decode<D, 2, F16>(k, v, a, ctas, s);
  if (nt == 3) return launch_decode<D, 3, F16>(k, v, a, ctas, s);
  return launch_decode<D, 4, F16>(k, v, a, ctas, s);
}

cudaError_t launch_kernel(int D, bool f16, int nt, const CUtensorMap& k, const CUtensorMap& v, const PagedArgs& a,
                          int ctas, cudaStream_t s) {
  if (D == 128) return f16 ? launch_rows<128, true>(nt, k, v, a, ctas, s) : launch_rows<128, false>(nt, k, v, a, ctas, s);
  return f16 ? launch_rows<64, true>(nt, k, v, a, ctas, s) : launch_rows<64, false>(nt, k, v, a, ctas, s);
}

// Whether a batch of up to `tokens` per sequence goes to the tcgen05 kernel (its
// tiles hold whole tokens, and its row maxima want a scale that is not
// negative): by the rows of a sequence and KV head. Beyond 32 mma.sync would
// take several tiles and read the keys for each (48 rows over 1000 keys of a
// shared prefix 30.7 us by mma.sync, 24.4 by tcgen05, both with the suffix's
// launches of then); with 128 dims its tile of 32 rows does not fit the 168
// registers that a thread of nine warps can have (592 bytes are spilled, 176 of
// a tile of 24). mma.sync and tcgen05, us, 64 sequences of 2000 keys, 2 KV heads
// of 128 dims: 24 rows 49.0 and 49.9, 28 rows 88.6 and 50.2, 32 rows 88.6 and
// 48.6 (one sequence of 300 keys: 9.6 and 13.8, 13.4 and 13.8, 13.5 and 13.4);
// of 64 dims: 24 rows 28.9 and 39.5, 32 rows 31.9 and 39.2.
int64_t tc_from(int D) { return D == 128 ? 25 : 33; }
bool takes_tc(int64_t tokens, int64_t G, int D, float scale) {
  return tokens * G >= tc_from(D) && G <= 128 && scale >= 0.f;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
// Room for the pieces of a launch over `tokens` per sequence, and what the runs note of their split items.
size_t pieces_bytes(int64_t tokens, int64_t G, int D, int ctas) {
  const size_t rows = takes_tc(tokens, G, D, 1.f) ? kTcRows : 32;
  return round256((size_t)ctas * (2 * rows * (D + 2) * sizeof(float) + sizeof(SplitItem)));
}
size_t state_bytes(int64_t T, int64_t Hq, int D) { return (size_t)(T * Hq) * (D + 2) * sizeof(float); }
size_t workspace_bytes_for(int64_t T, int64_t Hq, int64_t Hkv, int D, int64_t most, bool prefix, int ctas) {
  return pieces_bytes(most, Hq / Hkv, D, ctas) +
         (prefix ? pieces_bytes(T, Hq / Hkv, D, ctas) + state_bytes(T, Hq, D) : 0);
}

struct Call {
  const qi4_paged_kv* kv;
  const void* q;
  int64_t q_tok, q_head;
  void* out;
  int64_t T, B, Hq;
  const int32_t* cu;
  const int32_t* lengths;
  int64_t max_tokens;
  float scale;
  int causal;
  const int32_t* prefix_table;
  int64_t prefix_width, prefix_len;
  void* ws;
  size_t ws_bytes;
  cudaStream_t stream;
};

int attend(const Call& c, const char* what) {
  clear_error();
  int rc = check_paged_kv(c.kv, what);
  if (rc) return rc;
  const qi4_paged_kv& kv = *c.kv;
  if (c.T < 0 || c.B <= 0 || c.T > (1ll << 30) || c.B > (1ll << 30) || c.Hq <= 0 || c.Hq > 65535 || c.max_tokens < 0) {
    set_error("%s: B and Hq must be positive, T and max_tokens not negative", what);
    return QI4_ERR_ARGUMENT;
  }
  if (c.T == 0) return QI4_OK;
  if (!c.q || !c.out || !c.lengths) {
    set_error("%s: q, out and lengths must be non-null", what);
    return QI4_ERR_ARGUMENT;
  }
  if (!c.cu && c.T % c.B) {
    set_error("%s: without cu_tokens every sequence has T / B tokens (got T = %lld, B = %lld)", what, (long long)c.T,
              (long long)c.B);
    return QI4_ERR_SHAPE;
  }
  if ((kv.head_dim != 64 && kv.head_dim != 128) || c.Hq % kv.kv_heads) {
    set_error("%s supports head_dim 64 and 128 and query heads that are a multiple of the KV heads (got %d, %lld/%d)",
              what, kv.head_dim, (long long)c.Hq, kv.kv_heads);
    return QI4_ERR_SHAPE;
  }
  if (c.T * c.Hq >= (1ll << 31)) {
    set_error("%s: at most 2^31 rows (tokens x query heads)", what);
    return QI4_ERR_SHAPE;
  }
  auto al = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!al(c.q, 16) || !al(c.out, 32) || c.q_tok % 8 || c.q_head % 8 || c.q_tok < (c.T > 1) || c.q_head < (c.Hq > 1)) {
    set_error("%s: q must be 16-byte and out 32-byte aligned, q with positive strides that are multiples of 8 elements",
              what);
    return QI4_ERR_ALIGNMENT;
  }
  const bool prefix = c.prefix_len > 0;
  if (c.prefix_len < 0 || (prefix && (!c.prefix_table || c.prefix_width <= 0))) {
    set_error("%s: a prefix needs its page table and a length that is not negative", what);
    return QI4_ERR_ARGUMENT;
  }
  if (c.prefix_len > (1ll << 30)) {
    set_error("%s: a prefix has at most 2^30 keys (got %lld)", what, (long long)c.prefix_len);
    return QI4_ERR_SHAPE;
  }
  const int64_t prefix_pages = (c.prefix_len + kv.page_size - 1) / kv.page_size;  // of the table, those that are read
  if (prefix && prefix_pages > c.prefix_width) {
    set_error("%s: the prefix is longer (%lld) than its page table covers", what, (long long)c.prefix_len);
    return QI4_ERR_SHAPE;
  }
  const int D = kv.head_dim;
  const int64_t G = c.Hq / kv.kv_heads;
  // Tokens of a sequence at most, as far as the host knows.
  const int64_t most = c.cu ? (c.max_tokens ? std::min(c.max_tokens, c.T) : c.T) : c.T / c.B;
  // Units are counted in 32 bits (paged_attention.cuh): tiles of the batch times units of the longest item.
  {
    auto units = [&](int64_t tokens, int64_t seqs, int64_t per_seq, int64_t keys) {
      const int64_t rows = takes_tc(per_seq, G, D, c.scale) ? kTcRows / 2 : 8;
      return (double)(tokens * G / rows + seqs) * kv.kv_heads * (keys / kBlockKeys + 2);
    };
    if (units(c.T, c.B, most, (int64_t)kv.table_width * kv.page_size) >= 2147483647.0 ||
        (prefix && units(c.T, 1, c.T, c.prefix_len) >= 2147483647.0)) {
      set_error("%s: %lld tokens of %lld sequences over up to %lld keys are too many for one call", what,
                (long long)c.T, (long long)c.B, (long long)kv.table_width * kv.page_size);
      return QI4_ERR_SHAPE;
    }
  }
  int sms = 0;
  rc = require_device(&sms);
  if (rc) return rc;
  if (sms > kMaxCtas) sms = kMaxCtas;  // (CTAs of a launch; a B200 has 148)
  const size_t need = workspace_bytes_for(c.T, c.Hq, kv.kv_heads, D, most, prefix, sms);
  char* ws = static_cast<char*>(c.ws);
  if (ws && (c.ws_bytes < need || !al(ws, 16))) {
    set_error("%s: the workspace needs %zu bytes, 16-byte aligned (got %zu)", what, need, c.ws_bytes);
    return QI4_ERR_ARGUMENT;
  }
  CUtensorMap qmap, kmap, vmap;
  const uint32_t box_rows = (uint32_t)std::min(kv.page_size, kBlockKeys);
  if (!tensor_map_pages(&kmap, kv.k, kv, box_rows) || !tensor_map_pages(&vmap, kv.v, kv, box_rows)) return QI4_ERR_LAUNCH;
  if (takes_tc(prefix ? c.T : most, G, D, c.scale) &&
      !tensor_map_rows3(&qmap, c.q, kv.dtype == QI4_DTYPE_F16, D, c.Hq, c.T, c.q_head, c.q_tok, (uint32_t)G,
                        (uint32_t)(kTcRows / G)))
    return QI4_ERR_LAUNCH;
  void* own = nullptr;
  if (!ws) {
    if (scratch_alloc(&own, need, c.stream) != cudaSuccess) {
      cudaGetLastError();
      set_error("%s: cannot allocate %zu bytes of scratch", what, need);
      return QI4_ERR_LAUNCH;
    }
    ws = static_cast<char*>(own);
  }
  PagedArgs a = {};
  a.q = static_cast<const uint16_t*>(c.q);
  a.q_tok = c.q_tok, a.q_head = c.q_head;
  a.out = static_cast<uint16_t*>(c.out);
  a.page_shift = __builtin_ctz((unsigned)kv.page_size), a.box_shift = __builtin_ctz(box_rows);
  a.pages = kv.pages;
  a.v = static_cast<const uint16_t*>(kv.v);
  a.v_page = kv.page_stride, a.v_head = kv.head_stride, a.v_slot = kv.slot_stride;
  a.Hkv = kv.kv_heads, a.G = (int)(c.Hq / kv.kv_heads);
  a.scale_log2 = c.scale * 1.4426950408889634f;
  const bool f16 = kv.dtype == QI4_DTYPE_F16;
  cudaError_t e = cudaSuccess;
  // One launch: pieces at `at`, the kernel for `tokens` per sequence. The
  // mma.sync tile is the smallest of 8, 16, 24 and 32 rows that holds them (the
  // 20 rows of each of 24 ragged sequences of up to 6005 keys, 64 dims: 36.4 us in tiles of 24, 44.6 in tiles of 32
  // before the look at odd values, 38.1 in tiles of 24 now).
  auto launch = [&](PagedArgs& x, char* at, int64_t tokens) {
    const bool tc = takes_tc(tokens, G, D, c.scale);
    const size_t rows = takes_tc(tokens, G, D, 1.f) ? kTcRows : 32;
    x.ws = reinterpret_cast<float*>(at);
    const int R = tc ? kTcRows : tokens * G <= 8 ? 8 : tokens * G <= 16 ? 16 : tokens * G <= 24 ? 24 : 32;
    x.tile_tokens = (int)(R / G);
    x.tile_rows = G <= R ? x.tile_tokens * (int)G : R;
    x.one_tile = tokens * G <= x.tile_rows;
    x.by_tile_rows = FastDiv::of(x.tile_rows);
    x.by_G = FastDiv::of(G);
    x.by_ctas = FastDiv::of(sms);
    x.unsplit = !x.late && x.cap <= (tc || (int64_t)x.r.B * x.Hkv * 2 > sms ? kWholeKeys : kWholeKeys / 2);
    x.splits = reinterpret_cast<SplitItem*>(at + (size_t)sms * 2 * rows * (D + 2) * sizeof(float));
    if (tc) return launch_paged_tc(D, f16, qmap, kmap, vmap, x, sms, c.stream);
    return launch_kernel(D, f16, R / 8, kmap, vmap, x, sms, c.stream);
  };
  a.table = kv.block_table, a.table_stride = kv.table_stride, a.table_width = kv.table_width;
  a.r = {c.cu, c.lengths, (int)c.B, (int)c.T, (int)(c.T / c.B)};
  a.fixed_len = -1, a.cap = kv.table_width * kv.page_size, a.causal = c.causal;
  if (prefix) {
    // First each sequence's own keys, into a state per row; then all tokens as
    // one sequence over the prefix, each row seeing all of it and taking up its
    // state at the end (so the second launch need not wait for the first).
    char* at = ws + pieces_bytes(most, G, D, sms);
    float* state = reinterpret_cast<float*>(at + pieces_bytes(c.T, G, D, sms));
    a.state_acc = state, a.state_ml = state + c.T * c.Hq * D;
    e = launch(a, ws, most);
    PagedArgs p = a;
    p.table = c.prefix_table, p.table_stride = 0, p.table_width = (int)prefix_pages;
    p.r = {nullptr, nullptr, 1, (int)c.T, (int)c.T};
    p.fixed_len = (int)c.prefix_len, p.cap = (int)c.prefix_len, p.causal = 0;
    p.prior_acc = a.state_acc, p.prior_ml = a.state_ml, p.late = 1;
    p.state_acc = p.state_ml = nullptr;
    if (e == cudaSuccess) e = launch(p, at, c.T);
  } else {
    e = launch(a, ws, most);
  }
  if (own) scratch_free(own, c.stream);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("%s launch failed: %s", what, cudaGetErrorString(e));
    return QI4_ERR_LAUNCH;
  }
  return QI4_OK;
}

}  // namespace
}  // namespace qi4

extern "C" QI4_API int qi4_paged_attention(const qi4_paged_kv* kv, const void* q, int64_t q_token_stride,
                                           int64_t q_head_stride, void* out, int64_t T, int64_t B, int64_t Hq,
                                           const int32_t* cu_tokens, const int32_t* lengths, int64_t max_tokens,
                                           float scale, int causal, void* workspace, size_t workspace_bytes,
                                           void* stream) {
  return qi4::attend({kv, q, q_token_stride, q_head_stride, out, T, B, Hq, cu_tokens, lengths, max_tokens, scale,
                      causal ? 1 : 0, nullptr, 0, 0, workspace, workspace_bytes, static_cast<cudaStream_t>(stream)},
                     "paged attention");
}

extern "C" QI4_API int qi4_shared_prefix_attention(const qi4_paged_kv* kv, const void* q, int64_t q_token_stride,
                                                   int64_t q_head_stride, void* out, int64_t T, int64_t B, int64_t Hq,
                                                   const int32_t* prefix_table, int64_t prefix_pages,
                                                   int64_t prefix_length, const int32_t* cu_tokens,
                                                   const int32_t* lengths, int64_t max_tokens, float scale,
                                                   void* workspace, size_t workspace_bytes, void* stream) {
  return qi4::attend({kv, q, q_token_stride, q_head_stride, out, T, B, Hq, cu_tokens, lengths, max_tokens, scale, 1,
                      prefix_table, prefix_pages, prefix_length, workspace, workspace_bytes,
                      static_cast<cudaStream_t>(stream)},
                     "shared-prefix attention");
}

extern "C" QI4_API size_t qi4_paged_attention_workspace(int64_t T, int64_t Hq, int64_t kv_heads, int head_dim,
                                                        int64_t max_tokens, int prefix) {
  if (T < 0 || Hq <= 0 || kv_heads <= 0 || Hq % kv_heads || head_dim <= 0 || max_tokens < 0) return 0;
  int sms = 0;
  if (qi4::require_device(&sms)) return 0;
  sms = std::min(sms, qi4::kMaxCtas);
  return qi4::workspace_bytes_for(T, Hq, kv_heads, head_dim, max_tokens ? std::min(max_tokens, T) : T, prefix != 0, sms);
}
