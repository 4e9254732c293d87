// Verification of drafted tokens against the target's probabilities (sm_100a).
//
// Per sequence, with drafted tokens t_0 .. t_{n-1}, the draft's and the
// target's distributions q_i, p_i and uniform numbers u_0 .. u_K in [0, 1):
// draft i stands while u_i q_i(t_i) < p_i(t_i) and every draft before it
// stands. With a drafts standing, the token after them is drawn at u_K (the
// number that no draft is tested against: that of a refused draft is not
// uniform any more) from the weights
//   max(p_a - q_a, 0)   (a draft was refused), or   p_a   (none was),
// so that the tokens are distributed as the target's own. The weights count in
// whole units of 2^-40 (truncated; a weight above 1 counts as 1) and are
// summed as 64-bit integers: the drawn token, the first v whose running sum
// exceeds floor(u_K 2^24) / 2^24 of the total, does not depend on the order of
// the sums. Where no weight is left (p <= q throughout, after rounding) the
// token is drawn from p_a; where p_a has none either it is -1.
//
// Bound by one pass over two vocabulary rows. One cluster of 8 or 16 CTAs per
// sequence: each finds `a` for itself (the drafts side by side in one warp),
// sums its share of the vocabulary, a contiguous stretch per warp, one sum
// for every step of the warp's loads; the sums are exchanged over distributed
// shared memory, and the one warp whose stretch holds the drawn share finds the
// step among its sums and reads that step again (from L2) for the token.
// Measured (device time, 151,936 tokens, FP32): one sequence of 4 drafts 6.1 us,
// all of it latency; 64 of up to 5 drafts 16.0 us, 8.1 of them the rows' bytes.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "paged.cuh"

namespace qi4 {

__device__ int g_verify_error;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxVocab = 1 << 21;
constexpr int kMaxSteps = kMaxVocab / (8 * kWarps) / 128;  // steps of a warp at most (of 128 elements at least)

struct VerifyArgs {
  const int64_t* tokens;  // [B, K]
  const void* target;     // [B, K + 1, V] at the given strides
  const void* draft;      // [B, K, V], or null: each draft was certain (q = 1 at its token)
  int64_t t_batch, t_pos, d_batch, d_pos;
  const float* uniforms;  // [B, K + 1]
  const int32_t* counts;  // [B], or null: K each
  int64_t* out;           // [B, K + 1]
  int32_t* accepted;      // [B]
  int K, V;
};

template <int T>
struct Elem;
template <>
struct Elem<QI4_DTYPE_F32> {
  using type = float;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ void split(uint4 w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
  }
};
template <>
struct Elem<QI4_DTYPE_BF16> {
  using type = uint16_t;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
  static __device__ __forceinline__ void split(uint4 w, float (&x)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(a[i] << 16);
      x[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Elem<QI4_DTYPE_F16> {
  using type = uint16_t;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(uint16_t x) { return __half2float(__ushort_as_half(x)); }
  static __device__ __forceinline__ void split(uint4 w, float (&x)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};

// The weights of one position of a sequence.
template <int T>
struct Weights {
  using E = typename Elem<T>::type;
  static constexpr int kVec = Elem<T>::kVec;
  const E* p;
  const E* q;   // null: only `skip` is taken out
  int skip;     // a vocabulary index of weight zero, or -1
  bool vec;     // rows 16-byte aligned

  static __device__ __forceinline__ long long units(float w) {
    return __float2ll_rz(fminf(fmaxf(w, 0.f), 1.f) * 1099511627776.f);  // 2^40; a NaN counts as nothing
  }
  // Elements v .. v + kVec - 1 in units, those from `end` on without weight.
  __device__ __forceinline__ long long load(int v, int end, long long (&n)[kVec]) const {
    float x[kVec], y[kVec];
    long long sum = 0;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      x[i] = y[i] = 0.f;
      if (v + i < end) {
        x[i] = Elem<T>::get(__ldg(p + v + i));
        if (q) y[i] = Elem<T>::get(__ldg(q + v + i));
      }
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) sum += n[i] = v + i == skip ? 0 : units(x[i] - y[i]);
    return sum;
  }
  // The sums of kAtOnce whole steps from v on, all their loads at once.
  template <int kAtOnce>
  __device__ __forceinline__ void load_whole(int v, long long (&sum)[kAtOnce]) const {
    uint4 a[kAtOnce], b[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) a[j] = __ldg(reinterpret_cast<const uint4*>(p + v + j * 32 * kVec));
    if (q) {
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) b[j] = __ldg(reinterpret_cast<const uint4*>(q + v + j * 32 * kVec));
    } else {
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) b[j] = make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      float x[kVec], y[kVec];
      Elem<T>::split(a[j], x);
      Elem<T>::split(b[j], y);
      sum[j] = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) sum[j] += v + j * 32 * kVec + i == skip ? 0 : units(x[i] - y[i]);
    }
  }
};

// Sums over the lanes up to each.
__device__ __forceinline__ long long scan(long long x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

template <int T, int kCluster>
__global__ void __launch_bounds__(kThreads) verify_kernel(const VerifyArgs a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  using W = Weights<T>;
  using E = typename W::E;
  constexpr int kStep = 32 * W::kVec;
  __shared__ int accepted_s, refused_s;
  __shared__ long long warp_sum[kWarps];
  __shared__ long long step_sum[kWarps][kMaxSteps];
  __shared__ long long cta_sum[2];  // by attempt
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / kCluster, rank = blockIdx.x % kCluster;
  pdl_wait();
  pdl_launch_dependents();

  const E* target = static_cast<const E*>(a.target) + b * a.t_batch;
  const E* draft = a.draft ? static_cast<const E*>(a.draft) + b * a.d_batch : nullptr;
  const float* u = a.uniforms + (int64_t)b * (a.K + 1);
  const int64_t* tokens = a.tokens + (int64_t)b * a.K;
  if (warp == 0) {
    const int n = a.counts ? max(0, min(__ldg(a.counts + b), a.K)) : a.K;
    int stand = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      bool ok = false;
      if (i < n) {
        const int64_t t = __ldg(tokens + i);
        if (t >= 0 && t < a.V) {
          const float p = Elem<T>::get(__ldg(target + i * a.t_pos + t));
          const float q = draft ? Elem<T>::get(__ldg(draft + i * a.d_pos + t)) : 1.f;
          ok = __ldg(u + i) * q < p;
        } else {
          atomicOr(&g_verify_error, QI4_DEVICE_BAD_TOKEN);  // never stands
        }
      }
      const int run = __ffs(~__ballot_sync(0xffffffffu, ok)) - 1;  // -1: all 32 stand
      stand += run < 0 ? 32 : run;
      if (run >= 0) break;
    }
    if (lane == 0) {
      accepted_s = stand;
      refused_s = stand < n;
    }
  }
  __syncthreads();
  const int acc = accepted_s;
  const bool refused = refused_s != 0;

  // This warp's stretch of the vocabulary (whole steps of the warp's loads).
  const int stretch = ((a.V + kCluster * kWarps - 1) / (kCluster * kWarps) + kStep - 1) / kStep * kStep;
  const int v0 = min(a.V, (rank * kWarps + warp) * stretch), v1 = min(a.V, v0 + stretch);
  W w;
  w.p = target + acc * a.t_pos;
  w.q = refused && draft ? draft + acc * a.d_pos : nullptr;
  w.skip = refused && !draft ? (int)min(max(__ldg(tokens + acc), (int64_t)-1), (int64_t)a.V) : -1;
  w.vec = ((reinterpret_cast<uintptr_t>(w.p) | reinterpret_cast<uintptr_t>(w.q)) & 15) == 0;

  long long token = -1;
  for (int attempt = 0; attempt < 2; ++attempt) {
    long long sum = 0;
    // A step's sum over the warp: below 32 x kVec x 2^40, so that its halves' sums fit 32 bits.
    auto keep = [&](long long here, int step) {
      const long long all = (long long)__reduce_add_sync(0xffffffffu, (unsigned)(here & 0xFFFFFF)) +
                            ((long long)__reduce_add_sync(0xffffffffu, (unsigned)(here >> 24)) << 24);
      if (lane == 0) step_sum[warp][step] = all;
      sum += all;
    };
    constexpr int kAtOnce = 4;
    int step = 0;
    if (w.vec)
      for (; v0 + (step + kAtOnce) * kStep <= v1; step += kAtOnce) {
        long long here[kAtOnce];
        w.template load_whole<kAtOnce>(v0 + step * kStep + lane * W::kVec, here);
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) keep(here[j], step + j);
      }
    if (w.vec)
      for (; v0 + (step + 1) * kStep <= v1; ++step) {
        long long here[1];
        w.template load_whole<1>(v0 + step * kStep + lane * W::kVec, here);
        keep(here[0], step);
      }
#pragma unroll 2
    for (; v0 + step * kStep < v1; ++step) {
      long long n[W::kVec];
      keep(w.load(v0 + step * kStep + lane * W::kVec, v1, n), step);
    }
    const int steps = step;
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      long long s = 0;
      for (int i = 0; i < kWarps; ++i) s += warp_sum[i];
      cta_sum[attempt] = s;
    }
    cluster.sync();
    const long long theirs = lane < kCluster ? *cluster.map_shared_rank(&cta_sum[attempt], lane) : 0,
                    incl = scan(theirs, lane);
    const long long total = __shfl_sync(0xffffffffu, incl, 31);
    const long long share = (long long)fminf(fmaxf(__ldg(u + a.K) * 16777216.f, 0.f), 16777215.f);
    const long long goal = share * (total >> 24) + ((share * (total & 0xFFFFFF)) >> 24);
    const long long before = __shfl_sync(0xffffffffu, incl - theirs, rank);
    const long long own = __shfl_sync(0xffffffffu, theirs, rank);
    if (total == 0 && attempt == 0 && (w.q || w.skip >= 0)) {  // uniform over the cluster
      w.q = nullptr;
      w.skip = -1;
      w.vec = (reinterpret_cast<uintptr_t>(w.p) & 15) == 0;
      continue;
    }
    const bool mine = total > 0 && goal >= before && goal < before + own;
    if (mine || (total == 0 && rank == 0)) {
      // The CTA that holds the drawn share: its warp that does scans its stretch again.
      long long at = before;
      int holder = total == 0 ? 0 : -1;
      for (int i = 0; i < kWarps && holder < 0; ++i) {
        if (goal < at + warp_sum[i])
          holder = i;
        else
          at += warp_sum[i];
      }
      if (warp == holder) {
        if (total > 0) {
          // The step that holds the share, 32 sums at a time, then the element.
          for (int j0 = 0; j0 < steps && token < 0; j0 += 32) {
            const long long mine_sum = j0 + lane < steps ? step_sum[warp][j0 + lane] : 0;
            const long long upto = scan(mine_sum, lane);
            const unsigned in = __ballot_sync(0xffffffffu, goal < at + upto);
            if (!in) {
              at += __shfl_sync(0xffffffffu, upto, 31);
              continue;
            }
            const int j = __ffs(in) - 1, v = v0 + (j0 + j) * kStep + lane * W::kVec;
            at += __shfl_sync(0xffffffffu, upto - mine_sum, j);
            long long n[W::kVec];
            const long long here = w.load(v, v1, n), run = scan(here, lane);
            const unsigned hit = __ballot_sync(0xffffffffu, goal < at + run);
            long long s = at + run - here;
            int k = 0;
#pragma unroll
            for (int i = 0; i < W::kVec - 1; ++i)
              if (k == i && s + n[i] <= goal) {
                s += n[i];
                ++k;
              }
            token = __shfl_sync(0xffffffffu, v + k, __ffs(hit) - 1);
          }
        }
        int64_t* out = a.out + (int64_t)b * (a.K + 1);
        for (int i = lane; i <= a.K; i += 32) out[i] = i < acc ? __ldg(tokens + i) : i == acc ? token : -1;
        if (lane == 0) a.accepted[b] = acc;
      }
    }
    break;
  }
  cluster.sync();  // no CTA leaves while another may read its sum
}

template <int T, int kCluster>
cudaError_t launch_clusters(const VerifyArgs& a, int B, cudaStream_t stream) {
  auto kernel = verify_kernel<T, kCluster>;
  if constexpr (kCluster > 8) {
    static std::atomic<unsigned long long> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(configured.load(std::memory_order_relaxed) & bit)) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return e;
      configured.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * kCluster), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// Clusters of 16 while the CTAs are at most two per SM (a sequence's time is
// then the serial path of one: 6.1 us against 7.3 in clusters of 8 for one
// sequence of 151,936 tokens), else of 8 (64 sequences: 15.9 us against 22.5).
template <int T>
cudaError_t launch_verify(const VerifyArgs& a, int B, int sms, cudaStream_t stream) {
  return (int64_t)B * 16 <= 2 * sms ? launch_clusters<T, 16>(a, B, stream) : launch_clusters<T, 8>(a, B, stream);
}

}  // namespace

int read_verify_error(cudaStream_t stream) { return read_error_word(&g_verify_error, stream); }

}  // namespace qi4

extern "C" QI4_API int qi4_verify_draft(const int64_t* draft_tokens, const void* target_probs,
                                        int64_t target_batch_stride, int64_t target_pos_stride,
                                        const void* draft_probs, int64_t draft_batch_stride, int64_t draft_pos_stride,
                                        int dtype, const float* uniforms, const int32_t* draft_counts, int64_t B,
                                        int64_t K, int64_t V, int64_t* out_tokens, int32_t* accepted, void* stream) {
  using namespace qi4;
  clear_error();
  if (!target_probs || !uniforms || !out_tokens || !accepted || (K > 0 && !draft_tokens)) {
    set_error("draft verification: draft_tokens, target_probs, uniforms and the outputs must be non-null");
    return QI4_ERR_ARGUMENT;
  }
  if (dtype != QI4_DTYPE_F32 && dtype != QI4_DTYPE_BF16 && dtype != QI4_DTYPE_F16) {
    set_error("draft verification takes FP32, BF16 or FP16 probabilities");
    return QI4_ERR_DTYPE;
  }
  if (B <= 0 || K < 0 || V <= 0 || B > (1 << 26) || K > 4096 || V > kMaxVocab) {
    set_error("draft verification: B and V must be positive, K not negative (B <= 2^26, K <= 4096, V <= 2^21; got "
              "%lld, %lld, %lld)", (long long)B, (long long)K, (long long)V);
    return QI4_ERR_SHAPE;
  }
  if (target_batch_stride < 0 || target_pos_stride < 0 || draft_batch_stride < 0 || draft_pos_stride < 0) {
    set_error("draft verification: strides must not be negative");
    return QI4_ERR_ARGUMENT;
  }
  int sms = 0;
  const int rc = require_device(&sms);
  if (rc) return rc;
  VerifyArgs a = {draft_tokens, target_probs, draft_probs, target_batch_stride, target_pos_stride,
                  draft_batch_stride, draft_pos_stride, uniforms, draft_counts, out_tokens, accepted, (int)K, (int)V};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == QI4_DTYPE_F32    ? launch_verify<QI4_DTYPE_F32>(a, (int)B, sms, s)
                        : dtype == QI4_DTYPE_BF16 ? launch_verify<QI4_DTYPE_BF16>(a, (int)B, sms, s)
                                                  : launch_verify<QI4_DTYPE_F16>(a, (int)B, sms, s);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("draft verification launch failed: %s", cudaGetErrorString(e));
    return QI4_ERR_LAUNCH;
  }
  return QI4_OK;
}
