// Verification of sampled draft chains by rejection, sm_100a.
//
// Request r drafted x_1 .. x_n, x_d drawn from q_d. With the target's probabilities p_1 .. p_{n+1} and given coins u:
//   x_d is kept  <=>  u_d q_d(x_d) < p_d(x_d)                       (the first one that is not ends the chain)
//   bonus: the first one that is not kept is replaced by a draw from max(p_d - q_d, 0); if all are kept, a draw from
//   p_{n+1}. A draw takes the first index whose cumulative mass exceeds coin * total. Drafts without probabilities
//   (greedy drafts) have q = 1 at their token. The emitted tokens then follow p exactly.
// Products of two fp32 values and differences of probabilities are exact in fp64 and masses are summed in fp64, so the
// result does not depend on how the row is split over threads (up to a coin within 1e-15 of a border). Probabilities
// that are NaN, and residuals that are, count as 0.
//
// Only one row of p (and of q) per request is read in full, which one is known after the chain's few values.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include "common.cuh"

namespace phx {

namespace {

constexpr int kSvThreads = 256;
constexpr int kSvWarps = kSvThreads / 32;
constexpr int kSvResident = 3;          // CTAs per SM: 85 registers a thread, 16 loads of 16 bytes in flight without spills

struct SvArgs {
  const void *p, *q;              // q null: greedy drafts
  const int64_t* tokens;          // [R, D]
  const float* coins;             // [R, D + 2]
  const int* n_draft;             // [R] or null
  int64_t *acc, *bonus;
  int64_t p_r, p_d, q_r, q_d;     // strides of the requests and of the drafts (elements)
  int D, V;
};

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}

// weight of index i: max(p - q, 0); NaN gives 0
__device__ __forceinline__ double weight(float p, float q) { return p > q ? (double)p - (double)q : 0.0; }

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Accepted drafts of request r (warp-wide; every lane gets the count).
template <typename T>
__device__ __forceinline__ int accepted(const SvArgs& a, int r, int n, int lane) {
  int kept = 0;
  for (int d0 = 0; d0 < n; d0 += 32) {
    const int d = d0 + lane;
    bool ok = false;
    if (d < n) {
      const int64_t x = a.tokens[(int64_t)r * a.D + d];
      if (x >= 0 && x < a.V) {      // a token outside the vocabulary is never kept
        const float px = to_f(static_cast<const T*>(a.p)[r * a.p_r + d * a.p_d + x]);
        const float qx = a.q ? to_f(static_cast<const T*>(a.q)[r * a.q_r + d * a.q_d + x]) : 1.f;
        ok = (double)a.coins[(int64_t)r * (a.D + 2) + d] * (double)qx < (double)px;
      }
    }
    const unsigned m = __ballot_sync(0xffffffffu, ok);
    if (m != 0xffffffffu) return kept + __ffs(~m) - 1;
    kept += 32;
  }
  return min(kept, n);
}

// 16 bytes of a row from element i on, zeros past its end: one load where the row is 16-byte aligned, else element by
// element.
template <typename T>
__device__ __forceinline__ uint4 load16(const T* row, int i, int V, bool aligned) {
  constexpr int VEC = 16 / sizeof(T);
  if (aligned && i + VEC <= V) return *reinterpret_cast<const uint4*>(row + i);
  using Bits = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
  uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const uint32_t x = i + e < V ? reinterpret_cast<const Bits*>(row)[i + e] : 0;
    u[e * sizeof(T) / 4] |= x << (8 * (e * sizeof(T) % 4));
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
template <typename T, int E>
__device__ __forceinline__ float pick(const uint4& u) {      // element E of 16 bytes
  const uint32_t w = (E * sizeof(T) / 4) == 0 ? u.x : (E * sizeof(T) / 4) == 1 ? u.y : (E * sizeof(T) / 4) == 2 ? u.z : u.w;
  if constexpr (sizeof(T) == 4) return __uint_as_float(w);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)(w >> (16 * (E & 1)))));
  else return __uint_as_float((E & 1) ? w & 0xffff0000u : w << 16);
}

constexpr int kSteps = 4;               // 16-byte loads of a row a lane has in flight
constexpr int kMaxBlocks = 1024;        // block masses a CTA keeps
constexpr int kMaxCluster = 8;

// A cluster of CTAs (the grid's x) per request. The row is cut into blocks of kSteps x 32 lanes x 16 bytes, `span` times
// that for rows too long for the table of masses; a CTA takes `blocks` neighbouring ones, a warp every 8th of them. The
// CTAs exchange their masses through shared memory; the one in which the draw falls finds the block in its table and
// reads that block again, in order. So the row is read once.
// Bound: HBM for a full batch on a large vocabulary; else latency (chain values, row, cluster barrier, one block).
// Measured: see launch().
template <typename T>
__global__ void __launch_bounds__(kSvThreads, kSvResident) spec_verify_kernel(const SvArgs a, int blocks, int span) {
  constexpr int VEC = 16 / sizeof(T), kStep = 32 * VEC;
  __shared__ double mass[kMaxBlocks];
  __shared__ double totals[2][kMaxCluster];
  __shared__ int s_kept;
  const int cl = gridDim.x, rank = blockIdx.x, r = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (cl > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const int n = a.n_draft ? max(0, min(a.D, a.n_draft[r])) : a.D;
  if (warp == 0) {
    const int k = accepted<T>(a, r, n, lane);
    if (lane == 0) s_kept = k;
    if (rank == 0)
      for (int d = lane; d < a.D; d += 32) a.acc[(int64_t)r * a.D + d] = d < k ? d + 1 : -1;
  }
  __syncthreads();
  // every CTA of the cluster has started: its shared memory may be written
  if (cl > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int kept = s_kept;
  const T* p = static_cast<const T*>(a.p) + r * a.p_r + kept * a.p_d;
  const T* q = a.q && kept < n ? static_cast<const T*>(a.q) + r * a.q_r + kept * a.q_d : nullptr;
  int cut = -1;                           // greedy draft that was not kept: its token is taken out
  if (!a.q && kept < n) {
    const int64_t x = a.tokens[(int64_t)r * a.D + kept];
    cut = x >= 0 && x < a.V ? (int)x : -1;
  }
  const bool p16 = (reinterpret_cast<uintptr_t>(p) & 15) == 0, q16 = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  const int64_t start = (int64_t)rank * blocks * span * kSteps * kStep;      // this CTA's first element
  const int nb = (int)min((int64_t)blocks, max((int64_t)0, (a.V - start + span * kSteps * kStep - 1) / (span * kSteps * kStep)));
  // 16 bytes of each row for each of kSteps steps from element i0 on, and the weights of one step
  auto load = [&](int64_t i0, uint4 (&x)[kSteps], uint4 (&y)[kSteps]) {
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      const int i = (int)min(i0 + u * kStep + lane * VEC, (int64_t)a.V);
      x[u] = load16<T>(p, i, a.V, p16);
      y[u] = q ? load16<T>(q, i, a.V, q16) : make_uint4(0, 0, 0, 0);
    }
  };
  auto weights = [&](int64_t i0, int u, const uint4& x, const uint4& y, double (&w)[VEC]) {
    const int64_t i = i0 + u * kStep + lane * VEC;
    w[0] = weight(pick<T, 0>(x), pick<T, 0>(y)), w[1] = weight(pick<T, 1>(x), pick<T, 1>(y));
    w[2] = weight(pick<T, 2>(x), pick<T, 2>(y)), w[3] = weight(pick<T, 3>(x), pick<T, 3>(y));
    if constexpr (VEC == 8) {
      w[4] = weight(pick<T, 4>(x), pick<T, 4>(y)), w[5] = weight(pick<T, 5>(x), pick<T, 5>(y));
      w[6] = weight(pick<T, 6>(x), pick<T, 6>(y)), w[7] = weight(pick<T, 7>(x), pick<T, 7>(y));
    }
    if (cut >= i && cut < i + VEC) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (i + e == cut) w[e] = 0.0;
    }
  };
  const int per = (nb + 31) / 32;         // blocks of a lane's part of the table
  double total = 0.0, part = 0.0, upto = 0.0;
  const double* tot = totals[0];
  for (int pass = 0; pass < 2; ++pass) {
    tot = totals[pass];
    for (int b = warp; b < nb; b += kSvWarps) {
      double s = 0.0;
      for (int k = 0; k < span; ++k) {
        const int64_t i0 = start + ((int64_t)b * span + k) * kSteps * kStep;
        uint4 x[kSteps], y[kSteps];
        load(i0, x, y);
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
          double w[VEC];
          weights(i0, u, x[u], y[u], w);
#pragma unroll
          for (int e = 0; e < VEC; ++e) s += w[e];
        }
      }
      s = warp_sum(s);
      if (lane == 0) mass[b] = s;
    }
    __syncthreads();
    if (warp == 0) {
      part = 0.0;
      for (int b = lane * per; b < min(nb, lane * per + per); ++b) part += mass[b];
      upto = part;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      const double all = __shfl_sync(0xffffffffu, upto, 31);
      if (lane < cl) {
        const uint32_t at = mapa_shared(smem_u32(&totals[pass][rank]), lane);
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(all) : "memory");
      }
    }
    if (cl > 1) cluster_sync();
    else __syncthreads();
    total = 0.0;
    for (int c = 0; c < cl; ++c) total += tot[c];
    if (total > 0.0 || (!q && cut < 0)) break;
    // nothing is left of p above q (p = q up to rounding): the draw is from p itself. The second pass exchanges through
    // the other row of totals, so that no CTA rewrites what another still reads
    q = nullptr;
    cut = -1;
  }
  if (warp != 0) return;
  // From here on sums in another order than above may differ in the last bit. Only parts with mass are taken, and where
  // none passes `want` the last one with mass is: an index without mass is never drawn.
  const double want = (double)a.coins[(int64_t)r * (a.D + 2) + a.D + 1] * total;
  double before = 0.0;
  int own = 0;
  for (; own < cl - 1 && !(before + tot[own] > want); ++own) before += tot[own];
  if (rank != own) return;
  const unsigned some = __ballot_sync(0xffffffffu, part > 0.0);
  if (!some) {                            // a row without mass
    if (lane == 0) a.bonus[r] = a.V - 1;
    return;
  }
  const unsigned past = __ballot_sync(0xffffffffu, part > 0.0 && before + upto > want);
  const int src = past ? __ffs(past) - 1 : 31 - __clz(some);
  before += __shfl_sync(0xffffffffu, upto - part, src);
  int block = 0;
  double skipped = 0.0;
  for (int b = src * per; b < min(nb, src * per + per); ++b) {   // every lane walks the same few entries
    if (mass[b] > 0.0) {
      block = b;
      skipped = before;
      if (before + mass[b] > want) break;
    }
    before += mass[b];
  }
  before = skipped;
  int found = -1, last = a.V - 1;
  for (int k = 0; k < span && found < 0; ++k) {
    const int64_t i0 = start + ((int64_t)block * span + k) * kSteps * kStep;
    uint4 x[kSteps], y[kSteps];
    load(i0, x, y);
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      if (found >= 0) break;
      double w[VEC], lsum = 0.0;
      weights(i0, u, x[u], y[u], w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) lsum += w[e];
      double inc = lsum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      const unsigned any = __ballot_sync(0xffffffffu, lsum > 0.0);
      const unsigned hit = __ballot_sync(0xffffffffu, lsum > 0.0 && before + inc > want);
      if (any) {
        const int at = hit ? __ffs(hit) - 1 : 31 - __clz(any);
        int idx = -1;
        if (lane == at) {
          double acc = before + (inc - lsum);
          bool done = false;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            if (!done && w[e] > 0.0) {
              idx = (int)(i0 + u * kStep + lane * VEC + e);
              acc += w[e];
              done = hit && acc > want;
            }
          }
        }
        idx = __shfl_sync(0xffffffffu, idx, at);
        if (hit) found = idx;
        else last = idx;
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  if (lane == 0) a.bonus[r] = found >= 0 ? found : last;
}

template <typename T>
void launch(const SvArgs& a, int64_t R, cudaStream_t stream) {
  constexpr int kBlock = kSteps * 32 * (16 / sizeof(T));
  const int64_t all = (a.V + kBlock - 1) / kBlock;
  // CTAs per request: more while the machine's resident CTAs are not all used and a CTA has more blocks than warps (a CTA
  // with fewer gains nothing, and the cluster's barrier costs about a microsecond)
  int cl = 1;
  while (cl < kMaxCluster && R * cl * 2 <= kSvResident * 148 && all > (int64_t)cl * kSvWarps) cl *= 2;
  int64_t blocks = (all + cl - 1) / cl;
  const int64_t span = (blocks + kMaxBlocks - 1) / kMaxBlocks;
  blocks = (blocks + span - 1) / span;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)cl, (unsigned)R);
  cfg.blockDim = dim3(kSvThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cl;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, spec_verify_kernel<T>, a, (int)blocks, (int)span));
}

}  // namespace

void spec_verify_probs(torch::Tensor p, c10::optional<torch::Tensor> q, torch::Tensor tokens, torch::Tensor coins,
                       c10::optional<torch::Tensor> n_draft, torch::Tensor acc, torch::Tensor bonus) {
  TORCH_CHECK(tokens.dim() == 2 && tokens.is_contiguous() && tokens.scalar_type() == at::kLong, "tokens: int64 [R, D]");
  const int64_t R = tokens.size(0), D = tokens.size(1);
  TORCH_CHECK(p.dim() == 3 && p.size(0) == R && p.size(1) == D + 1 && p.size(2) > 0 && p.size(2) < (int64_t(1) << 30) &&
              p.stride(2) == 1, "target probabilities: [R, D + 1, V] with contiguous rows");
  TORCH_CHECK(p.scalar_type() == at::kFloat || p.scalar_type() == at::kBFloat16 || p.scalar_type() == at::kHalf,
              "probabilities: fp32, bf16 or fp16");
  if (q)
    TORCH_CHECK(q->dim() == 3 && q->size(0) == R && q->size(1) == D && q->size(2) == p.size(2) && q->stride(2) == 1 &&
                q->scalar_type() == p.scalar_type() && q->device() == p.device(),
                "draft probabilities: [R, D, V] with contiguous rows, of the target's type and device");
  TORCH_CHECK(coins.dim() == 2 && coins.is_contiguous() && coins.scalar_type() == at::kFloat && coins.size(0) == R &&
              coins.size(1) == D + 2, "coins: fp32 [R, D + 2]");
  if (n_draft)
    TORCH_CHECK(n_draft->is_contiguous() && n_draft->scalar_type() == at::kInt && n_draft->numel() == R &&
                n_draft->device() == p.device(), "n_draft: int32 [R]");
  TORCH_CHECK(tokens.device() == p.device() && coins.device() == p.device() && acc.device() == p.device() &&
              bonus.device() == p.device(), "all tensors must be on the probabilities' device");
  TORCH_CHECK(R < 65536, "at most 65535 requests");
  if (R == 0) return;
  SvArgs a{p.data_ptr(), q ? q->data_ptr() : nullptr, tokens.data_ptr<int64_t>(), coins.data_ptr<float>(),
           n_draft ? n_draft->data_ptr<int>() : nullptr, acc.data_ptr<int64_t>(), bonus.data_ptr<int64_t>(),
           p.stride(0), p.stride(1), q ? q->stride(0) : 0, q ? q->stride(1) : 0, (int)D, (int)p.size(2)};
  const at::cuda::CUDAGuard guard(p.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  if (p.scalar_type() == at::kFloat) launch<float>(a, R, stream);
  else if (p.scalar_type() == at::kHalf) launch<__half>(a, R, stream);
  else launch<__nv_bfloat16>(a, R, stream);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace phx
