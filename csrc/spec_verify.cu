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

constexpr int kSvThreads = 512;
constexpr int kSvWarps = kSvThreads / 32;

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

// One CTA per request: 512 threads take the row in segments of one warp each.
template <typename T>
__global__ void __launch_bounds__(kSvThreads) spec_verify_kernel(const SvArgs a) {
  __shared__ double seg[kSvWarps];
  __shared__ int s_kept;
  const int r = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = a.n_draft ? max(0, min(a.D, a.n_draft[r])) : a.D;
  if (warp == 0) {
    const int k = accepted<T>(a, r, n, lane);
    if (lane == 0) s_kept = k;
    for (int d = lane; d < a.D; d += 32) a.acc[(int64_t)r * a.D + d] = d < k ? d + 1 : -1;
  }
  __syncthreads();
  const int kept = s_kept;
  const T* p = static_cast<const T*>(a.p) + r * a.p_r + kept * a.p_d;
  const T* q = a.q && kept < n ? static_cast<const T*>(a.q) + r * a.q_r + kept * a.q_d : nullptr;
  int64_t cut = !a.q && kept < n ? a.tokens[(int64_t)r * a.D + kept] : -1;   // greedy draft: its token is taken out
  const int per = (a.V + kSvWarps - 1) / kSvWarps;
  const int lo = min(a.V, warp * per), hi = min(a.V, lo + per);
  auto w = [&](int i) { return i == cut ? 0.0 : weight(to_f(p[i]), q ? to_f(q[i]) : 0.f); };
  double total;
  while (true) {
    double s = 0.0;
    for (int i = lo + lane; i < hi; i += 32) s += w(i);
    s = warp_sum(s);
    if (lane == 0) seg[warp] = s;
    __syncthreads();
    total = 0.0;
    for (int j = 0; j < kSvWarps; ++j) total += seg[j];
    if (total > 0.0 || (!q && cut < 0)) break;
    q = nullptr;            // nothing is left of p above q (p = q up to rounding): the draw is from p itself
    cut = -1;
    __syncthreads();
  }
  const double want = (double)a.coins[(int64_t)r * (a.D + 2) + a.D + 1] * total;
  double before = 0.0;
  int own = 0;
  for (; own < kSvWarps - 1 && !(before + seg[own] > want); ++own) before += seg[own];
  if (warp != own) return;
  int found = -1, last = -1;
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    const double x = i < hi ? w(i) : 0.0;
    double inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    const unsigned m = __ballot_sync(0xffffffffu, before + inc > want), pos = __ballot_sync(0xffffffffu, x > 0.0);
    if (pos) last = i0 + 31 - __clz(pos);
    if (m) {
      found = i0 + __ffs(m) - 1;
      break;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  // the scan's sums may round below the segment's: the draw is then the segment's last index with any mass
  if (lane == 0) a.bonus[r] = found >= 0 ? found : last >= 0 ? last : a.V - 1;
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
  if (R == 0) return;
  SvArgs a{p.data_ptr(), q ? q->data_ptr() : nullptr, tokens.data_ptr<int64_t>(), coins.data_ptr<float>(),
           n_draft ? n_draft->data_ptr<int>() : nullptr, acc.data_ptr<int64_t>(), bonus.data_ptr<int64_t>(),
           p.stride(0), p.stride(1), q ? q->stride(0) : 0, q ? q->stride(1) : 0, (int)D, (int)p.size(2)};
  const at::cuda::CUDAGuard guard(p.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  if (p.scalar_type() == at::kFloat) spec_verify_kernel<float><<<(unsigned)R, kSvThreads, 0, stream>>>(a);
  else if (p.scalar_type() == at::kHalf) spec_verify_kernel<__half><<<(unsigned)R, kSvThreads, 0, stream>>>(a);
  else spec_verify_kernel<__nv_bfloat16><<<(unsigned)R, kSvThreads, 0, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace phx
