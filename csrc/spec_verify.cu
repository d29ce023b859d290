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
constexpr int kSvResident = 2;          // CTAs per SM: 32 warps, each with three times 16 bytes of both rows a lane in flight

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

// 16 bytes of a row from element i on, zeros past its end. A row that does not start on a 16-byte boundary is read in the
// two 16-byte granules around them (each holds bytes of the row, so it lies in the row's allocation) and shifted.
template <typename T>
__device__ __forceinline__ uint4 load16(const T* row, int i, int V) {
  if (i >= V) return make_uint4(0, 0, 0, 0);
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + i);
  const unsigned off = at & 15;
  const int left = (V - i) * (int)sizeof(T);
  const uint4* g = reinterpret_cast<const uint4*>(at - off);
  uint4 u = g[0];
  if (off) {
    const uint4 n = left > 16 - (int)off ? g[1] : make_uint4(0, 0, 0, 0);
    uint64_t w0 = (uint64_t)u.y << 32 | u.x, w1 = (uint64_t)u.w << 32 | u.z, w2 = (uint64_t)n.y << 32 | n.x,
             w3 = (uint64_t)n.w << 32 | n.z;
    if (off & 8) w0 = w1, w1 = w2, w2 = w3;
    const unsigned sh = (off & 7) * 8;
    if (sh) w0 = w0 >> sh | w1 << (64 - sh), w1 = w1 >> sh | w2 << (64 - sh);
    u = make_uint4((uint32_t)w0, (uint32_t)(w0 >> 32), (uint32_t)w1, (uint32_t)(w1 >> 32));
  }
  if (left < 16) {
    auto keep = [&](uint32_t x, int k) { return left >= 4 * k + 4 ? x : left > 4 * k ? x & 0xffffu : 0u; };
    u = make_uint4(keep(u.x, 0), keep(u.y, 1), keep(u.z, 2), keep(u.w, 3));
  }
  return u;
}
// element e of 16 bytes (e a constant after unrolling)
template <typename T>
__device__ __forceinline__ float pick(const uint4& u, int e) {
  const int k = e * (int)sizeof(T) / 4;
  const uint32_t w = k == 0 ? u.x : k == 1 ? u.y : k == 2 ? u.z : u.w;
  if constexpr (sizeof(T) == 4) return __uint_as_float(w);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)(w >> (16 * (e & 1)))));
  else return __uint_as_float((e & 1) ? w & 0xffff0000u : w << 16);
}
// The part in which the draw falls, of 32 lanes' consecutive parts: the first one with mass whose running sum passes
// `want`, else (sums in another order may differ in the last bit) the last one with mass, so that an index without mass is
// never drawn; -1 if none has. `before` grows by the mass of the parts ahead of it. `hit`: whether a sum passed.
__device__ __forceinline__ int find_part(double part, double& before, double want, int lane, bool& hit) {
  double upto = part;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  const unsigned some = __ballot_sync(0xffffffffu, part > 0.0), past = __ballot_sync(0xffffffffu, part > 0.0 && before + upto > want);
  hit = past != 0;
  if (!some) {
    before += __shfl_sync(0xffffffffu, upto, 31);
    return -1;
  }
  const int at = past ? __ffs(past) - 1 : 31 - __clz(some);
  before += __shfl_sync(0xffffffffu, upto - part, at);
  return at;
}

constexpr int kMaxCluster = 8;

// A cluster of CTAs (the grid's x) per request; each warp sums `span` neighbouring steps of 32 lanes x 16 bytes. The CTAs
// exchange their masses through shared memory. In the one where the draw falls, its warps share the steps of the warp
// where it falls, which are read a second time (from L2), and the warp that meets it finds the index. So the row comes
// from memory once, and the sum over a row has no exchange between lanes in it: fp64 additions are far apart.
// Bound: HBM for a full batch on a large vocabulary; else the chain of dependent reads (token, its probabilities, row,
// cluster barrier, steps), about 8 us with the launch. Measured (kernel
// alone, cold cache): 64 requests x 128256 fp32 29 us, 256 x 32000 bf16 17 us, 17 x 32003 bf16 without draft rows 10 us,
// 1 x 4096 8 us. With 4 x 16 bytes unrolled and a mass per 512 elements: 21 / 17 / 12 / 8, slower over a range of calls.
template <typename T>
__global__ void __launch_bounds__(kSvThreads, kSvResident) spec_verify_kernel(const SvArgs a, int span) {
  constexpr int VEC = 16 / sizeof(T), kStep = 32 * VEC;
  __shared__ double mass[2][kSvWarps];
  __shared__ double totals[2][kMaxCluster];
  __shared__ int s_kept;
  const int cl = gridDim.x, rank = blockIdx.x, r = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (cl > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const int n = a.n_draft ? max(0, min(a.D, a.n_draft[r])) : a.D;
  const float coin = a.coins[(int64_t)r * (a.D + 2) + a.D + 1];
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
  // this lane's first element of a step, its 16 bytes of each row, their weights and their sum
  const auto first = [&](int step) { return min(step * kStep + lane * VEC, a.V); };     // below 2^31: V is below 2^30
  const auto load = [&](int i, uint4& x, uint4& y) {
    x = load16<T>(p, i, a.V);
    y = q ? load16<T>(q, i, a.V) : make_uint4(0, 0, 0, 0);
  };
  const auto weights = [&](int i, const uint4& x, const uint4& y, double (&w)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[e] = i + e == cut ? 0.0 : weight(pick<T>(x, e), pick<T>(y, e));
    double m = (w[0] + w[1]) + (w[2] + w[3]);
    if constexpr (VEC == 8) m += (w[4] + w[5]) + (w[6] + w[7]);
    return m;
  };
  // mass of `count` steps from `step` on, the same in every lane; two loads ahead of the sums
  const auto steps_mass = [&](int step, int count) {
    double m = 0.0, w[VEC];
    uint4 x0, y0, x1, y1;
    load(count > 0 ? first(step) : a.V, x0, y0);
    load(count > 1 ? first(step + 1) : a.V, x1, y1);
#pragma unroll 1
    for (int k = 0; k < count; ++k) {
      const uint4 x = x0, y = y0;
      x0 = x1, y0 = y1;
      load(k + 2 < count ? first(step + k + 2) : a.V, x1, y1);
      m += weights(first(step + k), x, y, w);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    return m;
  };
  double total = 0.0;
  const double* tot = totals[0];
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    tot = totals[pass];
    const double m = steps_mass((rank * kSvWarps + warp) * span, span);
    if (lane == 0) mass[0][warp] = m;
    __syncthreads();
    if (warp == 0) {
      double all = lane < kSvWarps ? mass[0][lane] : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      if (lane < cl) {
        const uint32_t at = mapa_shared(smem_u32(&totals[pass][rank]), lane);
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(all) : "memory");
      }
    }
    if (cl > 1) cluster_sync();
    else __syncthreads();
    total = 0.0;
#pragma unroll 1
    for (int c = 0; c < cl; ++c) total += tot[c];
    if (total > 0.0 || (!q && cut < 0)) break;
    // nothing is left of p above q (p = q up to rounding): the draw is from p itself. The second pass exchanges through
    // the other row of totals, so that no CTA rewrites what another still reads
    q = nullptr;
    cut = -1;
  }
  const double want = (double)coin * total;
  double before = 0.0;
  bool hit;
  const int own = find_part(lane < cl ? tot[lane] : 0.0, before, want, lane, hit);
  if (own < 0) {                          // a row without mass
    if (rank == 0 && threadIdx.x == 0) a.bonus[r] = a.V - 1;
    return;
  }
  if (rank != own) return;
  const int ow = max(0, find_part(lane < kSvWarps ? mass[0][lane] : 0.0, before, want, lane, hit));
  const int sub = (span + kSvWarps - 1) / kSvWarps, base = (rank * kSvWarps + ow) * span;
  {
    const double m = steps_mass(base + warp * sub, max(0, min(sub, span - warp * sub)));
    if (lane == 0) mass[1][warp] = m;
  }
  __syncthreads();
  const int sw = max(0, find_part(lane < kSvWarps ? mass[1][lane] : 0.0, before, want, lane, hit));
  if (warp != sw) return;
  int found = a.V - 1;
  hit = false;
#pragma unroll 1
  for (int k = 0; k < min(sub, span - warp * sub) && !hit; ++k) {
    const int i = first(base + warp * sub + k);
    uint4 x, y;
    load(i, x, y);
    double w[VEC];
    const double lsum = weights(i, x, y, w);
    const int at = find_part(lsum, before, want, lane, hit);
    if (at < 0) continue;
    int idx = -1;
    bool done = false;
    double acc = before;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (!done && w[e] > 0.0) {
        idx = i + e;
        acc += w[e];
        done = hit && acc > want;
      }
    }
    found = __shfl_sync(0xffffffffu, idx, at);
    before += __shfl_sync(0xffffffffu, lsum, at);
  }
  if (lane == 0) a.bonus[r] = found;
}

template <typename T>
void launch(const SvArgs& a, int64_t R, cudaStream_t stream) {
  constexpr int kStep = 32 * (16 / sizeof(T));
  const int64_t steps = (a.V + kStep - 1) / kStep;
  // CTAs per request: more while all of them are resident at once (a second wave starts its chain of reads anew) and a warp has more than two steps (with
  // fewer a CTA gains nothing, and the cluster's barrier costs about a microsecond)
  int cl = 1;
  while (cl < kMaxCluster && R * cl * 2 <= kSvResident * 148 && steps > (int64_t)cl * 2 * kSvWarps) cl *= 2;
  const int64_t span = (steps + cl * kSvWarps - 1) / (cl * kSvWarps);
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
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, spec_verify_kernel<T>, a, (int)span));
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
