// Gated delta rule over ragged token runs (prompt passes), sm_100a. Same recurrence as csrc/gdn.cu:
//   q^ = q / |q| * scale, k^ = k / |k| (eps 1e-6 in the root), per value head with S [128 key, 128 value] fp32
//   S <- e^g S;  v' = beta (v - S^T k^);  S <- S + k^ v'^T;  o = S^T q^
// q, k and v may be strided views (the layer's convolution output); rows past the last run are not touched.
//
// gdn_step_kernel: token by token, one CTA per (request, value head). Threads 2j and 2j + 1 own the halves of state
// column j in registers, so a token costs two pair-local dot products and a thread-local update.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"

namespace phx {

namespace {

constexpr int kDim = 128;

struct GdnArgs {
  const __nv_bfloat16 *q, *k, *v;
  const float *g, *beta;         // [T, HV]
  float* state;                  // [slots, HV, 128, 128]
  const int *tok_start, *slot;
  __nv_bfloat16* out;            // [T, HV, 128]
  int* status;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;   // strides of tokens and heads (elements)
  int T, R, HK, HV, slots;
  float scale;
};

// Tokens [t0, t1) and state of request r; false (and a status code) if they lie outside the buffers.
__device__ __forceinline__ bool request(const GdnArgs& a, int r, int& t0, int& t1, int& slot) {
  t0 = a.tok_start[r];
  t1 = a.tok_start[r + 1];
  slot = a.slot[r];
  const bool ok = t0 >= 0 && t0 <= t1 && t1 <= a.T && slot >= 0 && slot < a.slots;
  if (!ok && threadIdx.x == 0) atomicCAS(a.status, 0, kErrIndex);
  return ok;
}

constexpr int kStepTokens = 16;          // tokens whose q and k are normalised together
constexpr int kHalf = kDim / 2;
constexpr int kRowPad = kDim + 8;        // the second half starts 4 floats later: both halves' reads miss each other's banks

__global__ void __launch_bounds__(256) gdn_step_kernel(const GdnArgs a) {
  __shared__ __align__(16) float sq[kStepTokens][kRowPad], sk[kStepTokens][kRowPad];
  __shared__ float sdec[kStepTokens], sbeta[kStepTokens];
  const int h = blockIdx.y, hk = h / (a.HV / a.HK);
  int t0, t1, slot;
  if (!request(a, blockIdx.x, t0, t1, slot) || t0 == t1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = threadIdx.x >> 1, half = threadIdx.x & 1;
  const int hoff = half * (kHalf + 4);
  float* S = a.state + ((int64_t)slot * a.HV + h) * kDim * kDim + half * kHalf * kDim + j;
  float col[kHalf];
#pragma unroll
  for (int i = 0; i < kHalf; ++i) col[i] = S[i * kDim];
  for (int c0 = t0; c0 < t1; c0 += kStepTokens) {
    const int n = min(kStepTokens, t1 - c0);
    for (int u = warp; u < n; u += 8) {
      const __nv_bfloat16* qp = a.q + (int64_t)(c0 + u) * a.q_t + hk * a.q_h;
      const __nv_bfloat16* kp = a.k + (int64_t)(c0 + u) * a.k_t + hk * a.k_h;
      float qv[4], kv[4], qq = 0.f, kk = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        qv[e] = __bfloat162float(qp[lane + 32 * e]);
        kv[e] = __bfloat162float(kp[lane + 32 * e]);
        qq = fmaf(qv[e], qv[e], qq);
        kk = fmaf(kv[e], kv[e], kk);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        qq += __shfl_xor_sync(0xffffffffu, qq, o);
        kk += __shfl_xor_sync(0xffffffffu, kk, o);
      }
      const float qn = rsqrtf(qq + 1e-6f) * a.scale, kn = rsqrtf(kk + 1e-6f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = lane + 32 * e, pi = i < kHalf ? i : i + 4;
        sq[u][pi] = qv[e] * qn;
        sk[u][pi] = kv[e] * kn;
      }
      if (lane == 0) {
        sdec[u] = expf(a.g[(int64_t)(c0 + u) * a.HV + h]);
        sbeta[u] = a.beta[(int64_t)(c0 + u) * a.HV + h];
      }
    }
    __syncthreads();
    for (int u = 0; u < n; ++u) {
      const float vj = __bfloat162float(a.v[(int64_t)(c0 + u) * a.v_t + h * a.v_h + j]);
      const float decay = sdec[u];
      const float4* k4 = reinterpret_cast<const float4*>(&sk[u][hoff]);
      const float4* q4 = reinterpret_cast<const float4*>(&sq[u][hoff]);
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kHalf / 4; ++i) {
        const float4 kk = k4[i];
        s.x = fmaf(col[4 * i] *= decay, kk.x, s.x);
        s.y = fmaf(col[4 * i + 1] *= decay, kk.y, s.y);
        s.z = fmaf(col[4 * i + 2] *= decay, kk.z, s.z);
        s.w = fmaf(col[4 * i + 3] *= decay, kk.w, s.w);
      }
      float kv = (s.x + s.y) + (s.z + s.w);
      kv += __shfl_xor_sync(0xffffffffu, kv, 1);
      const float vp = (vj - kv) * sbeta[u];
      s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kHalf / 4; ++i) {
        const float4 kk = k4[i], qq = q4[i];
        s.x = fmaf(col[4 * i] = fmaf(kk.x, vp, col[4 * i]), qq.x, s.x);
        s.y = fmaf(col[4 * i + 1] = fmaf(kk.y, vp, col[4 * i + 1]), qq.y, s.y);
        s.z = fmaf(col[4 * i + 2] = fmaf(kk.z, vp, col[4 * i + 2]), qq.z, s.z);
        s.w = fmaf(col[4 * i + 3] = fmaf(kk.w, vp, col[4 * i + 3]), qq.w, s.w);
      }
      float o = (s.x + s.y) + (s.z + s.w);
      o += __shfl_xor_sync(0xffffffffu, o, 1);
      if (half == 0) a.out[((int64_t)(c0 + u) * a.HV + h) * kDim + j] = __float2bfloat16(o);
    }
    __syncthreads();   // the next tokens rewrite the shared rows
  }
#pragma unroll
  for (int i = 0; i < kHalf; ++i) S[i * kDim] = col[i];
}

}  // namespace

void gdn_chunked(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor g, torch::Tensor beta,
                 torch::Tensor state, torch::Tensor tok_start, torch::Tensor slot, double scale, torch::Tensor out,
                 torch::Tensor status) {
  TORCH_CHECK(q.dim() == 3 && v.dim() == 3 && q.sizes() == k.sizes() && q.size(0) == v.size(0) && q.size(2) == kDim &&
              v.size(2) == kDim, "q, k: [T, HK, 128], v: [T, HV, 128]");
  const int64_t T = q.size(0), HK = q.size(1), HV = v.size(1), R = slot.numel();
  TORCH_CHECK(HK > 0 && HV > 0 && HV % HK == 0, "value heads must be a multiple of key heads");
  for (const auto* x : {&q, &k, &v})
    TORCH_CHECK(x->scalar_type() == at::kBFloat16 && x->stride(2) == 1, "q, k, v: bf16 with contiguous heads");
  TORCH_CHECK(g.sizes() == beta.sizes() && g.dim() == 2 && g.size(0) == T && g.size(1) == HV && g.is_contiguous() &&
              beta.is_contiguous() && g.scalar_type() == at::kFloat && beta.scalar_type() == at::kFloat,
              "g, beta: fp32 [T, HV]");
  TORCH_CHECK(state.dim() == 4 && state.size(1) == HV && state.size(2) == kDim && state.size(3) == kDim &&
              state.is_contiguous() && state.scalar_type() == at::kFloat, "state: fp32 [slots, HV, 128, 128]");
  TORCH_CHECK(tok_start.numel() == R + 1 && tok_start.is_contiguous() && slot.is_contiguous() &&
              tok_start.scalar_type() == at::kInt && slot.scalar_type() == at::kInt, "tok_start [R + 1], slot [R]: int32");
  TORCH_CHECK(out.is_contiguous() && out.sizes() == v.sizes() && out.scalar_type() == at::kBFloat16, "out: bf16 [T, HV, 128]");
  for (const auto* x : {&k, &v, &g, &beta, &state, &tok_start, &slot, &out, &status})
    TORCH_CHECK(x->device() == q.device(), "all tensors must be on q's device");
  TORCH_CHECK(T < (int64_t(1) << 30) && HV < 65536, "too many tokens or heads");
  if (R == 0 || T == 0) return;
  auto P = [](const torch::Tensor& t) { return reinterpret_cast<const __nv_bfloat16*>(t.data_ptr()); };
  GdnArgs a{P(q), P(k), P(v), g.data_ptr<float>(), beta.data_ptr<float>(), state.data_ptr<float>(),
            tok_start.data_ptr<int>(), slot.data_ptr<int>(), reinterpret_cast<__nv_bfloat16*>(out.data_ptr()),
            status.data_ptr<int>(), q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
            (int)T, (int)R, (int)HK, (int)HV, (int)state.size(0), (float)scale};
  const at::cuda::CUDAGuard guard(q.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  gdn_step_kernel<<<dim3((unsigned)R, (unsigned)HV), 256, 0, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace phx
