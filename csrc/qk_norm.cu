// RMS norm of each query and key head, rotary embedding and paged-cache write in one pass, sm_100a.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                        (q heads: wq, k heads: wk; v heads are copied)
//   (y1, y2) -> (y1 c - y2 s, y2 c + y1 s)                    y1 = y[0 : rot/2], y2 = y[rot/2 : rot]
//   q -> [M, Hq, D], k and v -> the cache row of slots[t]; elements from rot on are normed and not rotated.
// The sum of squares, the norm and the rotation stay in fp32; each output is rounded to bf16 once (a chain of a norm
// op and a rotation op would round twice).
//
// Bound: HBM (each qkv row read once, written once; the cos/sin rows are shared by a token's heads and stay in L1/L2).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"

namespace phx {

namespace {

struct QkArgs {
  const __nv_bfloat16 *qkv, *wq, *wk;
  const int* pos;
  const int64_t* slots;      // null: nothing is written to the cache
  const float2* cos_sin;     // [max_pos, rot / 2]
  __nv_bfloat16 *q_out, *k_cache, *v_cache;
  int* status;
  int64_t ld, cap;           // row stride of qkv (elements); cache slots
  int M, Hq, Hkv, D, rot, page_size, max_pos;
  float eps;
};

// first cache element of (slot, KV head 0), KV heads page_size * D apart; negative: the row is not written
__device__ __forceinline__ int64_t cache_base(const QkArgs& a, int t) {
  if (!a.slots) return -1;
  const int64_t slot = a.slots[t];
  if (slot < 0) return -1;
  if (slot >= a.cap) {
    atomicCAS(a.status, 0, kErrIndex);
    return -1;
  }
  const int64_t page = slot / a.page_size;
  return (page * a.Hkv * a.page_size + (slot - page * a.page_size)) * a.D;
}

// A position outside the table is reported and its row takes the table's nearest one.
__device__ __forceinline__ int table_row(const QkArgs& a, int t) {
  const int p = a.pos[t];
  if (p >= 0 && p < a.max_pos) return p;
  atomicCAS(a.status, 0, kErrIndex);
  return p < 0 ? 0 : a.max_pos - 1;
}

// Any D and rot, any alignment: one warp per (token, head), element by element; the rotation partner is read again
// (an L1 hit).
__global__ void __launch_bounds__(256) qk_norm_rope_narrow_kernel(const QkArgs a) {
  const int nh = a.Hq + 2 * a.Hkv;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= (int64_t)a.M * nh) return;
  const int t = (int)(w / nh), h = (int)(w % nh), lane = threadIdx.x & 31;
  const __nv_bfloat16* src = a.qkv + (int64_t)t * a.ld + (int64_t)h * a.D;
  __nv_bfloat16* dst;
  if (h < a.Hq) {
    dst = a.q_out + ((int64_t)t * a.Hq + h) * a.D;
  } else {
    const int64_t base = cache_base(a, t);
    if (base < 0) return;
    const bool is_k = h < a.Hq + a.Hkv;
    const int kvh = h - a.Hq - (is_k ? 0 : a.Hkv);
    dst = (is_k ? a.k_cache : a.v_cache) + base + (int64_t)kvh * a.page_size * a.D;
    if (!is_k) {
      for (int d = lane; d < a.D; d += 32) dst[d] = src[d];
      return;
    }
  }
  const __nv_bfloat16* wt = h < a.Hq ? a.wq : a.wk;
  float ss = 0.f;
  for (int d = lane; d < a.D; d += 32) {
    const float x = __bfloat162float(src[d]);
    ss = fmaf(x, x, ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float inv = rsqrtf(ss / a.D + a.eps);
  const int half = a.rot / 2;
  const float2* cs = a.cos_sin + (int64_t)table_row(a, t) * half;
  for (int d = lane; d < a.D; d += 32) {
    float y = __bfloat162float(src[d]) * inv * __bfloat162float(wt[d]);
    if (d < a.rot) {
      const int pd = d < half ? d + half : d - half;
      const float yp = __bfloat162float(src[pd]) * inv * __bfloat162float(wt[pd]);
      const float2 c = cs[d < half ? d : pd];
      y = d < half ? y * c.x - yp * c.y : y * c.x + yp * c.y;
    }
    dst[d] = __float2bfloat16(y);
  }
}

}  // namespace

void qk_norm_rope_kv_write(torch::Tensor qkv, torch::Tensor wq, torch::Tensor wk, double eps, torch::Tensor pos,
                           c10::optional<torch::Tensor> slots, torch::Tensor cos_sin, torch::Tensor q_out,
                           c10::optional<torch::Tensor> k_cache, c10::optional<torch::Tensor> v_cache, int64_t Hq,
                           int64_t Hkv, int64_t D, torch::Tensor status) {
  TORCH_CHECK(qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16 && qkv.stride(1) == 1, "qkv: [M, width] bf16 rows");
  const int64_t M = qkv.size(0);
  TORCH_CHECK(Hq > 0 && Hkv >= 0 && D > 0 && qkv.size(1) == (Hq + 2 * Hkv) * D, "qkv width is not (hq + 2 hkv) d");
  TORCH_CHECK(wq.is_contiguous() && wk.is_contiguous() && wq.numel() == D && wk.numel() == D &&
              wq.scalar_type() == at::kBFloat16 && wk.scalar_type() == at::kBFloat16, "norm weights: [d] bf16");
  TORCH_CHECK(pos.is_contiguous() && pos.scalar_type() == at::kInt && pos.numel() == M, "pos: int32 [M]");
  TORCH_CHECK(cos_sin.dim() == 3 && cos_sin.size(2) == 2 && cos_sin.is_contiguous() &&
              cos_sin.scalar_type() == at::kFloat && cos_sin.size(0) > 0 && 2 * cos_sin.size(1) <= D,
              "cos_sin: [positions, rot / 2, 2] fp32 with rot <= d");
  TORCH_CHECK(q_out.is_contiguous() && q_out.scalar_type() == at::kBFloat16 && q_out.numel() == M * Hq * D,
              "q_out: [M, hq, d] bf16");
  TORCH_CHECK(k_cache.has_value() == v_cache.has_value() && (!slots || k_cache), "slots need both caches");
  QkArgs a{};
  if (k_cache) {
    for (const auto* c : {&*k_cache, &*v_cache})
      TORCH_CHECK(c->dim() == 4 && c->is_contiguous() && c->scalar_type() == at::kBFloat16 && c->size(1) == Hkv &&
                  c->size(3) == D && c->sizes() == k_cache->sizes() && c->device() == qkv.device(),
                  "caches: [pages, hkv, page_size, d] bf16 on qkv's device");
    a.k_cache = reinterpret_cast<__nv_bfloat16*>(k_cache->data_ptr());
    a.v_cache = reinterpret_cast<__nv_bfloat16*>(v_cache->data_ptr());
    a.page_size = (int)k_cache->size(2);
    a.cap = k_cache->size(0) * k_cache->size(2);
  }
  if (slots) {
    TORCH_CHECK(slots->is_contiguous() && slots->scalar_type() == at::kLong && slots->numel() == M, "slots: int64 [M]");
    a.slots = slots->data_ptr<int64_t>();
  }
  for (const auto* t : {&wq, &wk, &pos, &cos_sin, &q_out, &status})
    TORCH_CHECK(t->device() == qkv.device(), "all tensors must be on qkv's device");
  TORCH_CHECK(M * (Hq + 2 * Hkv) < (int64_t(1) << 33), "too many (row, head) pairs for one launch");
  if (M == 0) return;
  a.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv.data_ptr());
  a.wq = reinterpret_cast<const __nv_bfloat16*>(wq.data_ptr());
  a.wk = reinterpret_cast<const __nv_bfloat16*>(wk.data_ptr());
  a.pos = pos.data_ptr<int>();
  a.cos_sin = reinterpret_cast<const float2*>(cos_sin.data_ptr());
  a.q_out = reinterpret_cast<__nv_bfloat16*>(q_out.data_ptr());
  a.status = status.data_ptr<int>();
  a.ld = qkv.stride(0);
  a.M = (int)M;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.D = (int)D;
  a.rot = 2 * (int)cos_sin.size(1);
  a.max_pos = (int)cos_sin.size(0);
  a.eps = (float)eps;
  const at::cuda::CUDAGuard guard(qkv.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const int64_t warps = M * (Hq + 2 * Hkv);
  qk_norm_rope_narrow_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace phx
