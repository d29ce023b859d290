// RMS norm of each query and key head, rotary embedding and paged-cache write in one pass, sm_100a.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                        (q heads: wq, k heads: wk; v heads are copied)
//   (y1, y2) -> (y1 c - y2 s, y2 c + y1 s)                    y1 = y[0 : rot/2], y2 = y[rot/2 : rot]
//   q -> [M, Hq, D], k and v -> the cache row of slots[t]; elements from rot on are normed and not rotated.
// The sum of squares, the norm and the rotation stay in fp32; each output is rounded to bf16 once (a chain of a norm
// op and a rotation op would round twice).
//
// Bound: HBM (each qkv row read once, written once; the cos/sin rows are shared by a token's heads and stay in L1/L2), with
// instruction issue close behind. 8192 rows x 48 heads of 128: 44 us, 4.6 TB/s of its 206 MB; 1283 rows x 20 heads of 256: 10 us.
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

// Aligned rows and D = 8 L for L = 8, 16 or 32 lanes: a lane holds two runs of four elements of a head that are each
// other's rotation partners (elements 4 i and rot / 2 + 4 i; in the part that is not rotated, any two runs), so the
// rotation needs no exchange. A warp takes 32 / L heads of one token at a time and P such groups in all, whose loads are
// issued together. The norm's weights are folded into the rotation once per warp (again where its heads go from q to k):
//   o1 = inv (x1 (w1 c) - x2 (w2 s)),  o2 = inv (x2 (w2 c) + x1 (w1 s)).
template <int L, int P>
__global__ void __launch_bounds__(256, 4) qk_norm_rope_wide_kernel(const QkArgs a) {
  constexpr int kHeads = 32 / L, D = 8 * L;
  const int nh = a.Hq + 2 * a.Hkv;
  const unsigned groups = (nh + kHeads * P - 1) / (kHeads * P);
  const unsigned w = blockIdx.x * 8u + (threadIdx.x >> 5);
  const int t = (int)(w / groups), h0 = (int)(w - t * groups) * kHeads * P;
  if (t >= a.M) return;
  const int lane = threadIdx.x & 31, i = lane % L, sub = lane / L;
  const bool turned = i < (a.rot >> 3);
  const int e1 = turned ? 4 * i : a.rot + 4 * (i - (a.rot >> 3));
  const int e2 = e1 + (turned ? a.rot >> 1 : (D - a.rot) >> 1);
  const __nv_bfloat16* src = a.qkv + (int64_t)t * a.ld + (int64_t)(h0 + sub) * D;
  uint2 x1[P], x2[P];
#pragma unroll
  for (int u = 0; u < P; ++u) {
    x1[u] = x2[u] = make_uint2(0, 0);
    if (h0 + u * kHeads + sub < nh) {
      x1[u] = *reinterpret_cast<const uint2*>(src + u * kHeads * D + e1);
      x2[u] = *reinterpret_cast<const uint2*>(src + u * kHeads * D + e2);
    }
  }
  const int row = turned ? table_row(a, t) : 0;
  const int64_t base = h0 + kHeads * P > a.Hq ? cache_base(a, t) : -1;
  float c1[4], s1[4], c2[4], s2[4];       // w1 c, w2 s, w2 c, w1 s
  auto fold = [&](const __nv_bfloat16* wt) {
    const uint2 g1 = *reinterpret_cast<const uint2*>(wt + e1), g2 = *reinterpret_cast<const uint2*>(wt + e2);
    float2 cs[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) cs[e] = make_float2(1.f, 0.f);
    if (turned) {
      const float4* c4 = reinterpret_cast<const float4*>(a.cos_sin + (int64_t)row * (a.rot >> 1) + 4 * i);
      const float4 lo = c4[0], hi = c4[1];
      cs[0] = make_float2(lo.x, lo.y), cs[1] = make_float2(lo.z, lo.w);
      cs[2] = make_float2(hi.x, hi.y), cs[3] = make_float2(hi.z, hi.w);
    }
    const float2 a0 = unpack_bf16x2(g1.x), a1 = unpack_bf16x2(g1.y), b0 = unpack_bf16x2(g2.x), b1 = unpack_bf16x2(g2.y);
    const float w1[4] = {a0.x, a0.y, a1.x, a1.y}, w2[4] = {b0.x, b0.y, b1.x, b1.y};
#pragma unroll
    for (int e = 0; e < 4; ++e) c1[e] = w1[e] * cs[e].x, s1[e] = w2[e] * cs[e].y, c2[e] = w2[e] * cs[e].x, s2[e] = w1[e] * cs[e].y;
  };
  fold(h0 + sub < a.Hq ? a.wq : a.wk);
#pragma unroll
  for (int u = 0; u < P; ++u) {
    const int h = h0 + u * kHeads + sub;
    const float2 a0 = unpack_bf16x2(x1[u].x), a1 = unpack_bf16x2(x1[u].y), b0 = unpack_bf16x2(x2[u].x), b1 = unpack_bf16x2(x2[u].y);
    float ss = fmaf(a0.x, a0.x, a0.y * a0.y) + fmaf(a1.x, a1.x, a1.y * a1.y) +
               (fmaf(b0.x, b0.x, b0.y * b0.y) + fmaf(b1.x, b1.x, b1.y * b1.y));
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (h >= nh) continue;
    if (u > 0 && h >= a.Hq && h - kHeads < a.Hq) fold(a.wk);
    uint2 r1 = x1[u], r2 = x2[u];
    if (h < a.Hq + a.Hkv) {
      const float inv = rsqrtf(ss * (1.f / D) + a.eps);
      const float y[4] = {a0.x * inv, a0.y * inv, a1.x * inv, a1.y * inv}, z[4] = {b0.x * inv, b0.y * inv, b1.x * inv, b1.y * inv};
      float o1[4], o2[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o1[e] = y[e] * c1[e];
        o2[e] = z[e] * c2[e];
      }
      if (turned) {                        // an infinity in one run stays out of the other where nothing is rotated
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o1[e] = fmaf(-z[e], s1[e], o1[e]);
          o2[e] = fmaf(y[e], s2[e], o2[e]);
        }
      }
      r1 = make_uint2(pack_bf16x2(o1[0], o1[1]), pack_bf16x2(o1[2], o1[3]));
      r2 = make_uint2(pack_bf16x2(o2[0], o2[1]), pack_bf16x2(o2[2], o2[3]));
    }
    __nv_bfloat16* dst;
    if (h < a.Hq) {
      dst = a.q_out + ((int64_t)t * a.Hq + h) * D;
    } else {
      if (base < 0) continue;
      const bool is_k = h < a.Hq + a.Hkv;
      dst = (is_k ? a.k_cache : a.v_cache) + base + (int64_t)(h - a.Hq - (is_k ? 0 : a.Hkv)) * a.page_size * D;
    }
    *reinterpret_cast<uint2*>(dst + e1) = r1;
    *reinterpret_cast<uint2*>(dst + e2) = r2;
  }
}

template <int L>
void launch_wide(const QkArgs& a, cudaStream_t stream) {
  constexpr int kHeads = 32 / L, kP = 4;
  const int nh = a.Hq + 2 * a.Hkv;
  // Groups per warp: 4 share the cos/sin and weight loads, 1 spreads a small batch over more SMs. 8192 rows x 48 heads of
  // 128: 4 groups 44 us, 8 groups (93 registers, half the warps) 55 us, a group of raw 16-byte rows with exchanged partners 86 us.
  const auto warps = [&](int p) { return (int64_t)a.M * ((nh + kHeads * p - 1) / (kHeads * p)); };
  if (warps(kP) >= 148 * 32)
    qk_norm_rope_wide_kernel<L, kP><<<(unsigned)((warps(kP) + 7) / 8), 256, 0, stream>>>(a);
  else
    qk_norm_rope_wide_kernel<L, 1><<<(unsigned)((warps(1) + 7) / 8), 256, 0, stream>>>(a);
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
  TORCH_CHECK(M < (int64_t(1) << 31) && M * (Hq + 2 * Hkv) < (int64_t(1) << 32) - 8, "too many (row, head) pairs for one launch");
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
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool wide = a.rot % 8 == 0 && a.ld % 8 == 0 && aligned(a.qkv) && aligned(a.wq) && aligned(a.wk) &&
                    aligned(a.cos_sin) && aligned(a.q_out) && aligned(a.k_cache) && aligned(a.v_cache);
  if (wide && D == 64) launch_wide<8>(a, stream);
  else if (wide && D == 128) launch_wide<16>(a, stream);
  else if (wide && D == 256) launch_wide<32>(a, stream);
  else {
    const int64_t warps = M * (Hq + 2 * Hkv);
    qk_norm_rope_narrow_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, stream>>>(a);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace phx
