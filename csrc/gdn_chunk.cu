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
#include "tmap.h"

namespace phx {

namespace {

constexpr int kDim = 128;
constexpr double kLog2e = 1.4426950408889634;

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

// Mean tokens per request up to which tokens are taken one by one. Measured, us by steps / by chunks: 1 request x 8 heads,
// 16 tokens 14.5 / 16.5, 24 tokens 20.6 / 16.5; 64 requests x 16 heads, 8 tokens 58 / 78, 12 tokens 86 / 76; 200 x 32,
// 4 tokens 331 / 429, 12 tokens 612 / 438: a step costs each wave of CTAs 0.5 us, the chunk form each wave its set-up of
// 10 us. All tokens may belong to one request (lengths stay on the device), so steps are also bounded to 64 a wave, except
// where q, k, v or out are off the boundaries that the chunk form's copies need: those calls have no other form.
constexpr int kStepMeanOneWave = 16, kStepMean = 8, kStepsPerWave = 64;
constexpr int kStepTokens = 16;          // tokens whose q and k are normalised together
constexpr int kHalf = kDim / 2;
constexpr int kRowPad = kDim + 8;        // the second half starts 4 floats later: both halves' reads miss each other's banks

struct StepSmem {
  float q[kStepTokens][kRowPad], k[kStepTokens][kRowPad];
  float dec[kStepTokens], beta[kStepTokens];
};

// Tokens [t0, t1) of one request and value head, by 256 threads; `sync` joins them.
template <class Sync>
__device__ __forceinline__ void step_tokens(const GdnArgs& a, int h, int t0, int t1, int slot, int tid, StepSmem& s, Sync sync) {
  const int hk = h / (a.HV / a.HK);
  const int warp = tid >> 5, lane = tid & 31;
  const int j = tid >> 1, half = tid & 1;
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
        s.q[u][pi] = qv[e] * qn;
        s.k[u][pi] = kv[e] * kn;
      }
      if (lane == 0) {
        s.dec[u] = expf(a.g[(int64_t)(c0 + u) * a.HV + h]);
        s.beta[u] = a.beta[(int64_t)(c0 + u) * a.HV + h];
      }
    }
    sync();
    for (int u = 0; u < n; ++u) {
      const float vj = __bfloat162float(a.v[(int64_t)(c0 + u) * a.v_t + h * a.v_h + j]);
      const float decay = s.dec[u];
      const float4* k4 = reinterpret_cast<const float4*>(&s.k[u][hoff]);
      const float4* q4 = reinterpret_cast<const float4*>(&s.q[u][hoff]);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kHalf / 4; ++i) {
        const float4 kk = k4[i];
        sum.x = fmaf(col[4 * i] *= decay, kk.x, sum.x);
        sum.y = fmaf(col[4 * i + 1] *= decay, kk.y, sum.y);
        sum.z = fmaf(col[4 * i + 2] *= decay, kk.z, sum.z);
        sum.w = fmaf(col[4 * i + 3] *= decay, kk.w, sum.w);
      }
      float kv = (sum.x + sum.y) + (sum.z + sum.w);
      kv += __shfl_xor_sync(0xffffffffu, kv, 1);
      const float vp = (vj - kv) * s.beta[u];
      sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kHalf / 4; ++i) {
        const float4 kk = k4[i], qq = q4[i];
        sum.x = fmaf(col[4 * i] = fmaf(kk.x, vp, col[4 * i]), qq.x, sum.x);
        sum.y = fmaf(col[4 * i + 1] = fmaf(kk.y, vp, col[4 * i + 1]), qq.y, sum.y);
        sum.z = fmaf(col[4 * i + 2] = fmaf(kk.z, vp, col[4 * i + 2]), qq.z, sum.z);
        sum.w = fmaf(col[4 * i + 3] = fmaf(kk.w, vp, col[4 * i + 3]), qq.w, sum.w);
      }
      float o = (sum.x + sum.y) + (sum.z + sum.w);
      o += __shfl_xor_sync(0xffffffffu, o, 1);
      if (half == 0) a.out[((int64_t)(c0 + u) * a.HV + h) * kDim + j] = __float2bfloat16(o);
    }
    sync();   // the next tokens rewrite the shared rows
  }
#pragma unroll
  for (int i = 0; i < kHalf; ++i) S[i * kDim] = col[i];
}

__global__ void __launch_bounds__(256) gdn_step_kernel(const GdnArgs a) {
  __shared__ __align__(16) StepSmem s;
  int t0, t1, slot;
  if (!request(a, blockIdx.x, t0, t1, slot) || t0 == t1) return;
  step_tokens(a, blockIdx.y, t0, t1, slot, threadIdx.x, s, [] { __syncthreads(); });
}

// ------------------------------------------------------------------------------------------------
// Chunks of 64 tokens. With b_i the sum of g up to token i of a chunk, S0 the state before it:
//   (I + L) V' = diag(beta) (V - diag(e^b) K^ S0),   L_ij = beta_i e^(b_i - b_j) k^_i . k^_j   (j < i)
//   O  = diag(e^b) Q^ S0 + P V',                     P_ij = e^(b_i - b_j) q^_i . k^_j          (j <= i)
//   S1 = e^(b_C) S0 + sum_j e^(b_C - b_j) k^_j v'_j^T
// gdn_prep_kernel forms X = (I + L)^-1 - I, P and the tokens' factors for every chunk and head at once; gdn_chain_kernel
// walks the chunks of one (request, head) with the state in registers. The normalisation of k and q is folded into
// those factors, so the tensor core reads k and q as they are in memory (bf16, exact). Every fp32 operand goes in as bf16
// pieces, hi = bf16(x), lo = bf16(x - hi), off by at most 2^-18 of x: S, X, P and V' as two; R and V' c2, whose rounding
// the state would keep, as three (2^-27). With two for all of them the state after 2048 tokens was off by 2.7e-6 of its
// norm, of which V' c2 alone made 2.5e-6 and the product of the two lo pieces left out of R^T X^T 1.0e-6; now 0.7e-6.
// ------------------------------------------------------------------------------------------------
constexpr int kC = 64;                                   // tokens per chunk
constexpr int kTri = 5120;                               // one piece of a lower-triangular 64 x 64 matrix, see tri_offset
constexpr int kVecFloats = 4 * kC + 16;                  // beta, c1, c2, c3 per token; e^(b_C)
constexpr int kItemBytes = 4 * kTri + kVecFloats * 4;    // X hi, X lo, P hi, P lo, factors

// Bytes from the start of a piece to element (i, j), j / 16 <= i / 16. The 16-column step s = j / 16 holds rows 16 s to
// 63 as two columns of 8 x 16-byte core matrices (the tensor core's unswizzled K-major form), so the blocks above the
// diagonal are neither stored nor multiplied.
__host__ __device__ constexpr int tri_start(int s) { return 2048 * s - 256 * s * (s - 1); }
__host__ __device__ constexpr int tri_offset(int i, int j) {
  const int s = j / 16, rows = kC - 16 * s;
  return tri_start(s) + (j % 16 / 8) * rows * 16 + (i - 16 * s) * 16 + (j % 8) * 2;
}

// Request r of work item w: items of request r start at tok_start[r] / 64 + r, which leaves each at least the
// ceil(tokens / 64) it needs. At most T / 64 + R items in all.
__device__ __forceinline__ int first_item(const GdnArgs& a, int r) { return a.tok_start[r] / kC + r; }

__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(x0, x1);
  lo = pack_bf16x2(x0 - __uint_as_float(hi << 16), x1 - __uint_as_float(hi & 0xffff0000u));
}

// as split2, and what it leaves
__device__ __forceinline__ void split3(float x0, float x1, uint32_t& hi, uint32_t& lo, uint32_t& rest) {
  hi = pack_bf16x2(x0, x1);
  x0 -= __uint_as_float(hi << 16), x1 -= __uint_as_float(hi & 0xffff0000u);
  lo = pack_bf16x2(x0, x1);
  rest = pack_bf16x2(x0 - __uint_as_float(lo << 16), x1 - __uint_as_float(lo & 0xffff0000u));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// D += A B in fp32 to about 2^-21: each operand as two tf32 parts, the product of the two small ones left out
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_split(float (&d)[4], const float (&a)[4], const float (&b)[2]) {
  uint32_t ah[4], al[4], bh[2], bl[2];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    ah[e] = __float_as_uint(a[e]) & 0xffffe000u;
    al[e] = __float_as_uint(a[e] - __uint_as_float(ah[e]));
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    bh[e] = __float_as_uint(b[e]) & 0xffffe000u;
    bl[e] = __float_as_uint(b[e] - __uint_as_float(bh[e]));
  }
  mma_tf32(d, al, bh);
  mma_tf32(d, ah, bl);
  mma_tf32(d, ah, bh);
}

constexpr int kPrepRow = kDim + 8;     // bf16 elements of a padded shared row: ldmatrix's eight rows miss each other's banks
constexpr int kBlkRow = 20;            // floats of a padded row of a 16 x 16 block
constexpr int kWRow = 12;
struct PrepSmem {
  union {
    struct {
      __nv_bfloat16 k[kC][kPrepRow], q[kC][kPrepRow];
    } in;
    struct {
      float blk[10][16][kBlkRow];      // the blocks on and below the diagonal: L, then (I + L)^-1 in its place
      float w[4][32][kWRow];           // each warp's 8 columns of a product
    } inv;
  };
  float bh[kC], bl[kC];                // b / ln 2 as the sum of two floats: differences of far-down sums keep their digits
  float rk[kC], rq[kC], beta[kC];
};
__host__ __device__ constexpr int blk_of(int bi, int bj) { return bi * (bi + 1) / 2 + bj; }

// Bound: instruction issue (7500 warp instructions an item and head, half of them ALU; DRAM at a fifth). Measured: 9728
// items x heads in 140 us, 1024 in 25 us (one head a CTA; 96 instead of 128 registers: 145 and 30). Forward substitution of
// all 64 rows by one thread a column took 330 us: 2600 unrolled instructions, fetched anew by every CTA.
// One CTA per (work item, `heads` value heads of one key head). The Gram matrices come from mma.sync and stay in its
// registers; each head's P and factors go from there to memory (a warp's 4-byte stores fill 128 bytes). (I + L)^-1 by
// blocks of 16: the diagonal ones by forward substitution, one column per thread, then 16 -> 32 -> 64 by
// T_BA = -T_BB (L_BA T_AA). Each entry is a true entry of the inverse on the way (no powers of L, which can grow where
// keys repeat).
__global__ void __launch_bounds__(128, 4) gdn_prep_kernel(const GdnArgs a, uint8_t* __restrict__ items, int heads) {
  __shared__ __align__(128) PrepSmem s;
  const int w = blockIdx.x, hk = blockIdx.y * heads / (a.HV / a.HK);
  // the chain's CTAs may take the SMs that this grid leaves; they wait for its end before they read an item
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  int lo = 0, hi = a.R - 1;            // the last request whose items start at or before w
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first_item(a, mid) <= w) lo = mid;
    else hi = mid - 1;
  }
  int t0, t1, slot;
  if (!request(a, lo, t0, t1, slot) || w < first_item(a, lo)) return;
  t0 += (w - first_item(a, lo)) * kC;
  const int n = min(kC, t1 - t0);
  if (n <= 0) return;

  // ---- q and k rows (zeros past the request's end) ----
#pragma unroll
  for (int x0 = 0; x0 < kC * 16; x0 += 128) {
    const int row = (x0 + tid) >> 4, c = (tid & 15) * 8;
    uint4 kv = make_uint4(0, 0, 0, 0), qv = kv;
    if (row < n) {
      kv = *reinterpret_cast<const uint4*>(a.k + (int64_t)(t0 + row) * a.k_t + hk * a.k_h + c);
      qv = *reinterpret_cast<const uint4*>(a.q + (int64_t)(t0 + row) * a.q_t + hk * a.q_h + c);
    }
    *reinterpret_cast<uint4*>(&s.in.k[row][c]) = kv;
    *reinterpret_cast<uint4*>(&s.in.q[row][c]) = qv;
  }
  __syncthreads();
  {
    const int row = tid & 63;
    const uint4* src = reinterpret_cast<const uint4*>(tid < 64 ? s.in.k[row] : s.in.q[row]);
    float ss = 0.f, s2 = 0.f;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const uint4 u = src[c];
      const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack_bf16x2(x[e]);
        ss = fmaf(f.x, f.x, ss);
        s2 = fmaf(f.y, f.y, s2);
      }
    }
    (tid < 64 ? s.rk : s.rq)[row] = rsqrtf(ss + s2 + 1e-6f) * (tid < 64 ? 1.f : a.scale);
  }

  // ---- Gram matrices k k^T and q k^T: warp w has rows 16 w .. 16 w + 15, columns up to the diagonal block ----
  float kk[8][4], qk[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) kk[j][e] = qk[j][e] = 0.f;
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    uint32_t ak[4], aq[4];
    const int ar = warp * 16 + (lane & 15), ac = ks * 16 + (lane >> 4) * 8;
    ldmatrix_x4(ak, smem_u32(&s.in.k[ar][ac]));
    ldmatrix_x4(aq, smem_u32(&s.in.q[ar][ac]));
#pragma unroll
    for (int j = 0; j < 4; ++j) {        // two column tiles of 8 at a time
      if (j <= warp) {
        uint32_t b[4];
        ldmatrix_x4(b, smem_u32(&s.in.k[j * 16 + (lane >> 4) * 8 + (lane & 7)][ks * 16 + (lane >> 3 & 1) * 8]));
        mma_bf16(kk[2 * j], ak, b[0], b[1]);
        mma_bf16(kk[2 * j + 1], ak, b[2], b[3]);
        mma_bf16(qk[2 * j], aq, b[0], b[1]);
        mma_bf16(qk[2 * j + 1], aq, b[2], b[3]);
      }
    }
  }

  // a head's gates and betas: tokens 2 l and 2 l + 1 in lane l of warp 0 and of warp 1, loaded a head ahead
  float in0 = 0.f, in1 = 0.f;
  auto fetch = [&](int h) {
    const float* src = warp == 0 ? a.g : a.beta;
    if (warp < 2) {
      in0 = 2 * lane < n ? src[(int64_t)(t0 + 2 * lane) * a.HV + h] : 0.f;
      in1 = 2 * lane + 1 < n ? src[(int64_t)(t0 + 2 * lane + 1) * a.HV + h] : 0.f;
    }
  };
  fetch(blockIdx.y * heads);
  for (int hh = 0; hh < heads; ++hh) {
    const int h = blockIdx.y * heads + hh;
    uint8_t* item = items + ((int64_t)w * a.HV + h) * kItemBytes;
    // ---- the head's sums of g and betas ----
    if (warp == 0) {
      // e^-1e6 is 0 as e^-inf is, and its sums can be subtracted
      auto gate = [](float x) -> double { return x < -1e6f ? -1e6f : x; };
      double b0 = gate(in0);
      const double b1 = b0 + gate(in1);
      double inc = b1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      b0 += inc - b1;
      b0 *= kLog2e;
      inc *= kLog2e;
      s.bh[2 * lane] = (float)b0, s.bl[2 * lane] = (float)(b0 - (float)b0);
      s.bh[2 * lane + 1] = (float)inc, s.bl[2 * lane + 1] = (float)(inc - (float)inc);
    } else if (warp == 1) {
      s.beta[2 * lane] = in0, s.beta[2 * lane + 1] = in1;
    }
    if (hh + 1 < heads) fetch(h + 1);
    __syncthreads();     // the blocks take the place of k and q (or of the last head's blocks); the factors are complete
    float* vec = reinterpret_cast<float*>(item + 4 * kTri);
    if (tid < kC) {
      const float e = exp2_approx(s.bh[tid] + s.bl[tid]), last = s.bh[kC - 1], lastl = s.bl[kC - 1];
      vec[tid] = s.beta[tid];
      vec[kC + tid] = s.beta[tid] * e * s.rk[tid];
      vec[2 * kC + tid] = exp2_approx((last - s.bh[tid]) + (lastl - s.bl[tid])) * s.rk[tid];
      vec[3 * kC + tid] = e * s.rq[tid];
      if (tid < 16) vec[4 * kC + tid] = tid == 0 ? exp2_approx(last + lastl) : 0.f;
    }
#pragma unroll
    for (int e2 = 0; e2 < 2; ++e2) {
      const int i = warp * 16 + g + 8 * e2;
      const float bhi = s.bh[i], bli = s.bl[i], fk = s.beta[i] * s.rk[i], fq = s.rq[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j <= 2 * warp + 1) {
          const int c = j * 8 + t * 2;
          const float2 ch = *reinterpret_cast<const float2*>(&s.bh[c]), cl = *reinterpret_cast<const float2*>(&s.bl[c]);
          const float2 cr = *reinterpret_cast<const float2*>(&s.rk[c]);
          const float d0 = c <= i ? exp2_approx((bhi - ch.x) + (bli - cl.x)) * cr.x : 0.f;
          const float d1 = c < i ? exp2_approx((bhi - ch.y) + (bli - cl.y)) * cr.y : 0.f;
          const float l0 = c < i ? kk[j][2 * e2] * d0 * fk : 0.f, l1 = c + 1 < i ? kk[j][2 * e2 + 1] * d1 * fk : 0.f;
          *reinterpret_cast<float2*>(&s.inv.blk[blk_of(warp, j >> 1)][i & 15][c & 15]) = make_float2(l0, l1);
          uint32_t ph, pl;
          split2(qk[j][2 * e2] * d0 * fq, qk[j][2 * e2 + 1] * d1 * fq, ph, pl);
          *reinterpret_cast<uint32_t*>(item + 2 * kTri + tri_offset(i, c)) = ph;
          *reinterpret_cast<uint32_t*>(item + 3 * kTri + tri_offset(i, c)) = pl;
        }
      }
    }
    __syncwarp();
    // ---- diagonal blocks: warp w has block w, lane j < 16 column j ----
    float (*D)[kBlkRow] = s.inv.blk[blk_of(warp, warp)];
    {
      float x[16];
      const int col = lane & 15;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float l[16];
#pragma unroll
        for (int k = 0; k < i; k += 4) *reinterpret_cast<float4*>(&l[k]) = *reinterpret_cast<const float4*>(&D[i][k]);
        float a0 = i == col ? 1.f : 0.f, a1 = 0.f;
#pragma unroll
        for (int k = 0; k < i; k += 2) {
          a0 = fmaf(-l[k], x[k], a0);
          if (k + 1 < i) a1 = fmaf(-l[k + 1], x[k + 1], a1);
        }
        x[i] = a0 + a1;
      }
      __syncwarp();
      if (lane < 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) D[i][col] = x[i];
      }
    }
    __syncthreads();
    float (*W)[kWRow] = s.inv.w[warp];
    auto load_a = [&](float (&f)[4], const float (*b)[kBlkRow], int k0) {
      f[0] = b[g][k0 + t], f[1] = b[g + 8][k0 + t], f[2] = b[g][k0 + t + 4], f[3] = b[g + 8][k0 + t + 4];
    };
    // ---- 16 -> 32: warp w has pair w / 2 and columns 8 (w % 2) .. of its block ----
    {
      const int lo_b = (warp >> 1) * 2, c0 = (warp & 1) * 8;
      float (*BA)[kBlkRow] = s.inv.blk[blk_of(lo_b + 1, lo_b)];
      const float (*AA)[kBlkRow] = s.inv.blk[blk_of(lo_b, lo_b)], (*BB)[kBlkRow] = s.inv.blk[blk_of(lo_b + 1, lo_b + 1)];
      float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k0 = 0; k0 < 16; k0 += 8) {
        float fa[4], fb[2] = {AA[k0 + t][c0 + g], AA[k0 + t + 4][c0 + g]};
        load_a(fa, BA, k0);
        mma_split(d, fa, fb);
      }
      W[g][2 * t] = d[0], W[g][2 * t + 1] = d[1], W[g + 8][2 * t] = d[2], W[g + 8][2 * t + 1] = d[3];
      __syncthreads();            // both halves of the pair have read L_BA
      float r[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k0 = 0; k0 < 16; k0 += 8) {
        float fa[4], fb[2] = {W[k0 + t][g], W[k0 + t + 4][g]};
        load_a(fa, BB, k0);
        mma_split(r, fa, fb);
      }
      BA[g][c0 + 2 * t] = -r[0], BA[g][c0 + 2 * t + 1] = -r[1], BA[g + 8][c0 + 2 * t] = -r[2], BA[g + 8][c0 + 2 * t + 1] = -r[3];
    }
    __syncthreads();
    // ---- 32 -> 64: warp w has columns 8 w .. 8 w + 7 ----
    {
      const int bc = warp >> 1, c0 = (warp & 1) * 8;
      float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int bk = 0; bk < 2; ++bk) {          // T_AA: block (0, 1) is zero
        if (bk < bc) continue;
        const float (*AA)[kBlkRow] = s.inv.blk[blk_of(bk, bc)];
#pragma unroll
        for (int k0 = 0; k0 < 16; k0 += 8) {
          const float fb[2] = {AA[k0 + t][c0 + g], AA[k0 + t + 4][c0 + g]};
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            float fa[4];
            load_a(fa, s.inv.blk[blk_of(2 + m, bk)], k0);
            mma_split(d[m], fa, fb);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
        W[16 * m + g][2 * t] = d[m][0], W[16 * m + g][2 * t + 1] = d[m][1], W[16 * m + g + 8][2 * t] = d[m][2], W[16 * m + g + 8][2 * t + 1] = d[m][3];
      __syncthreads();            // every warp has read L_BA
      float r[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int bk = 0; bk < 2; ++bk)
#pragma unroll
        for (int k0 = 0; k0 < 16; k0 += 8) {
          const float fb[2] = {W[16 * bk + k0 + t][g], W[16 * bk + k0 + t + 4][g]};
#pragma unroll
          for (int m = bk; m < 2; ++m) {        // T_BB: block (2, 3) is zero
            float fa[4];
            load_a(fa, s.inv.blk[blk_of(2 + m, 2 + bk)], k0);
            mma_split(r[m], fa, fb);
          }
        }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float (*BA)[kBlkRow] = s.inv.blk[blk_of(2 + m, bc)];
        BA[g][c0 + 2 * t] = -r[m][0], BA[g][c0 + 2 * t + 1] = -r[m][1];
        BA[g + 8][c0 + 2 * t] = -r[m][2], BA[g + 8][c0 + 2 * t + 1] = -r[m][3];
      }
    }
    __syncthreads();
    // ---- X pieces: eight neighbouring columns of a row at a time ----
    for (int x = tid; x < 320; x += 128) {
      const int bi_bj = x >> 5, row = x & 15, c = (x >> 4 & 1) * 8;
      const int bi = bi_bj < 1 ? 0 : bi_bj < 3 ? 1 : bi_bj < 6 ? 2 : 3, bj = bi_bj - bi * (bi + 1) / 2;
      float f[8];
      *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(&s.inv.blk[bi_bj][row][c]);
      *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(&s.inv.blk[bi_bj][row][c + 4]);
      uint32_t xh[4], xl[4];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (bi == bj && c + e == row) f[e] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) split2(f[2 * e], f[2 * e + 1], xh[e], xl[e]);
      const int at = tri_offset(bi * 16 + row, bj * 16 + c);
      *reinterpret_cast<uint4*>(item + at) = make_uint4(xh[0], xh[1], xh[2], xh[3]);
      *reinterpret_cast<uint4*>(item + kTri + at) = make_uint4(xl[0], xl[1], xl[2], xl[3]);
    }
    __syncthreads();     // the next head rewrites the blocks
  }
}

// ------------------------------------------------------------------------------------------------
// The chain: one CTA per (request, value head). Everything is transposed, so that TMEM lanes are the 128 value columns
// and the state never leaves the registers of the warps that own those lanes:
//   warp 0       loader: k, q (128-byte swizzle), v tiles and the chunk's item, kStages ahead
//   warp 1       TMEM owner; issues the products (warps 2 and 3 only fill the warpgroup)
//   warps 4-11   state warps: a thread has lane v and the key columns g * 64 + half * 32 + 0..31, g = 0, 1, of S
//   warps 12-15  output warps: 32 value columns and the chunk's 64 tokens each
// Token columns of TMEM (D1 to D4) are read in 16 x 256-bit fragments: a thread has 8 pairs of neighbouring tokens instead
// of 32, so its factors are a few 8-byte loads, v comes by transposing ldmatrix and the output leaves by stmatrix. (One
// lane per value column, every token: 1500 shared-memory wavefronts a chunk, which were the chain's bound.)
// Registers move from the first warpgroup to the state warps: 56 + 2 x 168 + 112 = 504 of the launch's 4 x 128.
// Per chunk (A operands in TMEM, B operands in shared memory, fp32 accumulators in TMEM):
//   D1 = S^T k^T                          S pieces written by the state warps
//   D2 = S^T q^T
//   R  = beta v - c1 D1                   state warps; c1 = beta e^b / |k|
//   D3 = R^T X^T, V' = R + D3             the identity part of (I + L)^-1 stays in fp32
//   DS = (V' c2)^T k, S = e^(b_C) S + DS  c2 = e^(b_C - b) / |k|
//   D4 = V'^T P^T, o = c3 D2 + D4         c3 = e^b scale / |q|
// The chain's latency bounds it: S -> D1 -> R -> D3 -> V' -> DS -> S. S goes through in two halves of 64 key columns, so
// that converting one overlaps the products of the other; D2 and the last chunk's D4 run while the state warps work.
// TMEM columns: DS, then S pieces 128 | D1, then R 64 | D2 64 | D3, then V' c2 pieces 64 | V' pieces 64 | D4 64 | third
// pieces of R 32 and of V' c2 32.
// A later product overwrites what an earlier one read: the tensor core runs one thread's products in order.
// The products multiply whole blocks of a chunk, zeros above the diagonals among them, and 0 * NaN is NaN: a NaN, an
// infinity or an overflow in one token would reach tokens ahead of it, which the recurrence leaves alone. Whatever is not
// finite in k, v, g, beta, X or S makes V' so, and through it the state, which stays so: if an element of the last state
// is not finite, the state warps take the request's tokens one by one from the state in memory, which is written only at
// the end. A q that is not finite reaches its own token's outputs alone.
// Measured: 2.62 us a chunk (128 chunks of 8 heads in 336 us), 2.2 of them before R and V' c2 got their third pieces; the
// tensor core is busy for 1.2 us of it (a product with A in TMEM costs N / 2 cycles), the state warps' conversions for 1.
// One waiting lane at the issuer, all waits with a timer, one lane per value column in every token: 3.9 us. Requests in
// order of length, the longest first: 250 instead of 260 us for 48 requests of 16384 tokens, lost again on ordering them.
// ------------------------------------------------------------------------------------------------
constexpr int kStages = 3;
constexpr int kChainThreads = 16 * 32;
constexpr uint32_t kColS = 0, kColD1 = 128, kColD2 = 192, kColD3 = 256, kColV = 320, kColD4 = 384,
                   kColR3 = 448, kColV3 = 480, kTmemCols = 512;
constexpr int kStageTx = 3 * kC * kDim * 2 + kItemBytes;

struct ChainStage {
  uint8_t k[2][kC * 128];       // key dimensions 0-63 and 64-127, 128 bytes per token
  uint8_t q[2][kC * 128];
  uint8_t v[2][kC * 128];       // value columns 0-63 and 64-127; later the chunk's output
  uint8_t item[(kItemBytes + 1023) / 1024 * 1024];
};
struct ChainSmem {
  ChainStage st[kStages];
  uint64_t full[kStages], ready[kStages], empty[kStages];
  uint64_t s_ready[2], r_ready, v_ready, p_ready, d2_read, o_read, o_staged;     // written by warps
  uint64_t d1_full, d2_full, d3_full, ds_full[2], o_full;                        // committed by the tensor core
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
  int redo;                      // an element of the new state is not finite
};

// MN-major SWIZZLE_128B operand: `lbo` bytes between 64-element blocks along N, 1024 between 8-row groups along K.
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t saddr, uint32_t lbo) {
  return static_cast<uint64_t>((saddr & 0x3FFFF) >> 4) | static_cast<uint64_t>(lbo >> 4) << 16 |
         static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
// Unswizzled K-major operand: core matrices of 8 rows x 16 bytes, `lbo` bytes apart along K, 128 along N.
__device__ __forceinline__ uint64_t sdesc_core(uint32_t saddr, uint32_t lbo) {
  return static_cast<uint64_t>((saddr & 0x3FFFF) >> 4) | static_cast<uint64_t>(lbo >> 4) << 16 |
         static_cast<uint64_t>(128 >> 4) << 32 | static_cast<uint64_t>(1) << 46;
}

template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ float2 lds2(uint32_t addr) {
  float2 f;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(f.x), "=f"(f.y) : "r"(addr));
  return f;
}
// 8 x 8 tiles of 16-bit elements, transposed on the way: of tile j (register j) lane l has row l / 4, columns 2 (l % 4)
// and 2 (l % 4) + 1, where the tile's columns are the eight rows in memory that lanes 8 j .. 8 j + 7 point at
__device__ __forceinline__ void ldmatrix_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void stmatrix_x4_t(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}
// 16 TMEM lanes x 32 columns: for m = 0..3 lane l gets columns 8 m + 2 (l % 4), + 1 of TMEM lanes l / 4 and l / 4 + 8
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// 16 TMEM lanes x 16 columns: for m = 0..3 lane l has column 4 m + l % 4 of TMEM lanes l / 4 and l / 4 + 8
__device__ __forceinline__ void tmem_st_frag(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
               "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}

// 1-D bulk copy of global memory into this CTA's shared memory, counted on `bar`
__device__ __forceinline__ void bulk_load(uint64_t* bar, void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Bounded wait, kept to a few instructions: the chain's loops have to stay in the instruction cache (with a timer and a
// status write at each of its 20 waits the kernel was 115 KB of code and 1.5 times as slow). False: the bound was
// reached or another warp gave up; give_up() then reports it once.
__device__ __forceinline__ bool mbar_wait_n(uint64_t* bar, uint32_t parity, volatile int* abort) {
#pragma unroll 1
  for (int i = 0; i < (1 << 20); ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort) return false;
  }
  return false;
}
// The same without going to sleep between tries, for the one warp whose every wait is on the chain.
__device__ __forceinline__ bool mbar_spin_n(uint64_t* bar, uint32_t parity, volatile int* abort) {
#pragma unroll 1
  for (int i = 0; i < (1 << 26); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((i & 255) == 255 && *abort) return false;
  }
  return false;
}
__device__ __noinline__ void give_up(int* status, int code, volatile int* abort) {
  if (!*abort) atomicCAS(status, 0, code);
  *abort = 1;
}

__global__ void __launch_bounds__(kChainThreads, 1)
    gdn_chain_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmQ,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, const GdnArgs a,
                     const uint8_t* __restrict__ items) {
  extern __shared__ uint8_t smem_raw[];
  ChainSmem& s = *reinterpret_cast<ChainSmem*>(smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
  const int warp = warp_id(), lane = lane_id();
  const int r = blockIdx.y, h = blockIdx.x, hk = h / (a.HV / a.HK);
  int t0, t1, slot;
  if (!request(a, r, t0, t1, slot) || t0 == t1) {         // uniform, before any barrier or TMEM use
    asm volatile("griddepcontrol.wait;" ::: "memory");    // what follows in the stream follows the first kernel too
    return;
  }
  const int nchunks = (t1 - t0 + kC - 1) / kC;
  const int tail = t1 - t0 - (nchunks - 1) * kC;           // tokens of the last chunk

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.ready[i], 1);
      mbar_init(&s.empty[i], 2);       // the tensor core, and the output's way out
    }
    for (uint64_t* b : {&s.s_ready[0], &s.s_ready[1], &s.r_ready, &s.v_ready, &s.p_ready}) mbar_init(b, 8);
    for (uint64_t* b : {&s.d2_read, &s.o_read, &s.o_staged}) mbar_init(b, 4);
    for (uint64_t* b : {&s.d1_full, &s.d2_full, &s.d3_full, &s.ds_full[0], &s.ds_full[1], &s.o_full, &s.mma_done}) mbar_init(b, 1);
    s.abort = s.redo = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  volatile int* abort = &s.abort;
  int* status = a.status;

  if (warp < 4) regs_down<56>();
  if (warp == 0) {
    // ---------------- loader ----------------
    const int item0 = first_item(a, r);
    asm volatile("griddepcontrol.wait;" ::: "memory");      // the items are complete
    int issued = 0;
    bool ok = true;
    for (int c = 0; c < nchunks; ++c) {
      const int st = c % kStages;
      const uint32_t ph = (c / kStages) & 1;
      ChainStage& g = s.st[st];
      if (!(ok = __all_sync(0xffffffffu, mbar_wait_n(&s.empty[st], ph ^ 1, abort)))) break;
      if (lane == 0) {
        const int t = t0 + c * kC;
        mbar_arrive_expect_tx(&s.full[st], kStageTx);
        tma_load_3d(&tmK, &s.full[st], g.k[0], 0, hk, t);
        tma_load_3d(&tmK, &s.full[st], g.k[1], 64, hk, t);
        bulk_load(&s.full[st], g.item, items + ((int64_t)(item0 + c) * a.HV + h) * kItemBytes, kItemBytes);
        tma_load_3d(&tmQ, &s.full[st], g.q[0], 0, hk, t);
        tma_load_3d(&tmQ, &s.full[st], g.q[1], 64, hk, t);
        tma_load_3d(&tmV, &s.full[st], g.v[0], 0, h, t);
        tma_load_3d(&tmV, &s.full[st], g.v[1], 64, h, t);
      }
      ++issued;
      if (c == nchunks - 1 && tail < kC) {
        // k rows past the request's end belong to another request: the update multiplies them by 0, so they have to
        // be finite
        if (!(ok = __all_sync(0xffffffffu, mbar_wait_n(&s.full[st], ph, abort)))) break;
        for (int x = lane; x < (kC - tail) * 16; x += 32)
          *reinterpret_cast<uint4*>(&g.k[x & 1][(tail + (x >> 4)) * 128 + (x >> 1 & 7) * 16]) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(&s.ready[st]);
    }
    if (!ok) give_up(status, kErrTimeoutProducer, abort);
    // the copies in flight land before the CTA may exit (bounded)
    volatile int never = 0;
    for (int c = max(0, issued - kStages); c < issued; ++c) mbar_wait_n(&s.full[c % kStages], (c / kStages) & 1, &never);
  } else if (warp == 1) {
    // ---------------- product issuer: the whole warp walks the loop, one elected lane issues. (A branch for one lane
    // around the loop keeps descriptors out of the uniform registers: 78 instead of 32 cycles a 64-column product.)
    constexpr uint32_t id64 = idesc_make(128, 64, 1), id64mn = id64 | (1u << 16);
    auto wait = [&](uint64_t* bar, uint32_t ph) {
      if (!__all_sync(0xffffffffu, mbar_spin_n(bar, ph, abort))) return false;
      tc_fence_after();
      return true;
    };
    auto commit = [&](uint64_t* bar) {
      if (elect_one()) umma_commit(bar);
    };
    // D[128 x 64] += S^T B^T over key dimensions 64 g .. 64 g + 63, B = k or q (K-major)
    auto state_product = [&](uint32_t d, const uint8_t* b, int g) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const uint64_t db = sdesc_sw128(smem_u32(b)) + 2 * ks;
        const uint32_t hi = tmem + kColS + g * 64 + (ks >> 1) * 32 + (ks & 1) * 8;
        if (elect_one()) umma_f16_ts(tmem + d, hi, db, id64, g > 0 || ks > 0);
        if (elect_one()) umma_f16_ts(tmem + d, hi + 16, db, id64, 1);
      }
    };
    // D[128 x 64] = A B^T, B lower triangular in two pieces; A in two pieces of 16 columns per 32 tokens, or three
    auto tri_product = [&](uint32_t d, uint32_t acol, const uint8_t* b, auto third) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const int rows = kC - 16 * ks;
        const uint32_t id = idesc_make(128, rows, 1), base = smem_u32(b) + tri_start(ks);
        const uint64_t hi = sdesc_core(base, rows * 16), lo = sdesc_core(base + kTri, rows * 16);
        const uint32_t ahi = tmem + acol + (ks >> 1) * 32 + (ks & 1) * 8, alo = ahi + 16, dd = tmem + d + 16 * ks;
        if (elect_one()) umma_f16_ts(dd, ahi, hi, id, ks > 0);
        if (elect_one()) umma_f16_ts(dd, alo, hi, id, 1);
        if (elect_one()) umma_f16_ts(dd, ahi, lo, id, 1);
        if constexpr (third.value) {
          if (elect_one()) umma_f16_ts(dd, alo, lo, id, 1);
          if (elect_one()) umma_f16_ts(dd, tmem + kColR3 + ks * 8, hi, id, 1);
        }
      }
    };
    // D[128 x 64] = (V' c2)^T k over the chunk's tokens, key dimensions 64 b .. 64 b + 63 (k MN-major)
    auto state_update = [&](ChainStage& g, int b) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const uint64_t db = sdesc_mn(smem_u32(g.k[b]) + ks * 2048, kC * 128);
        const uint32_t ahi = tmem + kColD3 + (ks >> 1) * 32 + (ks & 1) * 8;
        if (elect_one()) umma_f16_ts(tmem + kColS + 64 * b, ahi, db, id64mn, ks > 0);
        if (elect_one()) umma_f16_ts(tmem + kColS + 64 * b, ahi + 16, db, id64mn, 1);
        if (elect_one()) umma_f16_ts(tmem + kColS + 64 * b, tmem + kColV3 + ks * 8, db, id64mn, 1);
      }
      commit(&s.ds_full[b]);
    };
    auto output_product = [&](int c) {               // D4 of chunk c, the last use of its tiles
      if (!wait(&s.p_ready, c & 1) || (c > 0 && !wait(&s.o_read, (c & 1) ^ 1))) return false;
      tri_product(kColD4, kColV, s.st[c % kStages].item + 2 * kTri, std::false_type{});
      commit(&s.o_full);
      commit(&s.empty[c % kStages]);
      return true;
    };
    int c = 0;
    for (; c < nchunks; ++c) {
      const int st = c % kStages;
      const uint32_t ph = c & 1;
      ChainStage& g = s.st[st];
      if (c == 0 && (!wait(&s.full[0], 0) || !wait(&s.ready[0], 0))) break;
      if (!wait(&s.s_ready[0], ph)) break;
      state_product(kColD1, g.k[0], 0);
      if (!wait(&s.s_ready[1], ph)) break;
      state_product(kColD1, g.k[1], 1);
      commit(&s.d1_full);
      if (c > 0 && (!output_product(c - 1) || !wait(&s.d2_read, ph ^ 1))) break;
      state_product(kColD2, g.q[0], 0);
      if (!wait(&s.r_ready, ph)) break;
      tri_product(kColD3, kColD1, g.item, std::true_type{});
      commit(&s.d3_full);
      state_product(kColD2, g.q[1], 1);
      commit(&s.d2_full);
      if (c + 1 < nchunks) {                             // the next chunk's tiles, while there is time
        const int nst = (c + 1) % kStages;
        const uint32_t nph = ((c + 1) / kStages) & 1;
        if (!wait(&s.full[nst], nph) || !wait(&s.ready[nst], nph)) break;
      }
      if (!wait(&s.v_ready, ph)) break;
      state_update(g, 0);
      state_update(g, 1);
    }
    if (c == nchunks && !output_product(nchunks - 1)) --c;
    if (c < nchunks) give_up(status, kErrTimeoutMma, abort);
    commit(&s.mma_done);
    volatile int never = 0;
    mbar_wait_n(&s.mma_done, 0, &never);
  } else if (warp >= 4 && warp < 12) {
    // ---------------- state warps ----------------
    regs_up<168>();
    const int half = (warp - 4) >> 2, quad = warp & 3, v = quad * 32 + lane;
    const uint32_t tl = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    float* gS = a.state + (((int64_t)slot * a.HV + h) * kDim + half * 32) * kDim + v;
    float S[64];
#pragma unroll
    for (int j = 0; j < 64; ++j) S[j] = gS[((j >> 5) * 64 + (j & 31)) * kDim];
    // 16 floats -> two bf16 pieces of 8 TMEM columns each
    auto store_pieces = [&](uint32_t hi_col, uint32_t lo_col, const float* x) {
      uint32_t hi[8], lo[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) split2(x[2 * e], x[2 * e + 1], hi[e], lo[e]);
      tmem_st8(tl + hi_col, hi);
      tmem_st8(tl + lo_col, lo);
    };
    // 16 value columns x this half's 32 tokens -> two bf16 pieces of 16 TMEM columns each
    auto store_tokens = [&](int u, uint32_t col, const float (&x)[4][4]) {
      uint32_t hi[8], lo[8];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        split2(x[m][0], x[m][1], hi[2 * m], lo[2 * m]);
        split2(x[m][2], x[m][3], hi[2 * m + 1], lo[2 * m + 1]);
      }
      tmem_st_frag(tl + (u << 20) + col + half * 32, hi);
      tmem_st_frag(tl + (u << 20) + col + half * 32 + 16, lo);
    };
    // the same in three pieces, the third at `col3`
    auto store_tokens3 = [&](int u, uint32_t col, uint32_t col3, const float (&x)[4][4]) {
      uint32_t hi[8], lo[8], rest[8];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        split3(x[m][0], x[m][1], hi[2 * m], lo[2 * m], rest[2 * m]);
        split3(x[m][2], x[m][3], hi[2 * m + 1], lo[2 * m + 1], rest[2 * m + 1]);
      }
      tmem_st_frag(tl + (u << 20) + col + half * 32, hi);
      tmem_st_frag(tl + (u << 20) + col + half * 32 + 16, lo);
      tmem_st_frag(tl + (u << 20) + col3 + half * 16, rest);
    };
    const int t = lane & 3;
    // v tile (token row % 8 = lane % 8, value columns quad * 32 + 8 (lane / 8) ..) of a group of eight tokens
    const int vc = quad * 4 + (lane >> 3);
    const uint32_t vtile = (vc >> 3) * kC * 128 + (lane & 7) * 128 + (((vc & 7) ^ (lane & 7)) << 4);
    auto store_state = [&](int g) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t col = kColS + g * 64 + half * 32 + u * 8;     // where this thread's part of DS was
        store_pieces(col, col + 16, S + 32 * g + 16 * u);
      }
    };
    auto hand_over = [&](uint64_t* bar) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto wait = [&](uint64_t* bar, uint32_t ph) {
      if (!__all_sync(0xffffffffu, mbar_wait_n(bar, ph, abort))) return false;
      tc_fence_after();
      return true;
    };
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      store_state(g);
      hand_over(&s.s_ready[g]);
    }
    // R[u][m]: tokens half * 32 + 8 m + 2 t, + 1 of value columns quad * 32 + 16 u + lane / 4 (first two) and + 8
    float R[2][4][4], decay = 0.f;
    float2 f[4];
    uint32_t vec = 0;
    uint32_t raw[4][4];                // v of the next chunk as it is in memory
    auto load_v = [&](int c) {
      const int st = c % kStages;
      if (!__all_sync(0xffffffffu, mbar_wait_n(&s.full[st], (c / kStages) & 1, abort))) return false;
#pragma unroll
      for (int m = 0; m < 4; ++m) ldmatrix_x4_t(raw[m], smem_u32(s.st[st].v) + vtile + (half * 32 + 8 * m) * 128);
      return true;
    };
    auto start_chunk = [&](int c) {    // R = beta v, f = c1
      vec = smem_u32(s.st[c % kStages].item) + 4 * kTri + (half * 32 + 2 * t) * 4;
#pragma unroll
      for (int m = 0; m < 4; ++m) f[m] = lds2(vec + m * 32);
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 y = unpack_bf16x2(raw[m][e]);
          R[e >> 1][m][(e & 1) * 2] = y.x * f[m].x;
          R[e >> 1][m][(e & 1) * 2 + 1] = y.y * f[m].y;
        }
#pragma unroll
      for (int m = 0; m < 4; ++m) f[m] = lds2(vec + kC * 4 + m * 32);
    };
    bool ok = load_v(0);
    for (int c = 0; ok && c < nchunks; ++c) {
      const int n = c == nchunks - 1 ? tail : kC;
      const uint32_t ph = c & 1;
      start_chunk(c);
      if (!(ok = wait(&s.d1_full, ph))) break;
      {
        uint32_t d[2][16];
#pragma unroll
        for (int u = 0; u < 2; ++u) tmem_ld_frag(tl + (u << 20) + kColD1 + half * 32, d[u]);
        tmem_wait_ld();
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              R[u][m][e] = fmaf(e & 1 ? -f[m].y : -f[m].x, __uint_as_float(d[u][4 * m + e]), R[u][m][e]);
      }
      if (n < kC) {                                // tokens past the request's end
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (half * 32 + 8 * m + 2 * t + (e & 1) >= n) R[u][m][e] = 0.f;
      }
      // every column of this half has been read before its pieces overwrite it
#pragma unroll
      for (int u = 0; u < 2; ++u) store_tokens3(u, kColD1, kColR3, R[u]);
      hand_over(&s.r_ready);

#pragma unroll
      for (int m = 0; m < 4; ++m) f[m] = lds2(vec + 2 * kC * 4 + m * 32);
      if (c + 1 < nchunks && !(ok = load_v(c + 1))) break;
      if (!(ok = wait(&s.d3_full, ph))) break;
      {
        uint32_t d[2][16];
#pragma unroll
        for (int u = 0; u < 2; ++u) tmem_ld_frag(tl + (u << 20) + kColD3 + half * 32, d[u]);
        tmem_wait_ld();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float x[4][4];
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              R[u][m][e] += __uint_as_float(d[u][4 * m + e]);
              x[m][e] = R[u][m][e] * (e & 1 ? f[m].y : f[m].x);
            }
          store_tokens3(u, kColD3, kColV3, x);
        }
      }
      hand_over(&s.v_ready);
      decay = lds2(vec + (4 * kC - half * 32 - 2 * t) * 4).x;
#pragma unroll
      for (int u = 0; u < 2; ++u) store_tokens(u, kColV, R[u]);
      hand_over(&s.p_ready);

#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (!(ok = wait(&s.ds_full[g], ph))) break;
        uint32_t d[32];
        tmem_ld32(tl + kColS + g * 64 + half * 32, d);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) S[32 * g + j] = fmaf(S[32 * g + j], decay, __uint_as_float(d[j]));
        if (c + 1 < nchunks) {
          store_state(g);
          hand_over(&s.s_ready[g]);
        }
      }
      if (!ok) break;
    }
    if (!ok) give_up(status, kErrTimeoutEpilogue, abort);
    float odd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 64; ++j) odd[j & 3] = fmaf(S[j], 0.f, odd[j & 3]);       // NaN if one is not finite
    if ((odd[0] + odd[1]) + (odd[2] + odd[3]) != 0.f) *static_cast<volatile int*>(&s.redo) = 1;
    asm volatile("bar.sync 1, 256;" ::: "memory");      // every state warp has looked
    const bool redo = *static_cast<volatile int*>(&s.redo);
    if (ok && !redo) {
#pragma unroll
      for (int j = 0; j < 64; ++j) gS[((j >> 5) * 64 + (j & 31)) * kDim] = S[j];
    }
    asm volatile("bar.sync 2, 384;" ::: "memory");      // the outputs are in memory; who gave up has said so
    // the stages' memory is free: every copy has landed and every product and store from it is complete
    if (__builtin_expect(redo && !*abort, 0))
      step_tokens(a, h, t0, t1, slot, threadIdx.x - 128, *reinterpret_cast<StepSmem*>(s.st),
                  [] { asm volatile("bar.sync 3, 256;" ::: "memory"); });
  } else if (warp >= 12) {
    // ---------------- output warps ----------------
    regs_down<112>();
    const int quad = warp & 3;
    const uint32_t tl = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    auto wait = [&](uint64_t* bar, uint32_t ph) {
      if (!__all_sync(0xffffffffu, mbar_wait_n(bar, ph, abort))) return false;
      tc_fence_after();
      return true;
    };
    auto arrive = [&](uint64_t* bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    const int vc = quad * 4 + (lane >> 3), t = lane & 3;
    const uint32_t vtile = (vc >> 3) * kC * 128 + (lane & 7) * 128 + (((vc & 7) ^ (lane & 7)) << 4);
    int c = 0;
    for (; c < nchunks; ++c) {
      const int st = c % kStages, n = c == nchunks - 1 ? tail : kC;
      const uint32_t ph = c & 1;
      uint32_t o[2][2][16];      // [32 tokens][16 value columns]
      if (!wait(&s.full[st], (c / kStages) & 1)) break;
      if (!wait(&s.d2_full, ph)) break;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int u = 0; u < 2; ++u) tmem_ld_frag(tl + (u << 20) + kColD2 + g * 32, o[g][u]);
      tmem_wait_ld();
      arrive(&s.d2_read);
      if (c > 0 && warp == 12) {                       // the last chunk's output has left shared memory
        if (lane == 0) {
          bulk_wait_read0();
          mbar_arrive(&s.empty[(c - 1) % kStages]);
        }
        __syncwarp();
      }
      if (!wait(&s.o_full, ph)) break;
      const uint32_t c3 = smem_u32(s.st[st].item) + 4 * kTri + (3 * kC + 2 * t) * 4;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t d[2][16];
        float2 f[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) tmem_ld_frag(tl + (u << 20) + kColD4 + g * 32, d[u]);
#pragma unroll
        for (int m = 0; m < 4; ++m) f[m] = lds2(c3 + (32 * g + 8 * m) * 4);
        tmem_wait_ld();
        if (g == 1) arrive(&s.o_read);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int u = e >> 1, k = 4 * m + (e & 1) * 2;
            x[e] = pack_bf16x2(fmaf(f[m].x, __uint_as_float(o[g][u][k]), __uint_as_float(d[u][k])),
                               fmaf(f[m].y, __uint_as_float(o[g][u][k + 1]), __uint_as_float(d[u][k + 1])));
          }
          // v has been read: its place takes the output, in the same swizzled form
          stmatrix_x4_t(smem_u32(s.st[st].v) + vtile + (32 * g + 8 * m) * 128, x);
        }
      }
      fence_proxy_async_smem();
      arrive(&s.o_staged);
      if (!wait(&s.o_staged, ph)) break;
      const int tok = t0 + c * kC;
      if (n == kC) {
        if (warp == 12 && lane == 0) {
          tma_store_3d(&tmO, s.st[st].v[0], 0, h, tok);
          tma_store_3d(&tmO, s.st[st].v[1], 64, h, tok);
          bulk_commit();
        }
      } else {                                         // the last rows are not this request's
        for (int x = (warp - 12) * 32 + lane; x < n * 16; x += 128) {
          const int row = x >> 4, cc = x & 15;
          const uint4 val = *reinterpret_cast<const uint4*>(&s.st[st].v[cc >> 3][row * 128 + (((cc & 7) ^ (row & 7)) << 4)]);
          *reinterpret_cast<uint4*>(a.out + ((int64_t)(tok + row) * a.HV + h) * kDim + cc * 8) = val;
        }
      }
    }
    if (c < nchunks) give_up(status, kErrTimeoutEpilogue, abort);
    if (warp == 12 && lane == 0) bulk_wait0();
    __syncwarp();
    asm volatile("bar.sync 2, 384;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
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
  auto head_stride = [](const torch::Tensor& t) { return t.size(1) == 1 ? kDim : t.stride(1); };   // one head: any stride
  auto rows16 = [&](const torch::Tensor& t) {   // what 16-byte loads and tensor maps need
    return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 && t.stride(0) % 8 == 0 && head_stride(t) % 8 == 0 &&
           t.stride(0) > 0 && head_stride(t) > 0;
  };
  const int64_t waves = (R * HV + 147) / 148, mean = waves == 1 ? kStepMeanOneWave : kStepMean;
  if ((T <= mean * R && T <= kStepsPerWave * waves) || !rows16(q) || !rows16(k) || !rows16(v) || !rows16(out)) {
    gdn_step_kernel<<<dim3((unsigned)R, (unsigned)HV), 256, 0, stream>>>(a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    return;
  }
  TORCH_CHECK(R < 65536, "at most 65535 requests");
  const int64_t n_items = T / kC + R;
  torch::Tensor items = torch::empty({n_items * HV * kItemBytes}, q.options().dtype(at::kByte));
  auto map = [&](const torch::Tensor& t, int64_t heads) {
    return make_tmap_3d(t.data_ptr(), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kDim, heads, T, head_stride(t) * 2, t.stride(0) * 2, 64, 1, kC,
                        CU_TENSOR_MAP_SWIZZLE_128B);
  };
  const CUtensorMap tk = map(k, HK), tq = map(q, HK), tv = map(v, HV), to = map(out, HV);
  int dev = 0;
  cudaGetDevice(&dev);
  static bool opted[64] = {};   // the opt-in belongs to each device's context
  TORCH_CHECK(dev < 64, "device index out of range");
  constexpr int chain_smem = sizeof(ChainSmem) + 1024;
  if (!opted[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(gdn_chain_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, chain_smem));
    opted[dev] = true;
  }
  uint8_t* it = items.data_ptr<uint8_t>();
  // value heads of one key head in turn share its loads and Gram matrices, where that leaves CTAs enough for the machine
  const int rep = (int)(HV / HK), heads = n_items * HK >= 4 * 148 ? rep : 1;
  gdn_prep_kernel<<<dim3((unsigned)n_items, (unsigned)(HV / heads)), 128, 0, stream>>>(a, it, heads);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  // The chain starts while the items are still being made: its set-up and first loads of the state need none. Everything
  // before the two kernels is complete by then (the first one is launched in order), and every CTA of the first has
  // started before one of the second takes an SM.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)HV, (unsigned)R);
  cfg.blockDim = dim3(kChainThreads);
  cfg.dynamicSmemBytes = chain_smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, gdn_chain_kernel, tk, tq, tv, to, a, (const uint8_t*)it));
}

}  // namespace phx
