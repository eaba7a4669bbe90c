// Paged KV cache held in 8 bits: append (with q/k-norm + RoPE on the way), decode attention, load.
//
// Cache of one layer: k, v e4m3 codes [pages, Hkv, P, 128] and k_scale, v_scale e8m0 powers of two
// [pages, Hkv, P], one per (token, head); byte e stands for 2^(e - 127), byte 255 for NaN.  A slot is
// page * P + offset.  One scale per token and head means that appending a token touches no byte of
// another token (the pages of a shared prefix stay as they are), and a power of two means that
// code * scale is exact in bf16, so every reader sees the same values.  No counterpart in the reference
// beyond its rollout engine's kv_cache_dtype option (axrl/configs.py RolloutWorkerConfig).
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"

namespace ax {
namespace kv8 {

constexpr int D = 128;

// The least power of two s with amax <= 448 s, as its e8m0 byte: amax = 1.m x 2^x, 448 = 1.75 x 2^8.
// `bits`: the largest |value| as raw bits (an unsigned maximum of these keeps infinities and NaN).
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
  const uint32_t x = bits >> 23;
  if (x == 255u) return 255u;  // not finite: the row stands for NaN
  if (bits == 0u) return 127u;
  const int e = (int)x - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(e, 1);
}
__device__ __forceinline__ float scale_value(uint32_t byte) { return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte ? byte << 23 : 0x400000u); }
// 1 / scale, 0 for a row that is not finite (its codes are 0).
__device__ __forceinline__ float inv_scale(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }

// Two floats to two e4m3 codes (a in the low byte), round to nearest even.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// Two e4m3 codes to two halves (exact).
__device__ __forceinline__ uint32_t to_f16x2(uint32_t codes) {
  uint32_t r;
  asm("{.reg .b16 t;\n cvt.u16.u32 t, %1;\n cvt.rn.f16x2.e4m3x2 %0, t;}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t codes) {
  const uint32_t h = to_f16x2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

struct Cache {
  uint8_t *k, *v, *ks, *vs;
  long pages;
  int Hkv, P;
};

// ----------------------------------------------------------------------------- append
// One quarter-warp per (token, head): lane l of 8 holds elements 8l .. 8l + 7 of both halves, so a
// rotation pair stays in one thread and every access is 16 bytes (codes: 8).  The four quarters of a
// warp take four heads at a time; the angles of the token are computed once per warp.
//   n = x rsqrt(mean x^2 + eps) w;  rotated by pos * inv_freq (angle reduced in 64 bits: at position
//   10^5 a 32-bit angle is off by 4e-3);  code = rne(x / scale), one rounding from the fp32 value.
__global__ void __launch_bounds__(256) append_k(const bf16* __restrict__ qkv, const bf16* __restrict__ qw, const bf16* __restrict__ kw,
                                                const int* __restrict__ pos, const float* __restrict__ inv_freq, bf16* __restrict__ q,
                                                bf16* __restrict__ ko, bf16* __restrict__ vo, int T, int nq, int nkv, float eps, Cache c,
                                                const int64_t* __restrict__ slots, int parts) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, l8 = lane & 7;
  const long warp = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (warp >= (long)T * parts) return;
  const int t = (int)(warp / parts), part = (int)(warp % parts);
  const int nh = nq + 2 * nkv;
  const int groups = (nh + 3) >> 2;  // of four heads
  const int g0 = (int)((long)groups * part / parts), g1 = (int)((long)groups * (part + 1) / parts);
  float cs[8], sn[8];
  {
    const double turns_per_pos = 0.15915494309189535;  // 1 / (2 pi)
    const double p = (double)pos[t] * turns_per_pos;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      double a = p * (double)inv_freq[8 * l8 + i];
      a -= rint(a);
      sincospif((float)(2.0 * a), &sn[i], &cs[i]);
    }
  }
  const long slot = slots[t];
  const bool live = slot >= 0 && slot < c.pages * c.P;
  const long page = live ? slot / c.P : 0, off = live ? slot % c.P : 0;
  for (int g = g0; g < g1; ++g) {
    const int h = g * 4 + (lane >> 3);
    const bool in = h < nh;
    const int hh = in ? h : nh - 1;
    const bf16* src = qkv + ((long)t * nh + hh) * D + 8 * l8;
    float a[8], b[8];
    load8(src, a);
    load8(src + 64, b);
    const bool isv = hh >= nq + nkv, isq = hh < nq;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!isv) {
      const float r = rsqrtf(ss / D + eps);
      const bf16* w = isq ? qw : kw;
      float wa[8], wb[8];
      load8(w + 8 * l8, wa);
      load8(w + 64 + 8 * l8, wb);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = a[i] * r * wa[i], y = b[i] * r * wb[i];
        a[i] = x * cs[i] - y * sn[i];
        b[i] = y * cs[i] + x * sn[i];
      }
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, max(__float_as_uint(fabsf(a[i])), __float_as_uint(fabsf(b[i]))));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!in) continue;
    if (isq) {
      bf16* dst = q + ((long)t * nq + hh) * D + 8 * l8;
      store8(dst, a);
      store8(dst + 64, b);
      continue;
    }
    const int hv = hh - nq - (isv ? nkv : 0);
    const uint32_t e = scale_byte(m);
    const float inv = inv_scale(e);
    uint32_t ca[2] = {0, 0}, cb[2] = {0, 0};
    if (e != 255u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ca[i >> 1] |= to_e4m3x2(a[2 * i] * inv, a[2 * i + 1] * inv) << (16 * (i & 1));
        cb[i >> 1] |= to_e4m3x2(b[2 * i] * inv, b[2 * i + 1] * inv) << (16 * (i & 1));
      }
    }
    if (live) {
      const long row = (page * c.Hkv + hv) * c.P + off;
      uint8_t* dst = (isv ? c.v : c.k) + row * D + 8 * l8;
      *reinterpret_cast<uint2*>(dst) = make_uint2(ca[0], ca[1]);
      *reinterpret_cast<uint2*>(dst + 64) = make_uint2(cb[0], cb[1]);
      if (l8 == 0) (isv ? c.vs : c.ks)[row] = (uint8_t)e;
    }
    if (ko != nullptr) {  // the values that the cache stands for
      const float s = scale_value(e);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = from_e4m3x2(ca[i >> 1] >> (16 * (i & 1))), y = from_e4m3x2(cb[i >> 1] >> (16 * (i & 1)));
        a[2 * i] = x.x * s, a[2 * i + 1] = x.y * s, b[2 * i] = y.x * s, b[2 * i + 1] = y.y * s;
      }
      bf16* dst = (isv ? vo : ko) + ((long)t * nkv + hv) * D + 8 * l8;
      store8(dst, a);
      store8(dst + 64, b);
    }
  }
}

// ----------------------------------------------------------------------------- load
// Rows of the cache as bf16: one thread per 16 codes of K or V; exact.
__global__ void __launch_bounds__(256) load_k(Cache c, const int64_t* __restrict__ slots, bf16* __restrict__ ko, bf16* __restrict__ vo, long T) {
  const long n = T * c.Hkv * 16;  // 8 chunks of 16 codes for K, then for V
  for (long i = blockIdx.x * (long)blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x) {
    const int ch = (int)(i & 7), isv = (int)(i >> 3) & 1;
    const long th = i >> 4;
    const int h = (int)(th % c.Hkv);
    const long t = th / c.Hkv;
    const long slot = slots[t];
    uint4 w = make_uint4(0, 0, 0, 0);
    float s = 0.f;
    if (slot >= 0 && slot < c.pages * c.P) {
      const long row = ((slot / c.P) * c.Hkv + h) * c.P + slot % c.P;
      w = *reinterpret_cast<const uint4*>((isv ? c.v : c.k) + row * D + ch * 16);
      s = scale_value((isv ? c.vs : c.ks)[row]);
    }
    bf16* dst = (isv ? vo : ko) + th * D + ch * 16;
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = from_e4m3x2(ws[2 * half + (j >> 1)] >> (16 * (j & 1)));
        f[2 * j] = x.x * s, f[2 * j + 1] = x.y * s;
      }
      store8(dst + 8 * half, f);
    }
  }
}

// ----------------------------------------------------------------------------- decode
// One CTA per (sequence, kv head); warp w takes tokens w, w + 8, ...; lane l holds dims 4l .. 4l + 3.
// Online softmax per warp and q head, merged across the warps at the end.
constexpr int DW = 8, MAXG = 16;

__global__ void __launch_bounds__(DW * 32) decode_k(const bf16* __restrict__ q, Cache c, const int* __restrict__ bt, const int* __restrict__ lens,
                                                    bf16* __restrict__ out, int Hq, int max_pages, float scale_log2) {
  __shared__ float sO[DW][D];
  __shared__ float sM[DW][MAXG], sL[DW][MAXG];
  const int b = blockIdx.x, hk = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = Hq / c.Hkv;
  const int len = (int)min((long)max(lens[b], 0), (long)max_pages * c.P);
  float qf[MAXG][4], acc[MAXG][4], m[MAXG], l[MAXG];
#pragma unroll
  for (int g = 0; g < MAXG; ++g) {
    m[g] = -INFINITY, l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      qf[g][i] = g < G ? __bfloat162float(q[((long)b * Hq + hk * G + g) * D + 4 * lane + i]) : 0.f;
      acc[g][i] = 0.f;
    }
  }
  for (int t = warp; t < len; t += DW) {
    const int page = bt[(long)b * max_pages + t / c.P];
    if (page < 0 || page >= c.pages) continue;  // no such page: its tokens are not seen
    const long row = ((long)page * c.Hkv + hk) * c.P + t % c.P;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(c.k + row * D + 4 * lane), vw = *reinterpret_cast<const uint32_t*>(c.v + row * D + 4 * lane);
    const float ks = scale_value(c.ks[row]) * scale_log2, vs = scale_value(c.vs[row]);
    const float2 k0 = from_e4m3x2(kw), k1 = from_e4m3x2(kw >> 16), v0 = from_e4m3x2(vw), v1 = from_e4m3x2(vw >> 16);
#pragma unroll
    for (int g = 0; g < MAXG; ++g) {
      if (g >= G) break;
      const float s = warp_sum(qf[g][0] * k0.x + qf[g][1] * k0.y + qf[g][2] * k1.x + qf[g][3] * k1.y) * ks;
      const float mn = fmaxf(m[g], s), al = m[g] == -INFINITY ? 0.f : exp2f(m[g] - mn), p = exp2f(s - mn);
      m[g] = mn;
      l[g] = l[g] * al + p;
      const float pv = p * vs;
      acc[g][0] = acc[g][0] * al + pv * v0.x, acc[g][1] = acc[g][1] * al + pv * v0.y;
      acc[g][2] = acc[g][2] * al + pv * v1.x, acc[g][3] = acc[g][3] * al + pv * v1.y;
    }
  }
#pragma unroll
  for (int g = 0; g < MAXG; ++g)
    if (lane == 0) sM[warp][g] = m[g], sL[warp][g] = l[g];
  __syncthreads();
#pragma unroll
  for (int g = 0; g < MAXG; ++g) {
    if (g >= G) break;
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < DW; ++w) M = fmaxf(M, sM[w][g]);
    for (int w = 0; w < DW; ++w) L += sM[w][g] == -INFINITY ? 0.f : sL[w][g] * exp2f(sM[w][g] - M);
    const float f = m[g] == -INFINITY ? 0.f : exp2f(m[g] - M);
#pragma unroll
    for (int i = 0; i < 4; ++i) sO[warp][4 * lane + i] = acc[g][i] * f;
    __syncthreads();
    if (threadIdx.x < D) {
      float o = 0.f;
      for (int w = 0; w < DW; ++w) o += sO[w][threadIdx.x];
      out[((long)b * Hq + hk * G + g) * D + threadIdx.x] = __float2bfloat16(L == 0.f ? 0.f : o / L);
    }
    __syncthreads();
  }
}

static Cache checked(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs) {
  AX_CHECK(k.is_cuda() && k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn, "fp8 cache: k, v e4m3 on a CUDA device");
  AX_CHECK(ks.scalar_type() == at::kFloat8_e8m0fnu && vs.scalar_type() == at::kFloat8_e8m0fnu, "fp8 cache: scales e8m0");
  AX_CHECK(k.dim() == 4 && k.size(3) == D && v.sizes() == k.sizes(), "fp8 cache: k, v (pages, Hkv, P, 128)");
  AX_CHECK(ks.sizes() == k.sizes().slice(0, 3) && vs.sizes() == ks.sizes(), "fp8 cache: scales (pages, Hkv, P)");
  AX_CHECK(k.is_contiguous() && v.is_contiguous() && ks.is_contiguous() && vs.is_contiguous(), "fp8 cache: contiguous tensors");
  AX_CHECK(v.device() == k.device() && ks.device() == k.device() && vs.device() == k.device(), "fp8 cache: one device");
  AX_CHECK((reinterpret_cast<uintptr_t>(k.data_ptr()) & 15) == 0 && (reinterpret_cast<uintptr_t>(v.data_ptr()) & 15) == 0, "fp8 cache: k, v start on a 16-byte boundary");
  return Cache{(uint8_t*)k.data_ptr(), (uint8_t*)v.data_ptr(), (uint8_t*)ks.data_ptr(), (uint8_t*)vs.data_ptr(), (long)k.size(0), (int)k.size(1), (int)k.size(2)};
}
static void aligned16(const at::Tensor& t, const char* name) {
  AX_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, name, " starts on a 16-byte boundary");
}

}  // namespace kv8

std::vector<at::Tensor> qknorm_rope_cache_fp8(at::Tensor qkv, at::Tensor qw, at::Tensor kw, at::Tensor pos, at::Tensor inv_freq, int64_t nq,
                                              int64_t nkv, double eps, at::Tensor k, at::Tensor v, at::Tensor ks, at::Tensor vs, at::Tensor slots,
                                              bool want_kv) {
  using namespace kv8;
  const Cache c = checked(k, v, ks, vs);
  const auto dev = k.device();
  AX_CHECK(nq >= 0 && nkv >= 1 && nkv == c.Hkv, "nkv must be the cache's head count");
  AX_CHECK(qkv.device() == dev && qkv.scalar_type() == at::kBFloat16 && qkv.dim() == 2 && qkv.is_contiguous() && qkv.size(1) == (nq + 2 * nkv) * D,
           "qkv: contiguous bf16 (T, (nq + 2 nkv) 128) on the cache's device");
  const int64_t T = qkv.size(0);
  AX_CHECK(T < (1LL << 31), "too many tokens");
  for (const at::Tensor* w : {&qw, &kw})
    AX_CHECK(w->device() == dev && w->scalar_type() == at::kBFloat16 && w->numel() == D && w->is_contiguous(), "norm weights: contiguous bf16 (128,) on the cache's device");
  AX_CHECK(pos.device() == dev && pos.scalar_type() == at::kInt && pos.numel() == T && pos.is_contiguous(), "pos: contiguous int32 (T,)");
  AX_CHECK(inv_freq.device() == dev && inv_freq.scalar_type() == at::kFloat && inv_freq.numel() == D / 2 && inv_freq.is_contiguous(), "inv_freq: contiguous fp32 (64,)");
  AX_CHECK(slots.device() == dev && slots.scalar_type() == at::kLong && slots.numel() == T && slots.is_contiguous(), "slots: contiguous int64 (T,)");
  aligned16(qkv, "qkv"), aligned16(qw, "q norm weight"), aligned16(kw, "k norm weight");
  const c10::cuda::CUDAGuard guard(dev);
  const auto opt = qkv.options();
  auto q = at::empty({T, nq, D}, opt);
  auto ko = at::empty({want_kv ? T : 0, nkv, D}, opt), vo = at::empty({want_kv ? T : 0, nkv, D}, opt);
  if (T == 0) return {q, ko, vo};
  const int groups = (int)((nq + 2 * nkv + 3) / 4);
  // warps per token: enough of them to fill the GPU when tokens are few
  const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(groups, (int64_t)num_sms() * 16 / T));
  const long warps = T * (long)parts;
  launch_pdl(append_k, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, stream(), (const bf16*)qkv.data_ptr(), (const bf16*)qw.data_ptr(),
             (const bf16*)kw.data_ptr(), (const int*)pos.data_ptr<int>(), (const float*)inv_freq.data_ptr<float>(), (bf16*)q.data_ptr(),
             (bf16*)(want_kv ? ko.data_ptr() : nullptr), (bf16*)(want_kv ? vo.data_ptr() : nullptr), (int)T, (int)nq, (int)nkv, (float)eps, c,
             (const int64_t*)slots.data_ptr<int64_t>(), parts);
  AX_LAUNCH_OK();
  return {q, ko, vo};
}

void gather_kv_fp8(at::Tensor k, at::Tensor v, at::Tensor ks, at::Tensor vs, at::Tensor slots, at::Tensor ko, at::Tensor vo) {
  using namespace kv8;
  const Cache c = checked(k, v, ks, vs);
  const auto dev = k.device();
  AX_CHECK(slots.device() == dev && slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.is_contiguous(), "slots: contiguous int64 (T,)");
  const long T = slots.numel();
  for (const at::Tensor* o : {&ko, &vo}) {
    AX_CHECK(o->device() == dev && o->scalar_type() == at::kBFloat16 && o->dim() == 3 && o->size(0) == T && o->size(1) == c.Hkv && o->size(2) == D && o->is_contiguous(),
             "outputs: contiguous bf16 (T, Hkv, 128) on the cache's device");
    aligned16(*o, "output");
  }
  if (T == 0 || c.Hkv == 0) return;
  const c10::cuda::CUDAGuard guard(dev);
  const long n = T * c.Hkv * 16;
  load_k<<<(unsigned)std::min<long>((n + 255) / 256, (long)num_sms() * 32), 256, 0, stream()>>>(c, slots.data_ptr<int64_t>(), (bf16*)ko.data_ptr(),
                                                                                               (bf16*)vo.data_ptr(), T);
  AX_LAUNCH_OK();
}

at::Tensor paged_decode_attn_fp8(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor ks, at::Tensor vs, at::Tensor block_table, at::Tensor seq_lens,
                                 double scale) {
  using namespace kv8;
  const Cache c = checked(k, v, ks, vs);
  const auto dev = k.device();
  AX_CHECK(q.device() == dev && q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.size(2) == D && q.is_contiguous(), "q: contiguous bf16 (B, Hq, 128) on the cache's device");
  const int64_t B = q.size(0), Hq = q.size(1);
  AX_CHECK(c.Hkv >= 1 && Hq >= 1 && Hq % c.Hkv == 0 && Hq / c.Hkv <= MAXG, "GQA group must be <= 16");
  AX_CHECK(block_table.device() == dev && block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == B && block_table.is_contiguous(),
           "block_table: contiguous int32 (B, pages)");
  AX_CHECK(seq_lens.device() == dev && seq_lens.scalar_type() == at::kInt && seq_lens.numel() == B && seq_lens.is_contiguous(), "seq_lens: contiguous int32 (B,)");
  AX_CHECK(c.P % 16 == 0 && c.P > 0, "page size must be a multiple of 16");
  aligned16(q, "q");
  const c10::cuda::CUDAGuard guard(dev);
  auto out = at::empty_like(q);
  if (B == 0) return out;
  decode_k<<<dim3((unsigned)B, (unsigned)c.Hkv), DW * 32, 0, stream()>>>((const bf16*)q.data_ptr(), c, block_table.data_ptr<int>(), seq_lens.data_ptr<int>(),
                                                                         (bf16*)out.data_ptr(), (int)Hq, (int)block_table.size(1),
                                                                         (float)(scale * 1.4426950408889634));
  AX_LAUNCH_OK();
  return out;
}

}  // namespace ax
