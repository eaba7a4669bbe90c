// Paged KV cache held in 8 bits: append (with q/k-norm + RoPE on the way), decode attention, load.
//
// Cache of one layer: k, v e4m3 codes [pages, Hkv, P, 128] and k_scale, v_scale e8m0 powers of two
// [pages, Hkv, P], one per (token, head); byte e stands for 2^(e - 127), byte 255 for NaN.  A slot is
// page * P + offset.  One scale per token and head means that appending a token touches no byte of
// another token (the pages of a shared prefix stay as they are), and a power of two means that
// code * scale is exact in bf16, so every reader sees the same values.  No counterpart in the reference
// beyond its rollout engine's kv_cache_dtype option (axrl/configs.py RolloutWorkerConfig).
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/zero.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda.h>

#include "common.cuh"
#include "tcgen05.cuh"

namespace ax {
namespace kv8 {

constexpr int D = 128;

// The least power of two s >= 2^-60 with amax <= 448 s, as its e8m0 byte: amax = 1.m x 2^x, 448 = 1.75 x 2^8.  The bound (values
// below 4e-16 lose bits, at most 2^-70 of error) keeps the scales of a sequence within what the decode's weights span.
// `bits`: the largest |value| as raw bits (an unsigned maximum of these keeps infinities and NaN).
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
  const uint32_t x = bits >> 23;
  if (x == 255u) return 255u;  // not finite: the row stands for NaN
  if (bits == 0u) return 127u;
  const int e = (int)x - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(e, 127 - 60);
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
//   n = x rsqrt(mean x^2 + eps) w;  rotated by pos * inv_freq;  code = rne(x / scale), one rounding from the fp32 value.
// Moves (nq + 2 nkv) 256 bytes a token in and nq 256 + nkv 258 (+ nkv 512) out; bound by that for many tokens.  A CTA of
// eight warps takes 8 / parts tokens, `parts` warps each.  Its threads first put the products of each token's 64 angles
// (reduced in 64 bits: at position 10^5 a 32-bit angle is off by 4e-3) with both norm weights into shared memory, once per
// token: a' = r (a wa cos - b wb sin), b' = r (b wb cos + a wa sin).  A warp works on four heads at a time, a quarter-warp
// each: lane l of 8 holds elements 8l .. 8l + 7 of both halves, so a rotation pair stays in one thread and every access is 16
// bytes (codes: 8); the next four heads are loaded before the current ones are computed.  16384 tokens of 32 q and 8 kv
// heads: one warp walking a token with its own angles 100 us, products in registers 113 us (14 warps an SM), this form 79 us,
// 84 % of the measured copy rate; 2049 tokens of 16 q and 8 kv heads 9.4 us (floor 5.8).
constexpr int AW = 8;  // warps

// Largest magnitude, a NaN if there is one (the sign of the result means nothing).
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__global__ void __launch_bounds__(AW * 32, 4) append_k(const bf16* __restrict__ qkv, const bf16* __restrict__ qw, const bf16* __restrict__ kw,
                                                       const int* __restrict__ pos, const float* __restrict__ inv_freq, bf16* __restrict__ q,
                                                       bf16* __restrict__ ko, bf16* __restrict__ vo, int T, int nq, int nkv, float eps, Cache c,
                                                       const int64_t* __restrict__ slots, int parts) {
  // [token][q, k][i][l] for pair 8 l + i; eight lanes read 128 consecutive bytes.  q: wa cos, wb sin, wb cos, wa sin.
  // k: wa, wb, cos, sin: a key is rounded to e4m3, whose borders turn a difference in the last bit into a whole code, so
  // keys are computed in the order of the definition, each factor rounded once.
  __shared__ float4 s_w[AW][2][8][8];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l8 = lane & 7, tokens = AW / parts;
  const int t0 = blockIdx.x * tokens;
  const int tt = warp / parts, part = warp % parts, t = t0 + tt;
  const int gq = (nq + 3) >> 2, groups = gq + ((2 * nkv + 3) >> 2);  // of four heads: q, then k and v
  const int g0 = groups * part / parts, g1 = groups * (part + 1) / parts;
  const bool any = t < T && g0 < g1;
  const bf16* src = qkv + (long)t * (nq + 2 * nkv) * D + 8 * l8;
  uint4 na = make_uint4(0, 0, 0, 0), nb = na;
  auto fetch = [&](int g) {
    const int h = 4 * (g < gq ? g : g - gq) + (lane >> 3);
    if (h < (g < gq ? nq : 2 * nkv)) {
      const bf16* at = src + (h + (g < gq ? 0 : nq)) * D;
      na = *reinterpret_cast<const uint4*>(at), nb = *reinterpret_cast<const uint4*>(at + 64);
    }
  };
  if (any) fetch(g0);
  const long slot = any ? slots[t] : -1;
  for (int i = threadIdx.x; i < tokens * (D / 2); i += AW * 32) {
    const int ti = i / (D / 2), f = i % (D / 2);
    if (t0 + ti < T) {
      double turns = (double)pos[t0 + ti] * 0.15915494309189535 * (double)inv_freq[f];  // 1 / (2 pi)
      turns = 2.0 * (turns - rint(turns));
      const float x = (float)turns, rest = (float)(turns - (double)x) * 3.14159265f;
      float s0, c0;
      sincospif(x, &s0, &c0);
      const float sn = fmaf(c0, rest, s0), cs = fmaf(-s0, rest, c0);  // what the rounding of x left out
      const float wa = __bfloat162float(qw[f]), wb = __bfloat162float(qw[f + 64]);
      s_w[ti][0][f & 7][f >> 3] = make_float4(wa * cs, wb * sn, wb * cs, wa * sn);
      s_w[ti][1][f & 7][f >> 3] = make_float4(__bfloat162float(kw[f]), __bfloat162float(kw[f + 64]), cs, sn);
    }
  }
  const bool live = slot >= 0 && slot < c.pages * c.P;
  const long row0 = live ? slot / c.P * c.Hkv * c.P + slot % c.P : 0;  // cache row of head 0
  __syncthreads();
  if (!any) return;
  for (int g = g0; g < g1; ++g) {
    const bool isq = g < gq;
    int h = 4 * (isq ? g : g - gq) + (lane >> 3);
    const bool in = h < (isq ? nq : 2 * nkv), isv = !isq && h >= nkv;
    if (isv) h -= nkv;
    float a[8], b[8];
    load8(reinterpret_cast<const bf16*>(&na), a);
    load8(reinterpret_cast<const bf16*>(&nb), b);
    if (g + 1 < g1) fetch(g + 1);
    if (!__all_sync(0xffffffffu, isv)) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss / D + eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 w = s_w[tt][isq ? 0 : 1][i][l8];
        float x = a[i] * r, y = b[i] * r;
        if (isq) {
          a[i] = x * w.x - y * w.y;
          b[i] = y * w.z + x * w.w;
        } else {
          x *= w.x, y *= w.y;
          const float ra = __fsub_rn(__fmul_rn(x, w.z), __fmul_rn(y, w.w)), rb = __fadd_rn(__fmul_rn(y, w.z), __fmul_rn(x, w.w));
          a[i] = isv ? a[i] : ra, b[i] = isv ? b[i] : rb;  // a group may hold keys and values
        }
      }
    }
    if (isq) {
      if (in) {
        bf16* dst = q + ((long)t * nq + h) * D + 8 * l8;
        store8(dst, a);
        store8(dst + 64, b);
      }
      continue;
    }
    float top = max_abs(a[0], b[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) top = max_abs(top, max_abs(a[i], b[i]));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) top = max_abs(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t m = __float_as_uint(top) & 0x7fffffffu;
    if (!in) continue;
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
      const long row = row0 + (long)h * c.P;
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
      bf16* dst = (isv ? vo : ko) + ((long)t * nkv + h) * D + 8 * l8;
      store8(dst, a);
      store8(dst + 64, b);
    }
  }
}

// ----------------------------------------------------------------------------- load
// Rows of the cache as bf16 (exact): 129 bytes in and 256 out for each of the 2 Hkv rows of a slot, bound by that.  A warp
// takes 16 rows (the rows of one slot with eight heads): lane i looks up row i, then two rows at a time are converted, 16
// lanes of 8 codes each, so that a store fills 512 bytes; all 16 rows are read before the first is written.  One thread per
// 16 codes, each looking up its own slot, took 395 us for 131072 slots of eight heads, this form 132 us, 94 % of the measured copy rate.
constexpr int LR = 16;

__global__ void __launch_bounds__(256) load_k(Cache c, const int64_t* __restrict__ slots, bf16* __restrict__ ko, bf16* __restrict__ vo, long rows) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long base = (((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5) * LR;  // rows: (slot, K or V, head)
  if (base >= rows) return;
  const long r = base + (lane & 15);
  const uint8_t* src = nullptr;  // nothing to read: zeros
  bf16* dst = nullptr;
  float scale = 0.f;
  if (r < rows) {
    const long t = r / (2 * c.Hkv);
    const int j = (int)(r - t * 2 * c.Hkv), isv = j >= c.Hkv, h = j - isv * c.Hkv;
    dst = (isv ? vo : ko) + (t * c.Hkv + h) * D;
    const long slot = slots[t];
    if (slot >= 0 && slot < c.pages * c.P) {
      const long page = slot / c.P, row = (page * c.Hkv + h) * c.P + (slot - page * c.P);
      src = (isv ? c.v : c.k) + row * D;
      scale = scale_value((isv ? c.vs : c.ks)[row]);
    }
  }
  uint2 w[LR / 2];
  const int l16 = lane & 15;
#pragma unroll
  for (int i = 0; i < LR / 2; ++i) {
    const uint8_t* p = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, (unsigned long long)src, 2 * i + (lane >> 4)));
    w[i] = p != nullptr ? *reinterpret_cast<const uint2*>(p + 8 * l16) : make_uint2(0, 0);
  }
#pragma unroll
  for (int i = 0; i < LR / 2; ++i) {
    bf16* d = reinterpret_cast<bf16*>(__shfl_sync(0xffffffffu, (unsigned long long)dst, 2 * i + (lane >> 4)));
    const float s = __shfl_sync(0xffffffffu, scale, 2 * i + (lane >> 4));
    const float2 x0 = from_e4m3x2(w[i].x), x1 = from_e4m3x2(w[i].x >> 16), x2 = from_e4m3x2(w[i].y), x3 = from_e4m3x2(w[i].y >> 16);
    const float f[8] = {x0.x * s, x0.y * s, x1.x * s, x1.y * s, x2.x * s, x2.y * s, x3.x * s, x3.y * s};
    if (d != nullptr) store8(d + 8 * l16, f);
  }
}

// ----------------------------------------------------------------------------- decode
// o = sum_t softmax_t(scale q.k_t) v_t with k_t = kc_t 2^{a_t}, v_t = vc_t 2^{e_t} (codes, exponents).
//
// Work: unit = 64 tokens of one (sequence, kv head).  The units of all (sequence, kv head) pairs in a row form
// one list, cut into contiguous ranges of equal cost, one per warp of the grid (one CTA per SM): every warp is busy equally
// long whatever the lengths are.  A pair that lies inside one range is finished by its warp; the others leave fp32
// partials in shared memory (at most two per warp), which the CTA, whose ranges are neighbours, joins at its end; what then
// lies in several CTAs (at most two partials each) is joined by merge_k.  While it streams a warp works alone: its own ring of
// 8 KB slots (K and V tiles in turn) filled by its own TMA loads (128-byte swizzle), no barrier with other warps.
//
// Both products are m16n8k16 with f16 operands and fp32 sums; f16 holds every e4m3 code exactly:
//   S^T (tokens x heads) = Kc Q^T,   O^T (dims x heads) += Vc^T P^T
// A lane gets four consecutive codes of a token row (ldmatrix) or of a column of V (its transposing byte form) in one
// register: two conversions make them the two halves of an A fragment, because the contraction index may be permuted as
// long as both operands agree.  P^T is the transpose (movmatrix) of the S^T fragment.  Rows of S^T map to tokens so
// that each ldmatrix phase meets eight tokens that differ mod 8: no bank conflicts on swizzled tiles.  Up to eight heads of a
// group fill the n = 8 columns; groups of 9 to 16 take two column tiles.  The e4m3 form of mma.sync needs no conversions in
// the source but is no faster here: measured 5.4 clk per 16 x 32 step on an SM with two 8-bit terms per head, against 6.3
// clk for the load, conversions and two products above, which serve twice the heads (256 short sequences with groups of
// eight: 56.5 us against 40.4).
//
// Softmax in the log2 domain on w_t = scale log2(e) q.k_t + e_t, the exponent of V folded in: P_t = 2^{w_t - max w + HEAD}
// rounds to f16 (2^-11, finer than bf16) and multiplies the codes themselves, and the normaliser is l = sum P_t 2^{-e_t} in
// fp32, unrounded. HEAD = 15 uses f16 up to 2^15: a weight is rounded in full down to 2^-29 of the largest and is off by at
// most 2^-40 of it below, so that a row whose codes are as small as codes get (2^-9 of 2^9) may have the largest weight and the
// others still keep what they add. A row of zeros adds nothing at any weight: it is weighed as if its scale were the smallest
// that append writes, 2^-60 (with its own it would set the maximum and push the rows that do add something out of f16: with one
// of 2^0, 8 above the others' scores, the outputs of 300 tokens of values of size 10^-3 were off by 35 % of the largest;
// telling such rows costs 0 to 1 % of the time). P itself leaves fp32 (and l) only where exponents of V in a sequence lie 100
// and more apart, which scales of at least 2^-60 do not below |v| = 10^14; l holds 10^6 rows of scales down to 2^-90. q rows
// are scaled by a power of two so that their largest is in [2^14, 2^15) and round to f16 exactly but for what is below 2^-28 of
// it.
constexpr int MAXG = 16, UNIT = 64, NW = 8, SLOTS = 2, TILE = UNIT * D;  // TILE: bytes of one slot
constexpr float HEAD = 15.f;
constexpr int MAXB = 2048, DIRECT_TOKENS = NW * UNIT;
constexpr int DEC_FIXED = NW * SLOTS * (TILE + UNIT + 8 + 4);
// Shared memory of a CTA: rings, scales, barriers, flags; q rows, partials of pairs that began before the warps' ranges (groups of
// up to eight heads; larger ones keep them in global memory while the ring is in use), their maxima and sums; cell prefix and
// lengths.
constexpr int dec_smem(int G, int B) { return 1024 + DEC_FIXED + NW * G * (D * 2 + (G <= 8 ? D * 4 : 0) + 16) + (2 * B + 1) * 4; }
static_assert(dec_smem(8, MAXB) <= 227 * 1024 - 256 && dec_smem(MAXG, MAXB) <= 227 * 1024 - 256, "shared memory");
static_assert(2 * MAXG * D * 4 <= SLOTS * TILE, "both partials of a warp fit its ring");
static_assert(DEC_FIXED % 16 == 0 && NW * SLOTS * (TILE + UNIT) % 8 == 0, "alignment of what follows");

__device__ int g_decode_err;  // first wait that gave up (0: none)

struct DecParams {
  const bf16* q;       // (B, Hq, 128)
  const int* bt;       // (B, max_pages)
  const int* lens;     // (B,)
  const uint8_t *ks, *vs;
  bf16* out;           // (B, Hq, 128)
  float* part_o;       // (CTAs, 2, G, 128): of the pair that began before the CTA's ranges, of the one that goes on behind them
  float2* part_ml;     // (CTAs, 2, G): max, sum
  float* part_w;       // (CTAs, NW, G, 128), groups above eight: the warps' first pairs that end before their ranges do
  long pages;
  int B, G, Hkv, P, max_pages, box;  // box: token rows of one TMA load, gcd(P, 64)
  float scale_log2;
  bool direct;         // one CTA per pair
};

// Bounded wait for a tile; records that it gave up.
__device__ __forceinline__ bool wait_tile(uint64_t* bar, uint32_t phase) {
  for (long it = 0; !tc::mbar_try_wait(bar, phase); ++it)
    if (it > tc::WAIT_LIMIT) {
      atomicCAS(&g_decode_err, 0, 1);
      return false;
    }
  return true;
}
// Costs are counted in cells: two for a unit and one for each pair (its q, its output; measured 2.4 to 2.8 us a unit and 1.0 us a
// pair, and 256 short sequences take 37.3 us with ranges of equal units, 35.3 us with equal cells).  Cell 0 of a pair is its own,
// unit u starts at cell 1 + 2 u, and a range does the units that start in it.  All ranges have the same even length, so as few
// as possible: with lengths that differ by a unit the longer ones end alone (two contexts of 100k, 20 and 21 units: 71.2 us,
// all 21: 69.3 us).  Two cells or more: a range inside a pair has a unit.
// The ranges are dealt to the CTAs evenly, neighbours together: `base` of them, one more for the first `extra` CTAs.
struct Ranges {
  int len, n, base, extra;
  __device__ Ranges(int cells, int ctas) {
    const int most = ctas * NW;
    len = max(((cells + most - 1) / most + 1) & ~1, 2);
    n = (cells + len - 1) / len;
    base = n / ctas, extra = n - base * ctas;
  }
  __device__ int lo(int r) const { return r * len; }
  __device__ int of(int x) const { return x / len; }
  __device__ int first(int cta) const { return cta * base + min(cta, extra); }
  __device__ int cta_of(int r) const { return r < extra * (base + 1) ? r / (base + 1) : extra + (r - extra * (base + 1)) / base; }
};
__device__ __forceinline__ int cells(int units) { return units > 0 ? 2 * units + 1 : 0; }

// Not volatile: the products may move behind later ldmatrix loads, which keep their order.
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four 8 x 16-byte matrices: the A fragment of 16 rows x 32 bytes.
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// Two 16 x 16-byte matrices, transposed: the A fragment of 16 columns x 32 rows.
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// Four codes as two pairs of halves.
__device__ __forceinline__ void halves(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{.reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void bulk_bytes(void* dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::s32(dst)), "l"(src), "r"(bytes), "r"(tc::s32(bar))
               : "memory");
}

// Four codes of row `lane` and four of row 32 + lane of a tile, each lane's from a bank of its own: 0 if one of the two rows may be
// a row of zeros (-0 is a zero too).
constexpr uint32_t MAGNITUDES = 0x7f7f7f7fu;
__device__ __forceinline__ uint32_t first_look(const char* tile, int lane) {
  const char* at = tile + lane * D + (lane & 7) * 16 + (lane >> 3) * 4;
  return min(*reinterpret_cast<const uint32_t*>(at) & MAGNITUDES, *reinterpret_cast<const uint32_t*>(at + 32 * D) & MAGNITUDES);
}
// The tile's rows of zeros, a bit a row.  All lanes of a warp; apart from the loop around it, which hardly ever comes here.
__device__ __noinline__ uint64_t zero_rows(const char* tile) {
  const int lane = threadIdx.x & 31;
  uint32_t a = 0, b = 0;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const uint4* at = reinterpret_cast<const uint4*>(tile + lane * D + ((i ^ lane) & 7) * 16);
    const uint4 x = at[0], y = at[32 * D / 16];
    a |= x.x | x.y | x.z | x.w, b |= y.x | y.y | y.z | y.w;
  }
  return __ballot_sync(0xffffffffu, (a & MAGNITUDES) == 0u) | (uint64_t)__ballot_sync(0xffffffffu, (b & MAGNITUDES) == 0u) << 32;
}

// Position of a warp's loads in its range.
struct Loader {
  int b, hk, u, U, len;  // unit that is loaded next
  int left;              // cells of the range from its start on; none left: the range is done
  int pi, off;           // this lane's chunk of that unit: index into the block table, token within the page
  int page;              // its page, fetched ahead; -1: nothing to load
};

struct Partial {  // of one head: lane l holds dims 4 l .. 4 l + 3
  float4 o;
  float m, l;
};
__device__ __forceinline__ Partial empty_partial() { return {make_float4(0, 0, 0, 0), -INFINITY, 0.f}; }
__device__ __forceinline__ Partial load_partial(const DecParams& p, int record, int lane) {
  const float2 ml = __ldcg(p.part_ml + record);
  return {__ldcg(reinterpret_cast<const float4*>(p.part_o + (long)record * D + 4 * lane)), ml.x, ml.y};
}
// The sum of N partials in the scale of the largest.
template <int N>
__device__ __forceinline__ Partial join(const Partial (&x)[N]) {
  Partial r = empty_partial();
#pragma unroll
  for (int k = 0; k < N; ++k) r.m = fmaxf(r.m, x[k].m);
  const float ref = r.m == -INFINITY ? 0.f : r.m;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float f = ex2(x[k].m - ref);
    r.l = fmaf(f, x[k].l, r.l);
    r.o.x = fmaf(f, x[k].o.x, r.o.x), r.o.y = fmaf(f, x[k].o.y, r.o.y), r.o.z = fmaf(f, x[k].o.z, r.o.z), r.o.w = fmaf(f, x[k].o.w, r.o.w);
  }
  return r;
}
__device__ __forceinline__ void store_output(bf16* dst, const Partial& x, int lane) {
  const float rl = x.l == 0.f ? 0.f : 1.f / x.l;
  *reinterpret_cast<bf162*>(dst + 4 * lane) = __floats2bfloat162_rn(x.o.x * rl, x.o.y * rl);
  *reinterpret_cast<bf162*>(dst + 4 * lane + 2) = __floats2bfloat162_rn(x.o.z * rl, x.o.w * rl);
}

// Cells of a kv head of the sequences before each (prefix[B]: of all), by all THREADS of the CTA; s_len: the lengths, where wanted.
template <int THREADS>
__device__ __forceinline__ void cell_prefix(const DecParams& p, int* prefix, int* s_len, int* s_warp) {
  const int per = (p.B + THREADS - 1) / THREADS, b0 = threadIdx.x * per, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int sum = 0;
  for (int i = b0; i < min(b0 + per, p.B); ++i) {
    const int n = (int)min((long)max(p.lens[i], 0), (long)p.max_pages * p.P);
    if (s_len != nullptr) s_len[i] = n;
    prefix[i] = cells((n + UNIT - 1) / UNIT);
    sum += prefix[i];
  }
  int x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int before = x - sum;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) before += w < warp ? s_warp[w] : 0;
  for (int i = b0; i < min(b0 + per, p.B); ++i) {
    const int n = prefix[i];
    prefix[i] = before;
    before += n;
  }
  if (threadIdx.x == THREADS - 1) prefix[p.B] = before;
  __syncthreads();
}
// The sequence whose cells of a kv head hold `pos`: the last b with prefix[b] <= pos.  All lanes of a warp.
__device__ __forceinline__ int sequence_of(const int* prefix, int B, int pos, int lane) {
  int lo = 0, n = B;  // b in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) >> 5, at = lo + lane * step;
    const int k = 31 - __clz(__ballot_sync(0xffffffffu, at < lo + n && prefix[min(at, B)] <= pos));
    n = min(step, lo + n - (lo + k * step));
    lo += k * step;
  }
  return lo;
}

// 192 registers a thread leave room for a CTA of merge_k on every SM, which waits there for this grid to end.
template <int NT>
__global__ void __maxnreg__(192) decode_k(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, DecParams p) {
  extern __shared__ char smem_raw[];
  char* sm = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  char* ring = sm + warp * SLOTS * TILE;
  uint8_t* sc = reinterpret_cast<uint8_t*>(sm + NW * SLOTS * TILE) + warp * SLOTS * UNIT;  // scale bytes of a slot's tokens
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + NW * SLOTS * (TILE + UNIT)) + warp * SLOTS;
  uchar4* meta = reinterpret_cast<uchar4*>(sm + NW * SLOTS * (TILE + UNIT + 8)) + warp * SLOTS;  // which chunks of a slot were loaded
  char* sq = sm + DEC_FIXED + warp * p.G * D * 2;  // q rows of the pair that is loaded next
  float* s_rec = reinterpret_cast<float*>(sm + DEC_FIXED + NW * p.G * D * 2);
  float2* s_ml = reinterpret_cast<float2*>(s_rec + (NT == 1 ? NW * p.G * D : 0));  // [warp][began before, goes on][head]
  int* prefix = reinterpret_cast<int*>(s_ml + NW * 2 * p.G);
  int* s_len = prefix + p.B + 1;
  __shared__ int s_warp[NW], s_head[NW], s_tail[NW], s_pair[NW];

  if (lane == 0) {
    for (int s = 0; s < SLOTS; ++s) tc::mbar_init(&full[s], UNIT / p.box);  // every loading lane arrives
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tv) : "memory");
  }
  {  // lengths and block table into L2, a hint that needs no order with earlier kernels: the first two of three dependent reads
    const long at = ((long)blockIdx.x * blockDim.x + threadIdx.x) * 128;
    if (at < p.B * 4L) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(p.lens) + at));
    if (at < (long)p.B * p.max_pages * 4) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(p.bt) + at));
  }
  pdl_wait();
  pdl_trigger();  // after the wait: merge_k reads the lengths before this grid ends
  int wpc = NW;  // ranges (warps) of a CTA
  int b = 0, hk = 0, u = 0, U = 0, len = 0, left = 0;  // unit that is worked on next, cells of the range from its start on
  auto next_pair = [&](int& b, int& hk, int& u, int& U, int& len) {
    u = 0;
    if (++hk < p.Hkv) return;
    hk = 0;
    do ++b;
    while (b < p.B - 1 && prefix[b + 1] == prefix[b]);
    if (b < p.B) U = (prefix[b + 1] - prefix[b]) / 2, len = s_len[b];
  };
  if (p.direct) {  // the pair's units dealt to the warps
    b = blockIdx.x / p.Hkv, hk = blockIdx.x % p.Hkv;
    len = (int)min((long)max(p.lens[b], 0), (long)p.max_pages * p.P);
    U = (len + UNIT - 1) / UNIT;
    const int each = (U + NW - 1) / NW;
    u = min(warp * each, U);
    left = 2 * (min(u + each, U) - u);
    if (U == 0)
      for (int i = threadIdx.x; i < p.G * D / 8; i += NW * 32) reinterpret_cast<uint4*>(p.out + (long)blockIdx.x * p.G * D)[i] = make_uint4(0, 0, 0, 0);
  } else {
    cell_prefix<NW * 32>(p, prefix, s_len, s_warp);
    const Ranges rg(prefix[p.B] * p.Hkv, gridDim.x);
    const int r = rg.first(blockIdx.x) + warp;
    wpc = rg.first(blockIdx.x + 1) - rg.first(blockIdx.x);
    if (warp < wpc) {
      const int x0 = rg.lo(r);
      b = sequence_of(prefix, p.B, x0 / p.Hkv, lane);
      const int pc = prefix[b + 1] - prefix[b], rem = x0 - prefix[b] * p.Hkv;
      U = pc / 2;
      hk = rem / pc;
      const int off = rem - hk * pc;
      u = off / 2;
      left = min(rg.lo(r + 1), prefix[p.B] * p.Hkv) - x0 - (1 + 2 * u - off);
      len = s_len[b];
      if (u == U) {  // the range starts in the second half of the last unit of a pair
        next_pair(b, hk, u, U, len);
        left -= 1;  // its own cell; the start of a unit U had been counted already
      }
    }
  }
  // lane `ch` < chunks loads the box of tokens [ch box, (ch + 1) box) of a unit
  const int chunks = UNIT / p.box;
  const bool loads = lane < chunks;
  const int pi0 = (unsigned)(lane * p.box) / (unsigned)p.P, off0 = lane * p.box - pi0 * p.P;
  auto fetch_page = [&](Loader& x) {
    x.page = -1;
    if (loads && x.u * UNIT + lane * p.box < x.len) {
      const int pg = p.bt[(long)x.b * p.max_pages + x.pi];
      x.page = pg < p.pages ? pg : -1;
    }
  };
  auto next_unit = [&](Loader& x) {
    x.left -= 2;
    if (++x.u < x.U) {
      x.off += UNIT;
      while (x.off >= p.P) x.off -= p.P, ++x.pi;
      return;
    }
    x.left -= 1;
    x.pi = pi0, x.off = off0;
    if (x.left > 0) next_pair(x.b, x.hk, x.u, x.U, x.len);
  };
  const unsigned t0 = (unsigned)u * UNIT + lane * p.box;
  Loader ld{b, hk, u, U, len, left, (int)(t0 / (unsigned)p.P), (int)(t0 % (unsigned)p.P), -1};
  if (left > 0) fetch_page(ld);
  int nj = 0, row = -1;     // next tile to load (even: K, odd: V of the same unit), its cache row
  bool new_pair = true;     // of `ld`: its q rows come with its K tile
  auto load_next = [&] {
    const bool is_k = (nj & 1) == 0;
    if (is_k) {
      if (ld.left <= 0) return;
      row = ld.page >= 0 ? (int)(((long)ld.page * p.Hkv + ld.hk) * p.P) + ld.off : -1;
    }
    const int s = nj % SLOTS;
    if (loads) {
      reinterpret_cast<uint8_t*>(&meta[s])[lane] = row >= 0;
      const int q_bytes = is_k && new_pair && lane == 0 ? p.G * D * 2 : 0;
      tc::mbar_expect_tx(&full[s], (row >= 0 ? p.box * (D + 1) : 0) + q_bytes);
      if (row >= 0) {
        tc::tma_2d(ring + s * TILE + lane * p.box * D, is_k ? &tk : &tv, 0, row, &full[s]);
        bulk_bytes(sc + s * UNIT + lane * p.box, (is_k ? p.ks : p.vs) + row, p.box, &full[s]);
      }
      if (q_bytes) bulk_bytes(sq, p.q + ((long)ld.b * p.Hkv + ld.hk) * p.G * D, q_bytes, &full[s]);
    }
    if (is_k) {
      next_unit(ld);
      if (ld.left > 0) {
        new_pair = ld.u == 0;
        fetch_page(ld);
      }
    }
    ++nj;
  };
  for (int i = 0; i < SLOTS; ++i) load_next();

  // row x of S^T is token x, row 8 + x token 8 + (x ^ 4) of 16
  const int tok_a = g, tok_b = 8 + (g ^ 4);
  uint32_t k_off[4], v_off;  // this lane's ldmatrix rows within a tile
  {
    const int x = lane & 7, tok = (lane >> 3 & 1) ? 8 + (x ^ 4) : x;
#pragma unroll
    for (int i = 0; i < 4; ++i) k_off[i] = tok * D + (((2 * i + (lane >> 4)) ^ (tok & 7)) << 4);
    const int y = (lane >> 1 & 6) + (lane & 1), tv16 = (lane >> 1 & 1) ? 8 + (y ^ 4) : y;  // rows of V in the order of P's fragment
    v_off = ((lane >> 4) * 16 + tv16) * D + ((tv16 & 7) << 4);
  }
  const uint32_t ring_a = tc::s32(ring);
  float acc[NT][8][4], m[NT][2], l[NT][2], qs[NT][2];  // columns 2c, 2c + 1 of a tile: heads 8 t + 2 c, + 1
  uint32_t qf[NT][16];
  bool fresh = true, begun_before = u > 0;  // the pair at the start of the range may have begun in an earlier one
  int j = 0, head = 0, tail = 0;  // a pair that began before this range has a partial (2: it ended before the range did); the pair that goes on behind it: 1 if it began before, 2 if in it
  while (left > 0) {
    const int sk = j % SLOTS, sv = (j + 1) % SLOTS;
    // --- scores of 64 tokens
    if (!__all_sync(0xffffffffu, wait_tile(&full[sk], (j / SLOTS) & 1))) break;
    if (fresh) {  // q columns of this pair: column g is head 8 t + g
      fresh = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int h = 8 * t + g;
        uint2 w[8];
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          w[k] = h < p.G ? *reinterpret_cast<const uint2*>(sq + h * D * 2 + 32 * k + 8 * c) : make_uint2(0, 0);
          top = max(top, max(max((w[k].x << 16) & 0x7fffffffu, w[k].x & 0x7fff0000u), max((w[k].y << 16) & 0x7fffffffu, w[k].y & 0x7fff0000u)));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^(141 - ex) takes the largest to [2^14, 2^15); a row that is not finite poisons its scores through the factor
        const uint32_t ex = top >> 23;
        const float down = ex < 15u ? 1.f : __uint_as_float((268u - min(ex, 254u)) << 23);
        const float up = ex == 255u ? __uint_as_float(0x7fffffffu) : p.scale_log2 * (ex < 15u ? 1.f : __uint_as_float((ex - 14u) << 23));
        qs[t][0] = __shfl_sync(0xffffffffu, up, 8 * c);  // column 2c
        qs[t][1] = __shfl_sync(0xffffffffu, up, 8 * c + 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          qf[t][2 * k] = pack_f16(__uint_as_float(w[k].x << 16) * down, __uint_as_float(w[k].x & 0xffff0000u) * down);
          qf[t][2 * k + 1] = pack_f16(__uint_as_float(w[k].y << 16) * down, __uint_as_float(w[k].y & 0xffff0000u) * down);
        }
        m[t][0] = m[t][1] = -INFINITY, l[t][0] = l[t][1] = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[t][d][0] = acc[t][d][1] = acc[t][d][2] = acc[t][d][3] = 0.f;
      }
    }
    const int nval = min(UNIT, len - u * UNIT);
    const uchar4 ld4 = meta[sk];
    const int loaded = ld4.x | (ld4.y & (chunks > 1)) << 1 | (chunks > 2 ? ld4.z << 2 | ld4.w << 3 : 0);
    const bool partial = nval < UNIT || __popc(loaded) < chunks;
    float s[NT][4][4];  // tokens tok_a, tok_b of 16 x the two columns
#pragma unroll
    for (int i16 = 0; i16 < 4; ++i16)
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t][i16][0] = s[t][i16][1] = s[t][i16][2] = s[t][i16][3] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t x[4][8];
#pragma unroll
      for (int i16 = 0; i16 < 4; ++i16) {
        uint32_t a[4];
        ldsm4(a, ring_a + sk * TILE + i16 * 16 * D + k_off[k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) halves(a[e], x[i16][2 * e], x[i16][2 * e + 1]);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i16 = 0; i16 < 4; ++i16)  // innermost: the four tiles' sums do not depend on each other
            mma_f16(s[t][i16], x[i16][4 * half], x[i16][4 * half + 2], x[i16][4 * half + 1], x[i16][4 * half + 3], qf[t][4 * k + 2 * half], qf[t][4 * k + 2 * half + 1]);
    }
#pragma unroll
    for (int i16 = 0; i16 < 4; ++i16) {
      const float ka = scale_value(sc[sk * UNIT + i16 * 16 + tok_a]), kb = scale_value(sc[sk * UNIT + i16 * 16 + tok_b]);
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t][i16][0] *= ka, s[t][i16][1] *= ka, s[t][i16][2] *= kb, s[t][i16][3] *= kb;
    }
    __syncwarp();
    load_next();
    // --- w = scale log2(e) q.k + e, and P = 2^{w - max w + HEAD}
    if (!__all_sync(0xffffffffu, wait_tile(&full[sv], ((j + 1) / SLOTS) & 1))) break;
    const uint32_t look = first_look(ring + sv * TILE, lane);
    uint64_t seen = ~0ull;  // tokens of the unit that count
    if (partial) {
      seen = 0;
      for (int k = 0; k < chunks; ++k)
        if (loaded >> k & 1) seen |= (p.box == 64 ? ~0ull : ((1ull << p.box) - 1)) << (k * p.box);
      if (nval < UNIT) seen &= (1ull << nval) - 1;
    }
    float inv[4][2];
#pragma unroll
    for (int i16 = 0; i16 < 4; ++i16)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const uint32_t byte = sc[sv * UNIT + i16 * 16 + (hh ? tok_b : tok_a)];
        const float e = byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(0x4b000000u + byte) - 8388735.f;  // byte - 127
        inv[i16][hh] = __uint_as_float((uint32_t)max((int)((254 - (int)byte) << 23), 0x400000));
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) s[t][i16][2 * hh + cc] = fmaf(s[t][i16][2 * hh + cc], qs[t][cc], e);
      }
    if (__any_sync(0xffffffffu, look == 0u)) {
      const uint64_t zero = zero_rows(ring + sv * TILE);
#pragma unroll
      for (int i16 = 0; i16 < 4; ++i16)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
          if (zero >> (i16 * 16 + (hh ? tok_b : tok_a)) & 1) {  // e becomes -60; a row that is not finite stays NaN
            const float to = (float)((int)(__float_as_uint(inv[i16][hh]) >> 23) - 127 - 60);
            inv[i16][hh] = 0x1p60f;
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t][i16][2 * hh] += to, s[t][i16][2 * hh + 1] += to;
          }
    }
    if (partial) {
#pragma unroll
      for (int i16 = 0; i16 < 4; ++i16)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
          if (!(seen >> (i16 * 16 + (hh ? tok_b : tok_a)) & 1)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t][i16][2 * hh] = s[t][i16][2 * hh + 1] = -INFINITY;
          }
    }
    uint32_t pf[NT][4][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float alpha[2], ref[2];
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        float mx = fmaxf(s[t][0][cc], s[t][0][2 + cc]);
#pragma unroll
        for (int i16 = 1; i16 < 4; ++i16) mx = fmaxf(mx, fmaxf(s[t][i16][cc], s[t][i16][2 + cc]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        // m: HEAD below the largest w, where the difference is exact to far less than the headroom above 2^15
        mx = fmaxf(m[t][cc], fabsf(mx) < 0x1p20f ? mx - HEAD : mx);
        ref[cc] = mx == -INFINITY ? 0.f : mx;  // nothing seen yet
        alpha[cc] = ex2(m[t][cc] - ref[cc]);
        m[t][cc] = mx;
        l[t][cc] *= alpha[cc];
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[t][d][0] *= alpha[0], acc[t][d][1] *= alpha[1], acc[t][d][2] *= alpha[0], acc[t][d][3] *= alpha[1];
      }
#pragma unroll
      for (int i16 = 0; i16 < 4; ++i16)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const float p0 = ex2(s[t][i16][2 * hh] - ref[0]), p1 = ex2(s[t][i16][2 * hh + 1] - ref[1]);
          l[t][0] = fmaf(p0, inv[i16][hh], l[t][0]);
          l[t][1] = fmaf(p1, inv[i16][hh], l[t][1]);
          pf[t][i16][hh] = transpose8x8(pack_f16(p0, p1));
        }
    }
    // --- outputs
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t keep[2] = {~0u, ~0u};
      if (partial) {  // what is not seen may hold a NaN code, and 0 x NaN is NaN
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int x = 2 * c + (e & 1), tok = k * 32 + half * 16 + (e >> 1 ? 8 + (x ^ 4) : x);
            if (!(seen >> tok & 1)) keep[half] &= ~(0xffu << (8 * e));
          }
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        uint32_t a[4], x[8];
        ldsm_t(a, (ring_a + sv * TILE + k * 32 * D + v_off) ^ (d << 4));
        if (partial) a[0] &= keep[0], a[1] &= keep[0], a[2] &= keep[1], a[3] &= keep[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) halves(a[e], x[2 * e], x[2 * e + 1]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma_f16(acc[t][d], x[0], x[2], x[1], x[3], pf[t][2 * k][0], pf[t][2 * k][1]);
          mma_f16(acc[t][d], x[4], x[6], x[5], x[7], pf[t][2 * k + 1][0], pf[t][2 * k + 1][1]);
        }
      }
    }
    __syncwarp();
    load_next();
    j += 2;
    // --- end of the pair, or of the range
    const bool ends = u == U - 1;
    left -= ends ? 3 : 2;
    if (ends || left <= 0) {
      const bool whole = ends && !begun_before;
      // at the end of the range the warp's ring is free: what goes on lies there, and behind it the large groups' first pair
      float* rec = reinterpret_cast<float*>(ring);
      if (begun_before) rec = NT == 1 ? s_rec + warp * p.G * D : left <= 0 ? rec + p.G * D : p.part_w + ((long)blockIdx.x * NW + warp) * p.G * D;
      float2* rec_ml = s_ml + (warp * 2 + !begun_before) * p.G;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          float sum = l[t][cc];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const int h = 8 * t + 2 * c + cc;
          if (h < p.G) {
            const float rl = sum == 0.f ? 0.f : 1.f / sum;
            bf16* dst = p.out + (((long)b * p.Hkv + hk) * p.G + h) * D + g;
            float* part = rec + h * D + g;
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              if (whole) dst[16 * d] = __float2bfloat16(acc[t][d][cc] * rl), dst[16 * d + 8] = __float2bfloat16(acc[t][d][2 + cc] * rl);
              else part[16 * d] = acc[t][d][cc], part[16 * d + 8] = acc[t][d][2 + cc];
            }
            if (!whole && g == 0) rec_ml[h] = make_float2(m[t][cc], sum);
          }
        }
      if (begun_before) head = left <= 0 ? 1 : 2;
      if (!ends) {
        tail = begun_before ? 1 : 2;
        if (lane == 0) s_pair[warp] = b * p.Hkv + hk;
      }
      fresh = true;
      begun_before = false;
    }
    if (++u == U && left > 0) next_pair(b, hk, u, U, len);
  }
  // after a wait that gave up: let the copies in flight land before the CTA's memory is released
  for (; j < nj; ++j) wait_tile(&full[j % SLOTS], (j / SLOTS) & 1);

  // Join the partials of pairs that lie in several ranges of this CTA: a warp takes a head and walks the ranges in order.
  if (NT == 2 && head == 2) {
    __syncwarp();
    const float4* from = reinterpret_cast<const float4*>(p.part_w + ((long)blockIdx.x * NW + warp) * p.G * D) + lane;
    float4* to = reinterpret_cast<float4*>(ring) + p.G * 32 + lane;
    float4 x[MAXG];
#pragma unroll
    for (int h = 0; h < MAXG; ++h)
      if (h < p.G) x[h] = __ldcg(from + 32 * h);
#pragma unroll
    for (int h = 0; h < MAXG; ++h)
      if (h < p.G) to[32 * h] = x[h];
  }
  if (lane == 0) s_head[warp] = head, s_tail[warp] = tail;
  __syncthreads();
  for (int h = warp; h < p.G; h += NW) {
    Partial y = empty_partial();
    int pair = -1, open = 0;  // the pair of y if it began in this CTA; y holds something
    auto record = [&](int w, int which) -> Partial {
      const char* ring_w = sm + w * SLOTS * TILE;
      const float4* rec = reinterpret_cast<const float4*>(which ? ring_w : NT == 1 ? reinterpret_cast<const char*>(s_rec + w * p.G * D) : ring_w + p.G * D * 4);
      const float2 ml = s_ml[(w * 2 + which) * p.G + h];
      return {rec[h * 32 + lane], ml.x, ml.y};
    };
    auto hand_on = [&](int which) {
      const int at = (blockIdx.x * 2 + which) * p.G + h;
      *reinterpret_cast<float4*>(p.part_o + (long)at * D + 4 * lane) = y.o;
      if (lane == 0) p.part_ml[at] = make_float2(y.m, y.l);
    };
#pragma unroll 1
    for (int w = 0; w < wpc; ++w) {
      if (s_head[w]) {
        const Partial two[2] = {y, record(w, 0)};
        y = join(two);
        open = 1;
        if (s_tail[w] != 1) {  // ends here
          if (pair >= 0) store_output(p.out + ((long)pair * p.G + h) * D, y, lane);
          else hand_on(0);
          y = empty_partial(), open = 0, pair = -1;
        }
      }
      if (s_tail[w] == 2) y = record(w, 1), open = 1, pair = s_pair[w];
    }
    if (open) hand_on(pair >= 0 ? 1 : 0);
  }
}

// The pairs that lie in several CTAs of decode_k: out = the joined partials of those CTAs; zeros for empty sequences.  CTA i looks
// for the pair that goes on behind CTA i before decode_k has ended.  The CTAs that a pair goes on behind share its heads;
// a CTA's MW warps are dealt to its heads and, where those are fewer, to stripes of the partials, whose loads are in flight
// together.  One warp walking the partials of all warps took 42 us for two contexts of 100k, CTAs of eight warps for every
// pair 6 us, and 5 us for 256 short sequences; this form 2 us.  With all heads left to the pair's first CTA, two sequences of
// 1943 tokens with two kv heads (31 CTAs a pair, 16 heads) took 23 us in all, shared 14
// (11.5 since the large groups' partials stay on the SM).
constexpr int MW = 8, MBATCH = 4;

__global__ void __launch_bounds__(MW * 32) merge_k(DecParams p) {
  extern __shared__ int prefix[];
  __shared__ int s_warp[MW];
  __shared__ float4 s_o[MW][32];
  __shared__ float2 s_ml[MW];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  cell_prefix<MW * 32>(p, prefix, nullptr, s_warp);  // decode_k lets this grid start only once the lengths are there
  const Ranges rg(prefix[p.B] * p.Hkv, gridDim.x);
  const int end = min(rg.lo(rg.first(blockIdx.x + 1)), prefix[p.B] * p.Hkv);  // of CTA i's cells
  int n = 0, i0 = 0;  // the pair that goes on lies in n CTAs from i0
  bf16* out = nullptr;
  if (end > 0 && end < prefix[p.B] * p.Hkv) {
    const int b = sequence_of(prefix, p.B, (end - 1) / p.Hkv, lane), pc = prefix[b + 1] - prefix[b];
    const int hk = (end - 1 - prefix[b] * p.Hkv) / pc, x0 = prefix[b] * p.Hkv + hk * pc + 1, last = x0 + pc - 3;
    if (x0 < end && last >= end) {
      i0 = rg.cta_of(rg.of(x0));
      n = rg.cta_of(rg.of(last)) - i0 + 1;
      out = p.out + ((long)b * p.Hkv + hk) * p.G * D;
    }
  }
  pdl_wait();
  for (int b = blockIdx.x; b < p.B; b += gridDim.x)
    if (prefix[b + 1] == prefix[b])
      for (int i = threadIdx.x; i < p.Hkv * p.G * D / 8; i += MW * 32) reinterpret_cast<uint4*>(p.out + (long)b * p.Hkv * p.G * D)[i] = make_uint4(0, 0, 0, 0);
  if (out == nullptr) return;
  // heads h0, h0 + n - 1, ... of the group: `mine` of them
  const int h0 = (int)blockIdx.x - i0, mine = h0 < p.G ? (p.G - 1 - h0) / (n - 1) + 1 : 0;
  if (mine == 0) return;
  const int stripes = mine >= MW ? 1 : MW / mine, stripe = warp / mine;  // (a head and a stripe) per warp, heads in turn if there are more
  if (stripes == 1 && stripe > 0) return;
  for (int i = warp % mine; i < mine; i += MW) {
    const int h = h0 + i * (n - 1);
    Partial y = empty_partial();
    if (stripe < stripes)
      for (int k = stripe; k < n; k += stripes * MBATCH) {
        Partial x[MBATCH + 1];
#pragma unroll
        for (int e = 0; e < MBATCH; ++e) {
          const int at = k + e * stripes;
          x[e] = at < n ? load_partial(p, ((i0 + at) * 2 + (at == 0)) * p.G + h, lane) : empty_partial();
        }
        x[MBATCH] = y;
        y = join(x);
      }
    if (stripes > 1) {
      s_o[warp][lane] = y.o;
      if (lane == 0) s_ml[warp] = make_float2(y.m, y.l);
      __syncthreads();  // mine < MW: every warp passes here once
      if (stripe > 0) return;
      for (int k = 1; k < stripes; ++k) {
        const float2 ml = s_ml[warp + k * mine];
        const Partial x[2] = {y, {s_o[warp + k * mine][lane], ml.x, ml.y}};
        y = join(x);
      }
    }
    store_output(out + h * D, y, lane);
  }
}

// Few short sequences: a CTA per (sequence, kv head), a unit per warp at most, does without the prefix over the lengths and
// without merge_k.  The block table bounds the lengths.  32 q and 8 kv heads: one sequence of 300 tokens 6.5 against 8.4 us,
// 16 of 512 7.2 against 10.1; with more units to a warp the ranges win (one sequence of 2048: 10.0 against 15.3).
static bool direct_path(int64_t B, int64_t Hkv, int64_t P, int64_t max_pages) { return B * Hkv <= num_sms() && max_pages * P <= DIRECT_TOKENS; }

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// A cache tensor as (pages Hkv P) rows of 128 codes; boxes of `box` rows, 128-byte swizzle.
static CUtensorMap codes_map(const void* base, long rows, int box) {
  static EncodeFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    AX_CHECK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && ptr, "cuTensorMapEncodeTiled");
    return reinterpret_cast<EncodeFn>(ptr);
  }();
  CUtensorMap m;
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)D};
  const cuuint32_t bx[2] = {(cuuint32_t)D, (cuuint32_t)box}, estr[2] = {1, 1};
  const CUresult r = fn(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, bx, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  AX_CHECK(r == CUDA_SUCCESS, "tensor map encode failed (", (int)r, ")");
  return m;
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
// New bf16 tensor without the dispatcher, which took 0.5 of the 7 us of a small call.
static at::Tensor empty_bf16(at::IntArrayRef sizes, const c10::Device& dev) { return at::detail::empty_cuda(sizes, at::kBFloat16, dev, c10::nullopt); }
// In the given type and contiguous; itself if it is.
static at::Tensor as(const at::Tensor& t, at::ScalarType ty) { return t.scalar_type() == ty ? t.contiguous() : t.to(ty).contiguous(); }
static void aligned16(const at::Tensor& t, const char* name) {
  AX_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, name, " starts on a 16-byte boundary");
}

}  // namespace kv8

std::tuple<at::Tensor, at::Tensor, at::Tensor> qknorm_rope_cache_fp8(const at::Tensor& qkv_, const at::Tensor& qw_, const at::Tensor& kw_,
                                                                     const at::Tensor& pos_, const at::Tensor& inv_freq_, int64_t nq,
                                                                     int64_t nkv, double eps, const at::Tensor& k, const at::Tensor& v,
                                                                     const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& slots_,
                                                                     bool want_kv) {
  using namespace kv8;
  const Cache c = checked(k, v, ks, vs);
  const auto dev = k.device();
  for (const at::Tensor* t : {&qkv_, &qw_, &kw_, &pos_, &inv_freq_, &slots_}) AX_CHECK(t->device() == dev, "inputs on the cache's device");
  const c10::cuda::CUDAGuard guard(dev);
  const auto qkv = qkv_.contiguous(), qw = as(qw_, at::kBFloat16), kw = as(kw_, at::kBFloat16), pos = as(pos_, at::kInt),
             inv_freq = as(inv_freq_, at::kFloat), slots = as(slots_, at::kLong);
  AX_CHECK(nq >= 0 && nkv >= 1 && nkv == c.Hkv, "nkv must be the cache's head count");
  AX_CHECK(qkv.scalar_type() == at::kBFloat16 && qkv.dim() == 2 && qkv.size(1) == (nq + 2 * nkv) * D, "qkv: bf16 (T, (nq + 2 nkv) 128)");
  const int64_t T = qkv.size(0);
  AX_CHECK(T < (1LL << 31), "too many tokens");
  TORCH_CHECK_NOT_IMPLEMENTED(2 * inv_freq.numel() == qw.numel(), "partial rotary embedding (", 2 * inv_freq.numel(), " of ", qw.numel(), " dims) has no CUDA kernel yet");
  AX_CHECK(qw.numel() == D && kw.numel() == D, "norm weights (128,)");
  AX_CHECK(pos.numel() == T && slots.numel() == T, "pos, slots: (T,)");
  aligned16(qkv, "qkv"), aligned16(qw, "q norm weight"), aligned16(kw, "k norm weight");
  auto q = empty_bf16({T, nq, D}, dev);
  at::Tensor ko, vo;
  if (want_kv) ko = empty_bf16({T, nkv, D}, dev), vo = empty_bf16({T, nkv, D}, dev);
  if (T == 0) return {q, ko, vo};
  // Warps per token: the most with which every CTA (eight warps) is resident at once, four on an SM, since the call then takes
  // as long as one CTA; beyond that two, so that four tokens share a CTA's start, or one where a token has few heads.  32 q and 8 kv
  // heads, us with 8 / 4 / 2 warps: 64 tokens 3.0 / 3.5 / 5.1, 592 (one wave with eight) 4.5 / 4.4 / 5.3, 593 5.6 / 6.0 / 8.0,
  // 1184 (one wave with four) 8.1 / 6.4 / 7.0, 1185 8.6 / 7.7 / 10.5, 2368 (one wave with two) 16.2 / 12.5 / 11.8, 9000 57 / 44 / 41.
  // 8 q and 1 kv head, two warps and one: 2368 tokens 5.3 / 5.6, 4736 9.4 / 8.8, 9000 17.7 / 16.1.
  const int64_t many = (int64_t)num_sms() * 4, groups = (nq + 3) / 4 + (2 * nkv + 3) / 4;
  const int parts = T <= many ? 8 : T <= 2 * many ? 4 : groups < 8 && T > 8 * many ? 1 : 2;
  launch_pdl(append_k, dim3((unsigned)((T + AW / parts - 1) / (AW / parts))), dim3(AW * 32), 0, stream(), (const bf16*)qkv.data_ptr(), (const bf16*)qw.data_ptr(),
             (const bf16*)kw.data_ptr(), (const int*)pos.data_ptr(), (const float*)inv_freq.data_ptr(), (bf16*)q.data_ptr(),
             (bf16*)(want_kv ? ko.data_ptr() : nullptr), (bf16*)(want_kv ? vo.data_ptr() : nullptr), (int)T, (int)nq, (int)nkv, (float)eps, c,
             (const int64_t*)slots.data_ptr(), parts);
  AX_LAUNCH_OK();
  return {q, ko, vo};
}

std::tuple<at::Tensor, at::Tensor> gather_kv_fp8(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs,
                                                 const at::Tensor& slots_, const c10::optional<at::Tensor>& out_k,
                                                 const c10::optional<at::Tensor>& out_v) {
  using namespace kv8;
  const Cache c = checked(k, v, ks, vs);
  const auto dev = k.device();
  AX_CHECK(slots_.device() == dev && slots_.dim() == 1, "slots: (T,) on the cache's device");
  const c10::cuda::CUDAGuard guard(dev);
  const auto slots = as(slots_, at::kLong);
  const long T = slots.numel();
  auto ko = out_k.has_value() ? *out_k : empty_bf16({T, c.Hkv, D}, dev), vo = out_v.has_value() ? *out_v : empty_bf16({T, c.Hkv, D}, dev);
  for (const at::Tensor* o : {&ko, &vo}) {
    AX_CHECK(o->device() == dev && o->scalar_type() == at::kBFloat16 && o->dim() == 3 && o->size(0) == T && o->size(1) == c.Hkv && o->size(2) == D && o->is_contiguous(),
             "outputs: contiguous bf16 (T, Hkv, 128) on the cache's device");
    aligned16(*o, "output");
  }
  if (T == 0 || c.Hkv == 0) return {ko, vo};
  const long rows = T * 2 * c.Hkv, ctas = (rows + 8 * LR - 1) / (8 * LR);
  AX_CHECK(ctas < (1L << 31), "too many slots");
  launch_pdl(load_k, dim3((unsigned)ctas), dim3(256), 0, stream(), c, (const int64_t*)slots.data_ptr(), (bf16*)ko.data_ptr(), (bf16*)vo.data_ptr(), rows);
  AX_LAUNCH_OK();
  return {ko, vo};
}

at::Tensor paged_decode_attn_fp8(const at::Tensor& q_, const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs,
                                 const at::Tensor& block_table_, const at::Tensor& seq_lens_, double scale) {
  using namespace kv8;
  const Cache c = checked(k, v, ks, vs);
  const auto dev = k.device();
  for (const at::Tensor* t : {&q_, &block_table_, &seq_lens_}) AX_CHECK(t->device() == dev, "inputs on the cache's device");
  const c10::cuda::CUDAGuard guard(dev);
  const auto q = q_.contiguous(), block_table = block_table_.contiguous(), seq_lens = seq_lens_.contiguous();
  AX_CHECK(q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.size(2) == D, "q: bf16 (B, Hq, 128)");
  const int64_t B = q.size(0), Hq = q.size(1);
  AX_CHECK(c.Hkv >= 1 && Hq >= 1 && Hq % c.Hkv == 0 && Hq / c.Hkv <= MAXG, "GQA group must be <= 16");
  AX_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == B, "block_table: int32 (B, pages)");
  AX_CHECK(seq_lens.scalar_type() == at::kInt && seq_lens.numel() == B, "seq_lens: int32 (B,)");
  AX_CHECK(c.P % 16 == 0 && c.P > 0, "page size must be a multiple of 16");
  aligned16(q, "q"), aligned16(ks, "fp8 cache: scale tensor"), aligned16(vs, "fp8 cache: scale tensor");
  AX_CHECK(B <= MAXB, "decode batch must be <= ", MAXB);
  const long rows = c.pages * c.Hkv * c.P;
  AX_CHECK(rows < (1L << 31), "fp8 cache: pages * Hkv * page size must be below 2^31");
  AX_CHECK(B * (2 * (block_table.size(1) * c.P / UNIT + 1) + 1) * c.Hkv < (1L << 30), "block_table: too many tokens");
  auto out = empty_bf16({B, Hq, D}, dev);
  if (B == 0) return out;
  if (rows == 0 || block_table.size(1) == 0) return out.zero_();
  const bool direct = direct_path(B, c.Hkv, c.P, block_table.size(1));
  const int G = (int)(Hq / c.Hkv), grid = direct ? (int)B * c.Hkv : num_sms();
  // partials: freed after the launches, so the memory is handed on in stream order (and is the graph's when captured)
  const long joined = (long)grid * 2 * G, kept = G <= 8 ? 0 : (long)grid * NW * G;
  const c10::DataPtr part = c10::cuda::CUDACachingAllocator::get()->allocate((joined * (D + 2) + kept * D) * sizeof(float));
  float* part_o = (float*)part.get();
  int box = 16;
  while (box < 64 && c.P % (2 * box) == 0) box *= 2;
  const CUtensorMap tk = codes_map(c.k, rows, box), tv = codes_map(c.v, rows, box);
  const DecParams p{(const bf16*)q.data_ptr(), (const int*)block_table.data_ptr(), (const int*)seq_lens.data_ptr(), c.ks, c.vs, (bf16*)out.data_ptr(),
                    part_o, (float2*)(part_o + joined * D), part_o + joined * (D + 2), c.pages, (int)B, G, c.Hkv, c.P,
                    (int)block_table.size(1), box, (float)(scale * 1.4426950408889634), direct};
  auto kern = G <= 8 ? decode_k<1> : decode_k<2>;
  smem_attr((const void*)kern, 227 * 1024 - 256);
  launch_pdl(kern, dim3(grid), dim3(NW * 32), dec_smem(G, (int)B), stream(), tk, tv, p);
  AX_LAUNCH_OK();
  if (direct) return out;
  launch_pdl(merge_k, dim3(grid), dim3(MW * 32), (B + 1) * sizeof(int), stream(), p);
  AX_LAUNCH_OK();
  return out;
}

// Kernels that paged_decode_attn_fp8 launches for these sizes.
int64_t paged_decode_attn_fp8_launches(int64_t B, int64_t pages, int64_t Hkv, int64_t P, int64_t max_pages) {
  if (B == 0 || pages * P == 0 || max_pages == 0) return 0;
  return kv8::direct_path(B, Hkv, P, max_pages) ? 1 : 2;
}

// 0, or the code of the first bounded wait of the decode kernel that gave up on the current device, in what the current stream
// was given so far; waits for that.
int64_t kv_fp8_error() {
  int v = 0;
  AX_CUDA_OK(cudaMemcpyFromSymbolAsync(&v, kv8::g_decode_err, sizeof(int), 0, cudaMemcpyDeviceToHost, stream()));
  AX_CUDA_OK(cudaStreamSynchronize(stream()));
  return v;
}

}  // namespace ax
