// Block-sparse attention over the paged GQA cache, the two parts beside the attention itself (attn_block_decode.cu):
// the cache writer that keeps an 8-bit bound of every finished page's keys, and the selection of the pages that a
// group of queries attends to.
//
// Bound of one page and kv head, from its 64 stored keys: lo_d, hi_d = min, max over the page, c = (lo + hi) / 2,
// w = (hi - lo) / 2, both as 8-bit codes of one power of two 2^e (max(|c|, w) 2^-e in [64, 128), clamped to 127).
// For any query q and any key k of the page  q . k <= sum_d q_d c_d + |q_d| w_d  (up to the codes' rounding), which
// is what the selection ranks pages by.  Codes, their products and sums are whole numbers below 2^24 and the scales
// powers of two, so every score is exact and the selection does not depend on the order of a sum.
#include "common.cuh"
#include "kernels.h"

namespace iob {
namespace {

constexpr int kPage = 64;
constexpr int kSumExpMin = -100;      // exponent range of the codes' scales (bf16 powers of two)

// Exponent of the scale 2^e of the 8-bit codes of values up to amax: amax = m 2^x, m in [0.5, 1) -> e = x - 7.
__device__ __forceinline__ int code_exp(float amax) {
  int x = 0;
  frexpf(amax, &x);
  return max(kSumExpMin, min(100, x - 7));
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int code8(float v, float inv) {
  return max(-127, min(127, __float2int_rn(v * inv)));
}

// ------------------------------------------------------------------------------------------ head vectors
// D / 16 lanes hold one head vector, so a warp holds 4, 2 or 1 of them (D = 128, 256, 512): lane l of a vector owns 8
// consecutive values of each half (16-byte accesses), so both members of every rotated pair (i, i + D / 2) are in one
// thread.  Values go in pairs: one instruction handles two fp32.
template <int D>
struct Lane {
  static constexpr int H2 = 8;          // values of one half
  static constexpr int P = H2 / 2;      // pairs of one half
  static constexpr int N = D / 16;      // lanes of a vector
  static constexpr int PER_WARP = 32 / N;
  static __device__ __forceinline__ int in_vector() { return lane_id() % N; }
  static __device__ __forceinline__ int vector() { return lane_id() / N; }
  static __device__ __forceinline__ uint32_t mask() {      // the lanes of this lane's vector
    return N == 32 ? 0xffffffffu : ((1u << (N & 31)) - 1u) << (vector() * N);
  }
};

template <int BYTES>
struct Raw;
template <> struct Raw<2> { using T = uint16_t; };
template <> struct Raw<4> { using T = uint32_t; };

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;\n\t}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 bf2(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t to_bf2(float2 v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A lane's share of a bf16 head vector as it lies in memory: pairs 0 .. P - 1 of the first half, then the second's.
template <int D>
struct Head {
  uint32_t w[2 * Lane<D>::P];
};
template <int P>
__device__ __forceinline__ void load_words(const void* src, uint32_t* w) {
  if constexpr (P == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(src);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(src);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  }
}
template <int P>
__device__ __forceinline__ void store_words(void* dst, const uint32_t* w) {
  if constexpr (P == 1) *reinterpret_cast<uint32_t*>(dst) = w[0];
  else if constexpr (P == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <int D>
__device__ __forceinline__ Head<D> fetch(const __nv_bfloat16* src, int lane) {
  Head<D> r;
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) load_words<Lane<D>::P>(src + hh * (D / 2) + lane * Lane<D>::H2, &r.w[hh * Lane<D>::P]);
  return r;
}
template <int D>
__device__ __forceinline__ void store_head(__nv_bfloat16* dst, int lane, const Head<D>& r) {
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) store_words<Lane<D>::P>(dst + hh * (D / 2) + lane * Lane<D>::H2, &r.w[hh * Lane<D>::P]);
}

// What a stored row holds, as 16-bit pairs in units of the pool's scale: bf16, or f16 for E4M3 values and for E2M1
// codes times their block's scale (both exact).
template <int FMT>
__device__ __forceinline__ float2 pair_value(uint32_t w) {
  if constexpr (FMT == kKvBf16) return bf2(w);
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// H2 E2M1 codes of one word (lowest nibble first) -> pairs of code * block scale in f16.  Twice the magnitudes
// {0, .5, 1, 1.5, 2, 3, 4, 6} are the bytes of a two-word table that a byte permute indexes; as f16 integers (an
// exponent glued to the byte, 1024 taken off) they are exact, and so are the products.
template <int H2>
__device__ __forceinline__ void widen_e2m1(uint32_t word, float sf, uint32_t* pairs) {
  const __half2 half_sf = __float2half2_rn(0.5f * sf);
#pragma unroll
  for (int j = 0; j < H2; j += 2) {
    const uint32_t c = (word >> (4 * j)) & 0x77u;
    uint32_t m = prmt(0x03020100u, 0x0C080604u, c) & 0xffffu;                 // two magnitude bytes
    m = prmt(m, 0x64646464u, 0x4140u);                                        // 1024 + magnitude, f16 pair
    __half2 v = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&m), __float2half2_rn(1024.f)), half_sf);
    const uint32_t sg = word >> (4 * j);
    pairs[j / 2] = *reinterpret_cast<uint32_t*>(&v) | ((sg & 8u) << 12) | ((sg & 0x80u) << 24);
  }
}

// x in units of the pool's scale (inv = 1 / unit).  bf16 values that lie halfway between two codes are common, and a
// product with the rounded reciprocal may move them off the tie, so the product's residual, which an fma has exactly, is
// added once (Markstein's correction): a quotient that is an fp32 number comes out as that number, any other within a
// last bit.  (E4M3, 7 x 219 rows of D = 256, scales 0.75 / 1.25: 26.7 us; the product alone 25.3, divisions 34.)
__device__ __forceinline__ float2 in_units(float2 x, float unit, float inv) {
  if (unit == 1.f) return x;
  const float2 q = mul2(x, make_float2(inv, inv));
  const float2 c = fma2(fma2(q, make_float2(-unit, -unit), x), make_float2(inv, inv), q);
  return make_float2(fabsf(q.x) < INFINITY ? c.x : q.x, fabsf(q.y) < INFINITY ? c.y : q.y);
}

// One row of a pool part (K or V of a page and head): stores x (one rounding, from fp32; `unit` is the pool's scale, `inv` its
// reciprocal) and returns what the row holds.
template <int D, int FMT>
__device__ __forceinline__ Head<D> store_row(uint8_t* part, int off, int lane, float unit, float inv,
                                             const float2 (&x)[2 * Lane<D>::P]) {
  constexpr int H2 = Lane<D>::H2, P = Lane<D>::P;
  Head<D> out;
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    const int e0 = hh * (D / 2) + lane * H2;
    if constexpr (FMT == kKvBf16) {
#pragma unroll
      for (int j = 0; j < P; ++j) out.w[hh * P + j] = to_bf2(x[hh * P + j]);
      store_words<P>(part + off * 2 * D + kv_swizzle_byte(2 * e0, off, 2 * D), &out.w[hh * P]);
    } else if constexpr (FMT == kKvFp8) {
      uint32_t word[P / 2] = {};
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float2 y = in_units(x[hh * P + j], unit, inv);
        const uint32_t e = f32x2_to_e4m3x2(y.x, y.y);
        out.w[hh * P + j] = e4m3x2_to_f16x2(static_cast<uint16_t>(e));
        word[j / 2] |= e << (16 * (j & 1));
      }
      *reinterpret_cast<uint2*>(part + off * D + kv_swizzle_byte(e0, off, D)) = make_uint2(word[0], word[1]);
    } else {
      constexpr int LPB = 16 / H2;       // lanes per 16-value block
      float2 y[P];
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        y[j] = in_units(x[hh * P + j], unit, inv);
        amax = fmaxf(amax, fmaxf(fabsf(y[j].x), fabsf(y[j].y)));
      }
#pragma unroll
      for (int o = 1; o < LPB; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(Lane<D>::mask(), amax, o));
      const uint8_t s8 = nvfp4_block_scale(amax);
      // E2M1 codes count the midpoints strictly below a magnitude (ties go down), so a reciprocal rounded down keeps a value
      // that is a midpoint times the block's scale on the right side
      const float sf = e4m3_to_float(s8), inv_sf = __frcp_rd(sf);
      if ((lane % LPB) == 0) part[kPage * (D / 2) + off * (D / 16) + e0 / 16] = s8;
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < P; ++j)
        word |= (e2m1_code(y[j].x * inv_sf) | (e2m1_code(y[j].y * inv_sf) << 4)) << (8 * j);
      *reinterpret_cast<uint32_t*>(part + off * (D / 2) + kv_swizzle_byte(e0 / 2, off, D / 2)) = word;
      widen_e2m1<H2>(word, sf, &out.w[hh * P]);
    }
  }
  return out;
}

template <int D, int FMT>
__device__ __forceinline__ Head<D> load_row(const uint8_t* part, int off, int lane) {
  constexpr int H2 = Lane<D>::H2, P = Lane<D>::P;
  Head<D> out;
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    const int e0 = hh * (D / 2) + lane * H2;
    if constexpr (FMT == kKvBf16) {
      load_words<P>(part + off * 2 * D + kv_swizzle_byte(2 * e0, off, 2 * D), &out.w[hh * P]);
    } else if constexpr (FMT == kKvFp8) {
      const uint2 word = *reinterpret_cast<const uint2*>(part + off * D + kv_swizzle_byte(e0, off, D));
#pragma unroll
      for (int j = 0; j < P; ++j)
        out.w[hh * P + j] = e4m3x2_to_f16x2(static_cast<uint16_t>((j < 2 ? word.x : word.y) >> (16 * (j & 1))));
    } else {
      const float sf = e4m3_to_float(part[kPage * (D / 2) + off * (D / 16) + e0 / 16]);
      const uint32_t word = *reinterpret_cast<const uint32_t*>(part + off * (D / 2) + kv_swizzle_byte(e0 / 2, off, D / 2));
      widen_e2m1<H2>(word, sf, &out.w[hh * P]);
    }
  }
  return out;
}

// Cosines and sines of one position, this lane's pairs.
template <int D>
struct Angles {
  float2 c[Lane<D>::P], s[Lane<D>::P], ns[Lane<D>::P];
  __device__ __forceinline__ void load(const float* cs, int lane) {
    constexpr int H2 = Lane<D>::H2;
    const float* cl = cs + lane * H2;
#pragma unroll
    for (int j = 0; j < H2; j += 4) {
      const float4 u = *reinterpret_cast<const float4*>(cl + j), v = *reinterpret_cast<const float4*>(cl + D / 2 + j);
      c[j / 2] = make_float2(u.x, u.y);
      c[j / 2 + 1] = make_float2(u.z, u.w);
      s[j / 2] = make_float2(v.x, v.y);
      s[j / 2 + 1] = make_float2(v.z, v.w);
    }
#pragma unroll
    for (int j = 0; j < H2 / 2; ++j) ns[j] = make_float2(-s[j].x, -s[j].y);
  }
};

// Norm (per head, optional) and rotation in fp32; nothing is rounded in between.  `gain` is the lane's share of the
// norm's weight.
template <int D>
__device__ __forceinline__ void norm_rope(const Head<D>& raw, float2 (&x)[2 * Lane<D>::P],
                                          const float2 (&gain)[2 * Lane<D>::P], bool norm, float eps,
                                          const Angles<D>& an) {
  constexpr int P = Lane<D>::P;
#pragma unroll
  for (int j = 0; j < 2 * P; ++j) x[j] = bf2(raw.w[j]);
  if (norm) {
    float2 ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 2 * P; ++j) ss = fma2(x[j], x[j], ss);
    float sum = ss.x + ss.y;
#pragma unroll
    for (int o = 1; o < Lane<D>::N; o <<= 1) sum += __shfl_xor_sync(Lane<D>::mask(), sum, o);
    const float inv = rsqrtf(sum / D + eps);
#pragma unroll
    for (int j = 0; j < 2 * P; ++j) x[j] = mul2(mul2(x[j], make_float2(inv, inv)), gain[j]);
  }
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const float2 a = x[j], b = x[P + j];
    x[j] = fma2(b, an.ns[j], mul2(a, an.c[j]));
    x[P + j] = fma2(a, an.s[j], mul2(b, an.c[j]));
  }
}
template <int D>
__device__ __forceinline__ void load_gain(const void* w, bool plus_one, int lane, float2 (&gain)[2 * Lane<D>::P]) {
  const Head<D> r = fetch<D>(reinterpret_cast<const __nv_bfloat16*>(w), lane);
#pragma unroll
  for (int j = 0; j < 2 * Lane<D>::P; ++j) {
    gain[j] = bf2(r.w[j]);
    if (plus_one) gain[j] = make_float2(1.f + gain[j].x, 1.f + gain[j].y);
  }
}

// Running bound of the rows seen by this lane, in the rows' 16-bit pairs (nothing is rounded; the pool's scale is
// positive).  NaN stays NaN.
template <int D, int FMT>
struct Bound {
  uint32_t lo[2 * Lane<D>::P], hi[2 * Lane<D>::P];
  static constexpr uint32_t kInf = FMT == kKvBf16 ? 0x7f807f80u : 0x7c007c00u;
  static __device__ __forceinline__ uint32_t low(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (FMT == kKvBf16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t high(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (FMT == kKvBf16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int j = 0; j < 2 * Lane<D>::P; ++j) { lo[j] = kInf; hi[j] = kInf | 0x80008000u; }
  }
  __device__ __forceinline__ void add(const Head<D>& r) {
#pragma unroll
    for (int j = 0; j < 2 * Lane<D>::P; ++j) { lo[j] = low(lo[j], r.w[j]); hi[j] = high(hi[j], r.w[j]); }
  }
};

constexpr int kWarps = 4;

// End of a page's bound: the warps' shares are joined and the codes and the scale of one page and head written.
template <int D, int FMT>
__device__ void finish_bound(const Bound<D, FMT>& bd, float unit, int8_t* codes, __nv_bfloat16* scale,
                             uint32_t (&sb)[2][kWarps][D / 2]) {
  constexpr int P = Lane<D>::P, NT = kWarps * 32;
  const int lane = lane_id(), warp = warp_id();
  __shared__ float smax[kWarps];
#pragma unroll
  for (int hh = 0; hh < 2; ++hh)
#pragma unroll
    for (int j = 0; j < P; ++j) {
      uint32_t lo = bd.lo[hh * P + j], hi = bd.hi[hh * P + j];
#pragma unroll
      for (int o = Lane<D>::N; o < 32; o <<= 1) {          // the warp's vectors
        lo = Bound<D, FMT>::low(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = Bound<D, FMT>::high(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      const int d = hh * (D / 4) + Lane<D>::in_vector() * P + j;
      if (Lane<D>::vector() == 0) {
        sb[0][warp][d] = lo;
        sb[1][warp][d] = hi;
      }
    }
  __syncthreads();
  constexpr int PER = D / 2 >= NT ? D / 2 / NT : 1;       // pairs of a thread (threads past D / 2 idle)
  const int d0 = threadIdx.x * PER;
  float c[2 * PER], w[2 * PER], amax = 0.f;
  bool bad = false;
  if (d0 < D / 2) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      uint32_t l = sb[0][0][d0 + i], h = sb[1][0][d0 + i];
#pragma unroll
      for (int k = 1; k < kWarps; ++k) {
        l = Bound<D, FMT>::low(l, sb[0][k][d0 + i]);
        h = Bound<D, FMT>::high(h, sb[1][k][d0 + i]);
      }
      const float2 lv = pair_value<FMT>(l), hv = pair_value<FMT>(h);
      const float lo2[2] = {lv.x * unit, lv.y * unit}, hi2[2] = {hv.x * unit, hv.y * unit};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        c[2 * i + k] = (lo2[k] + hi2[k]) * 0.5f;
        w[2 * i + k] = (hi2[k] - lo2[k]) * 0.5f;
        bad |= !(fabsf(lo2[k]) < INFINITY && fabsf(hi2[k]) < INFINITY);
        amax = fmaxf(amax, fmaxf(fabsf(c[2 * i + k]), w[2 * i + k]));
      }
    }
  }
  if (bad) amax = INFINITY;                       // as an overflow of lo + hi or hi - lo
  amax = warp_max(amax);
  if (lane == 0) smax[warp] = amax;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kWarps; ++k) amax = fmaxf(amax, smax[k]);
  bad = !(amax < INFINITY);
  const int e = code_exp(amax);
  const float inv = pow2(-e);
  using T = typename Raw<2 * PER>::T;
  if (d0 < D / 2) {
    uint32_t rc = 0, rw = 0;
#pragma unroll
    for (int i = 0; i < 2 * PER; ++i) {
      rc |= (bad ? 0u : static_cast<uint32_t>(code8(c[i], inv)) & 0xffu) << (8 * i);
      rw |= (bad ? 0u : static_cast<uint32_t>(code8(w[i], inv)) & 0xffu) << (8 * i);
    }
    reinterpret_cast<T*>(codes)[threadIdx.x] = static_cast<T>(rc);
    reinterpret_cast<T*>(codes + D)[threadIdx.x] = static_cast<T>(rw);
  }
  if (threadIdx.x == 0) *scale = __float2bfloat16(bad ? INFINITY : pow2(e));
  __syncthreads();                                // shared memory is used again by the next run
}

// ------------------------------------------------------------------------------------------ append
// Grid: y = slabs of `slab` rows; x < Hk: the K vectors of kv head x, else `heads` of the Hq + Hk q and v vectors (a
// slab's CTAs run together: K's, which wait for their rows, beside those that only move bytes).
// q and v: a warp takes a row and walks through the heads, the position's angles in registers and the next two heads'
// values on their way.  K: a CTA owns the page runs that start in its slab (consecutive rows at consecutive slots of
// one page): its warps share the run's rows, and when the run ends at the page's last row the CTA also reads the rows
// written by earlier calls and writes the page's bound, so the bound costs no launch and no second pass over the new
// keys.
// Bound by bytes: 8192 rows, 32 q and 16 kv heads of 512, bf16: 205 us for 1.09 GB (5.3 TB/s), E4M3 196 us for 0.96 GB;
// over FP4 caches by the encoding (309 us for 0.90 GB).  A step of 64 rows is bound by its chain of loads: 5.8 us, 7.5 MB,
// E4M3; FP4 9.3.  Mixing a slab's K and q / v CTAs in launch order instead of all K first:
// 205 against 214 us; 8 warps a CTA instead of 4: 330.
__device__ __forceinline__ int row_slot(const BlockAppendArgs& a, int t) {
  const int s = a.slot[t], p = a.pos[t];
  return (s < 0 || s >= a.slots || p < 0 || p >= a.max_pos) ? -1 : s;
}

template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32, 5) block_append_kernel(const BlockAppendArgs a) {
  __shared__ uint32_t red[2][kWarps][D / 2];
  constexpr int NV = Lane<D>::PER_WARP;
  const int warp = warp_id(), lane = lane_id(), ln = Lane<D>::in_vector(), vec = Lane<D>::vector();
  const int t0 = blockIdx.y * a.slab, t1 = min(a.T, t0 + a.slab);
  const __nv_bfloat16* qkv = reinterpret_cast<const __nv_bfloat16*>(a.qkv);
  constexpr int part = FMT == kKvBf16 ? kPage * 2 * D : FMT == kKvFp8 ? kPage * D : kPage * (D / 2 + D / 16);
  float2 x[2 * Lane<D>::P], gain[2 * Lane<D>::P];
  Angles<D> an;
  if (static_cast<int>(blockIdx.x) >= a.Hk) {
    // a warp per row where there are rows for it, else a warp per NV heads
    const int first = (blockIdx.x - a.Hk) * a.heads;
    const int vend = min(first + a.heads, a.Hq + a.Hk);
    const int v0 = first + (a.slab == 1 ? warp * NV : 0), vstep = a.slab == 1 ? kWarps * NV : NV;
    if (v0 >= vend) return;
    if (a.q_norm && v0 < a.Hq) load_gain<D>(a.q_norm, a.plus_one, ln, gain);
    const float inv = 1.f / a.v_scale;
    for (int t = t0 + (a.slab == 1 ? 0 : warp); t < t1; t += (a.slab == 1 ? 1 : kWarps)) {
      const __nv_bfloat16* src = qkv + static_cast<size_t>(t) * a.qkv_stride;
      auto head = [&](int v) {
        return v < vend ? fetch<D>(src + static_cast<size_t>(v < a.Hq ? v : v + a.Hk) * D, ln) : Head<D>{};
      };
      Head<D> next = head(v0 + vec), next2 = head(v0 + vstep + vec);
      const int p = a.pos[t], s = row_slot(a, t);
      const bool ok = p >= 0 && p < a.max_pos;
      if (ok && v0 < a.Hq) an.load(a.cos_sin + static_cast<size_t>(p) * D, ln);
      __nv_bfloat16* qrow = reinterpret_cast<__nv_bfloat16*>(a.q_out) + static_cast<size_t>(t) * a.Hq * D;
      uint8_t* vrow = a.pool + static_cast<size_t>(s < 0 ? 0 : s / kPage) * a.Hk * (2 * part) + part;
      for (int vb = v0; vb < vend; vb += vstep) {
        const int v = vb + vec;
        const Head<D> raw = next;
        next = next2;
        next2 = head(v + 2 * vstep);
        if (v < a.Hq && v < vend) {
          Head<D> o{};
          if (ok) {
            norm_rope<D>(raw, x, gain, a.q_norm != nullptr, a.eps, an);
#pragma unroll
            for (int j = 0; j < 2 * Lane<D>::P; ++j) o.w[j] = to_bf2(x[j]);
          }
          store_head<D>(qrow + static_cast<size_t>(v) * D, ln, o);
        } else if (v < vend && s >= 0) {
#pragma unroll
          for (int j = 0; j < 2 * Lane<D>::P; ++j) x[j] = bf2(raw.w[j]);
          store_row<D, FMT>(vrow + static_cast<size_t>(v - a.Hq) * (2 * part), s % kPage, ln, a.v_scale, inv, x);
        }
      }
    }
    return;
  }
  const int h = blockIdx.x;
  const float unit = FMT == kKvBf16 ? 1.f : a.k_scale, inv = 1.f / unit;
  if (a.k_norm) load_gain<D>(a.k_norm, a.plus_one, ln, gain);
  // rows of the slab (at most 32) that begin a run: every lane looks at one
  const int ts = t0 + lane;
  const int mine = ts < t1 ? row_slot(a, ts) : -1;
  const bool begins = mine >= 0 && (ts == 0 || mine % kPage == 0 || row_slot(a, ts - 1) != mine - 1);
  for (uint32_t todo = __ballot_sync(0xffffffffu, begins); todo != 0; todo &= todo - 1) {
    const int first = __ffs(todo) - 1, t = t0 + first;
    const int s = __shfl_sync(0xffffffffu, mine, first);
    const int page = s / kPage, off = s % kPage;
    // rows of the run (at most to the page's end): every lane looks at two
    bool in0 = off + lane < kPage && t + lane < a.T, in1 = off + lane + 32 < kPage && t + lane + 32 < a.T;
    in0 = in0 && row_slot(a, t + lane) == s + lane;
    in1 = in1 && row_slot(a, t + lane + 32) == s + lane + 32;
    const unsigned long long in = __ballot_sync(0xffffffffu, in0) |
                                  static_cast<unsigned long long>(__ballot_sync(0xffffffffu, in1)) << 32;
    const int n = ~in == 0ull ? kPage : __ffsll(~in) - 1;
    const bool last = off + n == kPage;
    uint8_t* base = a.pool + (static_cast<size_t>(page) * a.Hk + h) * (2 * part);
    Bound<D, FMT> bd;
    bd.reset();
    const __nv_bfloat16* src = qkv + static_cast<size_t>(t) * a.qkv_stride + static_cast<size_t>(a.Hq + h) * D;
    Head<D> next{};
    if (warp * NV + vec < n) next = fetch<D>(src + (warp * NV + vec) * a.qkv_stride, ln);
    for (int i = warp * NV + vec; i < n; i += kWarps * NV) {
      an.load(a.cos_sin + static_cast<size_t>(a.pos[t + i]) * D, ln);
      const Head<D> raw = next;
      if (i + kWarps * NV < n) next = fetch<D>(src + (i + kWarps * NV) * a.qkv_stride, ln);
      norm_rope<D>(raw, x, gain, a.k_norm != nullptr, a.eps, an);
      bd.add(store_row<D, FMT>(base, off + i, ln, unit, inv, x));
    }
    __syncwarp();
    if (!last) continue;
#pragma unroll 4
    for (int i = warp * NV + vec; i < off; i += kWarps * NV) bd.add(load_row<D, FMT>(base, i, ln));
    __syncwarp();
    const size_t ph = static_cast<size_t>(page) * a.Hk + h;
    finish_bound<D, FMT>(bd, unit, a.codes + ph * 2 * D, reinterpret_cast<__nv_bfloat16*>(a.scale) + ph, red);
  }
}

// Bounds of whole pages from their stored keys: one CTA per (page of the list, kv head).
template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32) block_summarize_kernel(const BlockAppendArgs a, const int* pages) {
  __shared__ uint32_t red[2][kWarps][D / 2];
  const int page = pages[blockIdx.x], h = blockIdx.y;
  if (page < 0 || page >= a.slots / kPage) return;
  constexpr int part = FMT == kKvBf16 ? kPage * 2 * D : FMT == kKvFp8 ? kPage * D : kPage * (D / 2 + D / 16);
  const uint8_t* base = a.pool + (static_cast<size_t>(page) * a.Hk + h) * (2 * part);
  Bound<D, FMT> bd;
  bd.reset();
#pragma unroll 4
  for (int i = warp_id() * Lane<D>::PER_WARP + Lane<D>::vector(); i < kPage; i += kWarps * Lane<D>::PER_WARP)
    bd.add(load_row<D, FMT>(base, i, Lane<D>::in_vector()));
  const size_t ph = static_cast<size_t>(page) * a.Hk + h;
  finish_bound<D, FMT>(bd, FMT == kKvBf16 ? 1.f : a.k_scale, a.codes + ph * 2 * D,
                       reinterpret_cast<__nv_bfloat16*>(a.scale) + ph, red);
}

// ------------------------------------------------------------------------------------------ select
// m16n8k32, 8-bit codes, 32-bit sums.
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// fp32 -> unsigned key of the same order (the scores are never NaN; -0, which a product that underflows can be, is 0).
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(__fadd_rn(f, 0.f));      // (an addition that is not fused with the product)
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One cluster of C CTAs per (group, kv head); the CTAs share the candidate pages, the first one selects.
// Scores: the 16 query rows' codes [q8 | |q8|] are the A operand (shared memory, rows padded by 64 bytes:
// conflict-free 16-byte reads), 8 pages' records of 2 D codes the B operand, read once from global memory, 16 bytes a
// thread and 16 of them in flight; the products' k order is permuted alike on both sides so that a thread's 16 bytes
// are two instructions' fragments.  Every CTA stores its scores' order keys in the first CTA's shared memory.
// Selection: radix, eight bits at a time from the highest bit in which the keys differ (scores share their leading
// bits, which would put every key in one bin), ending as soon as a digit's bin is taken whole.
// Bound by bytes for a batch (32 groups x 16 heads x up to 512 pages of D = 512: 38 us for 175 MB, 4.6 TB/s, the
// selection's few microseconds behind the last score included), by latency for one user (8 heads x 3200 pages of
// D = 128: 10.5 us, 6.6 MB), by issue for a prefill's many lists (512 x 8 x 544 pages of D = 128: 79 us).
template <int D, bool R8, int NT, int PP, int RES>
__global__ void __launch_bounds__(NT, RES) block_select_kernel(const BlockSelectArgs a, const int csize) {
  constexpr int RS = 2 * D + 64;        // bytes between query rows
  constexpr int U = 2 * D / 64;         // 64-byte pieces of a record
  constexpr int NWARP = NT / 32;
  extern __shared__ __align__(16) uint8_t dyn[];
  int8_t* qs = reinterpret_cast<int8_t*>(dyn);                     // [16][RS]
  uint32_t* keys = reinterpret_cast<uint32_t*>(dyn + 16 * RS);     // [N] (first CTA of the cluster)
  __shared__ float rscale[16];
  __shared__ int hist[256];
  __shared__ uint32_t wmin[NWARP], wmax[NWARP];
  __shared__ int wsum[NWARP];
  __shared__ int sdigit, sneed, scnt;
  const int b = blockIdx.x / csize, rank = blockIdx.x % csize, h = blockIdx.y;
  const int tid = threadIdx.x, warp = warp_id(), lane = lane_id();
  const int row = a.req_idx ? a.req_idx[b] : b;
  const int G = a.Hq / a.Hk, R = a.n_q * G;
  int* out = a.blocks + (static_cast<size_t>(b) * a.Hk + h) * a.budget;
  const int len = (row < 0 || row >= a.rows) ? 0 : min(a.kv_len[b], a.pt_stride * kPage);
  const int npages = len > 0 ? (len + kPage - 1) / kPage : 0;
  // ---- query codes, one warp per row (before the length is looked at: the loads overlap)
#pragma unroll
  for (int r = warp; r < (R8 ? 8 : 16); r += NWARP) {
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) +
                             static_cast<size_t>(b * a.n_q + r / G) * a.q_stride + (h * G + r % G) * D;
    // Sizes compare as the bits of |bf16| do (inf and NaN above every number); rounding is to the nearest even, by an
    // addition that leaves the whole number in the low byte.
    constexpr int V = D / 32, P = V / 2;  // consecutive values of a lane
    uint32_t raw[P] = {}, top = 0;
    if (r < R) {
#pragma unroll
      for (int j = 0; j < P; j += (P < 4 ? P : 4)) load_words<(P < 4 ? P : 4)>(q + lane * V + 2 * j, &raw[j]);
    }
#pragma unroll
    for (int j = 0; j < P; ++j) top = __vmaxu2(top, raw[j] & 0x7fff7fffu);
    top = __reduce_max_sync(0xffffffffu, max(top >> 16, top & 0xffffu));
    const bool bad = top >= 0x7f80u;
    const int e = code_exp(__uint_as_float(top << 16));
    const float inv = bad ? 0.f : pow2(-e), lim = bad ? 0.f : 127.f * pow2(e);
    constexpr float kRound = 12582912.f;  // 1.5 x 2^23
    uint32_t wc[V / 4], wa[V / 4];
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      uint32_t c[4], m[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = bf2(raw[(j + k) / 2]);
        const float x = fminf(fmaxf((k & 1) ? v.y : v.x, -lim), lim);
        c[k] = __float_as_uint(fmaf(x, inv, kRound));
        m[k] = __float_as_uint(fmaf(fabsf(x), inv, kRound));
      }
      wc[j / 4] = prmt(prmt(c[0], c[1], 0x0040u), prmt(c[2], c[3], 0x0040u), 0x5410u);
      wa[j / 4] = prmt(prmt(m[0], m[1], 0x0040u), prmt(m[2], m[3], 0x0040u), 0x5410u);
    }
    store_words<V / 4>(qs + r * RS + lane * V, wc);
    store_words<V / 4>(qs + r * RS + D + lane * V, wa);
    if (lane == 0) rscale[r] = (r < R && !bad) ? pow2(e) : -1.f;
  }
  if (rank == 0 && tid == 0) a.count[static_cast<size_t>(b) * a.Hk + h] = min(npages, a.budget);
  if (npages <= a.budget) {               // every page fits: nothing to rank (the whole cluster leaves here)
    if (rank == 0)
      for (int j = tid; j < a.budget; j += NT) out[j] = j < npages ? j : -1;
    return;
  }
  const int first_local = max(0, max(0, len - a.n_q) / kPage - (a.local - 1));
  const int lo = a.sink, n = first_local - a.sink;                   // candidates [lo, lo + n)
  const int want = a.budget - (npages - n);                          // how many of them are taken
  const int span = ((n + csize - 1) / csize + 7) & ~7;               // candidates of a CTA
  const int c0 = min(n, rank * span), c1 = min(n, c0 + span);
  const int g = lane >> 2, j4 = lane & 3;
  const int* pt = a.page_table + static_cast<size_t>(row) * a.pt_stride + lo;
  int phys[PP];                           // pages of this thread's octets, loaded one step ahead
#pragma unroll
  for (int i = 0; i < PP; ++i) phys[i] = c1 > c0 ? pt[min(c0 + (warp * PP + i) * 8 + g, c1 - 1)] : 0;
  if (csize > 1) cluster_sync_all();      // also: the first CTA runs, its shared memory may be written
  else __syncthreads();
  // ---- scores; the A operand stays in registers where it fits beside the records
  constexpr bool AREG = PP == 1 && U * (R8 ? 4 : 8) <= 32;
  uint4 ax[AREG ? U : 1], ay[AREG && !R8 ? U : 1];
  if constexpr (AREG) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ax[u] = *reinterpret_cast<const uint4*>(qs + g * RS + 64 * u + 16 * j4);
      if constexpr (!R8) ay[u] = *reinterpret_cast<const uint4*>(qs + (g + 8) * RS + 64 * u + 16 * j4);
    }
  }
  const float s0 = rscale[g], s1 = R8 ? -1.f : rscale[g + 8];
  const int8_t* rec0 = a.codes + h * (2 * D) + 16 * j4;
  const __nv_bfloat16* sc_h = reinterpret_cast<const __nv_bfloat16*>(a.scale) + h;
  const uint32_t rec_stride = static_cast<uint32_t>(a.Hk) * (2 * D), hk = static_cast<uint32_t>(a.Hk);
  const uint32_t pages = static_cast<uint32_t>(a.pages);
  const uint32_t key_addr = csize > 1 ? mapa_shared(smem_u32(keys), 0) : smem_u32(keys);
  for (int p0 = c0 + warp * PP * 8; p0 < c1; p0 += NWARP * PP * 8) {
    uint4 bv[PP][U];
    float sc[PP];
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const bool ok = static_cast<uint32_t>(phys[i]) < pages;
      const uint32_t pg = ok ? static_cast<uint32_t>(phys[i]) : 0u;
      const uint4* rec = reinterpret_cast<const uint4*>(rec0 + static_cast<uint64_t>(pg) * rec_stride);
#pragma unroll
      for (int u = 0; u < U; ++u) bv[i][u] = rec[4 * u];
      sc[i] = ok ? __bfloat162float(sc_h[static_cast<uint64_t>(pg) * hk]) : -1.f;
    }
    const int pn = p0 + NWARP * PP * 8;
#pragma unroll
    for (int i = 0; i < PP; ++i) phys[i] = pn < c1 ? pt[min(pn + i * 8 + g, c1 - 1)] : 0;
    int c[PP][4];
#pragma unroll
    for (int i = 0; i < PP; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) c[i][k] = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint4 x, y = make_uint4(0, 0, 0, 0);
      if constexpr (AREG) {
        x = ax[u];
        if constexpr (!R8) y = ay[u];
      } else {
        x = *reinterpret_cast<const uint4*>(qs + g * RS + 64 * u + 16 * j4);
        if constexpr (!R8) y = *reinterpret_cast<const uint4*>(qs + (g + 8) * RS + 64 * u + 16 * j4);
      }
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        mma_s8(c[i], x.x, y.x, x.y, y.y, bv[i][u].x, bv[i][u].y);
        mma_s8(c[i], x.z, y.z, x.w, y.w, bv[i][u].z, bv[i][u].w);
      }
    }
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      float m0 = -INFINITY, m1 = -INFINITY;           // pages 2 j4, 2 j4 + 1 of the octet
      if (s0 > 0.f) { m0 = static_cast<float>(c[i][0]) * s0; m1 = static_cast<float>(c[i][1]) * s0; }
      if (!R8 && s1 > 0.f) {
        m0 = fmaxf(m0, static_cast<float>(c[i][2]) * s1);
        m1 = fmaxf(m1, static_cast<float>(c[i][3]) * s1);
      }
      // largest of the rows: the first exchange leaves each lane one of its two pages, so that lanes 0 .. 7 end with
      // page 2 (lane & 3) + (lane >> 2)
      float m = (g & 1) ? m1 : m0;
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, (g & 1) ? m0 : m1, 4));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
      const int at = 2 * (lane & 3) + ((lane >> 2) & 1);
      const float sp = __shfl_sync(0xffffffffu, sc[i], 4 * at);
      const int p = p0 + 8 * i + at;
      // a page whose keys are not finite ranks first, one outside the pool last
      const float v = sp < 0.f ? -INFINITY : sp == INFINITY ? INFINITY : m * sp;
      if (lane < 8 && p < c1)
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(key_addr + 4 * p), "r"(order_key(v)) : "memory");
    }
  }
  if (csize > 1) {
    cluster_sync_all();
    if (rank != 0) return;                // nothing of this CTA is read any more
  } else {
    __syncthreads();
  }
  // ---- range of the keys: the digits start at the highest bit in which they differ
  uint32_t kmin = 0xffffffffu, kmax = 0;
  for (int i = tid; i < n; i += NT) {
    const uint32_t k = keys[i];
    kmin = min(kmin, k);
    kmax = max(kmax, k);
  }
  kmin = __reduce_min_sync(0xffffffffu, kmin);
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  if (lane == 0) { wmin[warp] = kmin; wmax[warp] = kmax; }
  for (int i = tid; i < 256; i += NT) hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NWARP; ++w) { kmin = min(kmin, wmin[w]); kmax = max(kmax, wmax[w]); }
  int top = 32 - __clz(kmin ^ kmax);               // bits that differ
  uint32_t mask = top >= 32 ? 0u : 0xffffffffu << top;
  uint32_t prefix = kmax & mask;
  int need = want, cnt = n;                        // keys equal to the prefix: how many are taken, how many there are
  if (want == 0) { mask = 0xffffffffu; prefix = 0xffffffffu; top = 0; }      // above every key
  while (top > 0 && need < cnt) {
    const int shift = max(0, top - 8);
    const uint32_t digits = (1u << (top - shift)) - 1;
    for (int i = tid; i < n; i += NT) {
      const uint32_t k = keys[i];
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & digits], 1);
    }
    __syncthreads();
    if (warp == 0) {
      int own = 0, c8[8];                          // lane l: digits 255 - 8 l .. 248 - 8 l
#pragma unroll
      for (int i = 0; i < 8; ++i) { c8[i] = hist[255 - 8 * lane - i]; own += c8[i]; }
      int before = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      before -= own;
      if (before < need && need <= before + own) {
        int acc = before;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (acc < need && need <= acc + c8[i]) { sdigit = 255 - 8 * lane - i; sneed = need - acc; scnt = c8[i]; }
          acc += c8[i];
        }
      }
    }
    __syncthreads();
    for (int i = tid; i < 256; i += NT) hist[i] = 0;
    prefix |= static_cast<uint32_t>(sdigit) << shift;
    mask |= digits << shift;
    need = sneed;
    cnt = scnt;
    top = shift;
    __syncthreads();
  }
  // ---- compaction in page order: thread t owns a contiguous run of candidates
  const int per = (n + NT - 1) / NT;
  const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
  int gt = 0, eq = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = keys[i] & mask;
    gt += k > prefix;
    eq += k == prefix;
  }
  // exclusive prefixes of both counts over the CTA (gt < 2^11, eq < 2^16: packed in one word)
  const int pack = (gt << 16) | eq;
  int inc = pack;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) wsum[warp] = inc;
  __syncthreads();
  int base = inc - pack;
#pragma unroll
  for (int w = 0; w < NWARP; ++w)
    if (w < warp) base += wsum[w];
  int gt_before = base >> 16, eq_before = base & 0xffff;
  if (gt + eq > 0)
    for (int i = i0; i < i1; ++i) {
      const uint32_t k = keys[i] & mask;
      if (k > prefix || (k == prefix && eq_before < need)) out[a.sink + gt_before + min(eq_before, need)] = lo + i;
      gt_before += k > prefix;
      eq_before += k == prefix;
    }
  for (int i = tid; i < a.sink; i += NT) out[i] = i;
  for (int i = first_local + tid; i < npages; i += NT) out[a.sink + want + (i - first_local)] = i;
}

template <int D, int FMT>
cudaError_t append_launch(const BlockAppendArgs& a, cudaStream_t s) {
  const dim3 grid(a.Hk + (a.Hq + a.Hk + a.heads - 1) / a.heads, (a.T + a.slab - 1) / a.slab);
  block_append_kernel<D, FMT><<<grid, kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}
template <int D, int FMT>
cudaError_t summarize_launch(const BlockAppendArgs& a, const int* pages, int n, cudaStream_t s) {
  block_summarize_kernel<D, FMT><<<dim3(n, a.Hk), kWarps * 32, 0, s>>>(a, pages);
  return cudaGetLastError();
}
template <int D, bool R8, int NT, int PP, int RES>
cudaError_t select_launch_v(const BlockSelectArgs& a, int cs, cudaStream_t s) {
  // (the limit is the widest table's, the same in every call: calls of several host threads do not lower it)
  constexpr int kRows = 16 * (2 * D + 64), kMost = kRows + 4 * kBlockSelectMaxPages;
  static_assert(kMost + 4096 <= 227 * 1024, "the widest table's keys fit");
  auto k = block_select_kernel<D, R8, NT, PP, RES>;
  IOB_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.B) * cs, a.Hk);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = kRows + 4 * a.pt_stride;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  while (cs > 1 && !cluster_fits(k, cfg)) {
    attr[0].val.clusterDim.x = --cs;
    cfg.gridDim.x = static_cast<unsigned>(a.B) * cs;
  }
  return cudaLaunchKernelEx(&cfg, k, a, cs);
}
template <int D, bool R8>
cudaError_t select_launch_r(const BlockSelectArgs& a, cudaStream_t s) {
  // Thousands of lists (a prefill chunk): small CTAs, many on an SM, so that one's selection runs under another's
  // scores.  Enough to fill the SMs twice over: the same with larger CTAs; up to twice: with twice as large ones, whose
  // selection is shorter.  Few: the candidates of a list are split over a cluster until the SMs have two CTAs each, as
  // long as a CTA keeps 64 pages, with 16 loads in flight per thread.  (The page table's width bounds the candidates.)
  // Measured, many / some / few: 512 groups x 8 heads x 544 pages of D = 128: 79 / 93 / 134 us; 32 x 16 x 512 pages of
  // D = 512: 50 / 38 / 45 us; 1 x 8 x 3200 pages of D = 128: 56 / 32 / 11 us; some with 256 / 512 threads: 32 x 16 lists
  // 38 / 43 us, 16 x 16 lists 29 / 23 us.
  const int units = a.B * a.Hk;
  const int var = units >= 148 * 8 ? 2 : units > 148 ? 1 : 0;
  int cs = 1;
  while (var == 0 && cs < 8 && units * cs * 2 <= 2 * 148 && a.pt_stride >= 128 * cs) cs *= 2;
  if (var == 2) return select_launch_v<D, R8, 128, 1, 8>(a, cs, s);
  if (var == 1 && units <= 2 * 148) return select_launch_v<D, R8, 512, 1, 2>(a, cs, s);
  if (var == 1) return select_launch_v<D, R8, 256, 1, 4>(a, cs, s);
  return select_launch_v<D, R8, 256, 1024 / (2 * D), 2>(a, cs, s);
}
template <int D>
cudaError_t select_launch(const BlockSelectArgs& a, cudaStream_t s) {
  return a.n_q * (a.Hq / a.Hk) <= 8 ? select_launch_r<D, true>(a, s) : select_launch_r<D, false>(a, s);
}

#define IOB_BY_D_FMT(fn, ...)                                                     \
  switch (a.D * 4 + a.fmt) {                                                      \
    case 128 * 4 + kKvBf16: return fn<128, kKvBf16>(__VA_ARGS__);                 \
    case 128 * 4 + kKvFp8: return fn<128, kKvFp8>(__VA_ARGS__);                   \
    case 128 * 4 + kKvNvfp4: return fn<128, kKvNvfp4>(__VA_ARGS__);               \
    case 256 * 4 + kKvBf16: return fn<256, kKvBf16>(__VA_ARGS__);                 \
    case 256 * 4 + kKvFp8: return fn<256, kKvFp8>(__VA_ARGS__);                   \
    case 256 * 4 + kKvNvfp4: return fn<256, kKvNvfp4>(__VA_ARGS__);               \
    case 512 * 4 + kKvBf16: return fn<512, kKvBf16>(__VA_ARGS__);                 \
    case 512 * 4 + kKvFp8: return fn<512, kKvFp8>(__VA_ARGS__);                   \
    case 512 * 4 + kKvNvfp4: return fn<512, kKvNvfp4>(__VA_ARGS__);               \
    default: return cudaErrorInvalidValue;                                        \
  }

}  // namespace

cudaError_t block_append(const BlockAppendArgs& a_, cudaStream_t s) {
  BlockAppendArgs a = a_;
  if (a.T == 0) return cudaSuccess;
  if (a.T > 65535 * 16) return cudaErrorInvalidValue;      // the grid's second dimension
  // A decode step (each row its own page) wants a CTA per row, a prefill fewer, longer CTAs.  The number of rows stands for
  // both.  Measured, a row / 16 rows a CTA: steps of 200 rows of D = 512, E4M3 14.8 / 22.7 us; verify of 32 x 4 rows
  // 8.5 / 9.4, of 64 x 4 16.6 / 12.7, of 65 x 4 of D = 128, bf16 6.3 / 6.9, of 200 x 4 14.3 / 9.5; one request of 100 rows of
  // D = 512, bf16 9.8 / 10.2, of 300 22.9 / 17.7, of 512 32.6 / 21.1.
  a.slab = a.T <= 256 ? 1 : 16;
  // Heads of a q / v CTA: one per vector of its warps for a step; in a prefill a warp walks through 4 (D = 512) or through
  // 2 vectors' worth, which shares the angles and keeps enough CTAs (7 x 219 rows of D = 256, E4M3: 26.1 us when it was chosen,
  // twice as many heads 28.0).
  a.heads = a.slab == 1 ? 4 * (512 / a.D) : a.D == 512 ? 4 : 2 * (512 / a.D);
  IOB_BY_D_FMT(append_launch, a, s)
}

cudaError_t block_summarize(const BlockAppendArgs& a, const int* pages, int n, cudaStream_t s) {
  if (n == 0) return cudaSuccess;
  IOB_BY_D_FMT(summarize_launch, a, pages, n, s)
}

cudaError_t block_select(const BlockSelectArgs& a, cudaStream_t s) {
  if (a.B == 0) return cudaSuccess;
  if (a.pt_stride > kBlockSelectMaxPages || a.budget > kBlockMaxList || a.budget < a.sink + a.local + 1 || a.sink < 0 || a.local < 1 ||
      a.n_q < 1 || a.Hk < 1 || a.Hq % a.Hk || a.n_q * (a.Hq / a.Hk) > 16)
    return cudaErrorInvalidValue;
  switch (a.D) {
    case 128: return select_launch<128>(a, s);
    case 256: return select_launch<256>(a, s);
    case 512: return select_launch<512>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace iob
