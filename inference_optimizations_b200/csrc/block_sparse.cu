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
// A warp holds one head vector of D values: lane l owns D / 64 consecutive values of each half, so both members of
// every rotated pair (i, i + D / 2) are in one thread.
template <int D>
struct Lane {
  static constexpr int H2 = D / 64, E = D / 32;
};

template <int BYTES>
struct Raw;
template <> struct Raw<1> { using T = uint8_t; };
template <> struct Raw<2> { using T = uint16_t; };
template <> struct Raw<4> { using T = uint32_t; };
template <> struct Raw<8> { using T = uint2; };
template <> struct Raw<16> { using T = uint4; };

template <int D>
__device__ __forceinline__ void load_bf16(const __nv_bfloat16* src, int lane, float (&x)[D / 32]) {
  constexpr int H2 = Lane<D>::H2;
  using T = typename Raw<2 * H2>::T;
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    const T raw = *reinterpret_cast<const T*>(src + hh * (D / 2) + lane * H2);
    const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&raw);
#pragma unroll
    for (int j = 0; j < H2; ++j) x[hh * H2 + j] = __bfloat162float(e[j]);
  }
}
template <int D>
__device__ __forceinline__ void store_bf16(__nv_bfloat16* dst, int lane, const float (&x)[D / 32]) {
  constexpr int H2 = Lane<D>::H2;
  using T = typename Raw<2 * H2>::T;
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    T raw;
    __nv_bfloat16* e = reinterpret_cast<__nv_bfloat16*>(&raw);
#pragma unroll
    for (int j = 0; j < H2; ++j) e[j] = __float2bfloat16(x[hh * H2 + j]);
    *reinterpret_cast<T*>(dst + hh * (D / 2) + lane * H2) = raw;
  }
}

// N E2M1 codes of one word (lowest nibble first) -> code * block scale * global scale.  Twice the magnitudes
// {0, .5, 1, 1.5, 2, 3, 4, 6} are the bytes of a two-word table that a byte permute indexes.
template <int N>
__device__ __forceinline__ void widen_e2m1(uint32_t word, float sf, float scale, float* x) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t c = word >> (4 * j);
    const float m = 0.5f * static_cast<float>(prmt(0x03020100u, 0x0C080604u, c & 7u) & 0xffu);
    x[j] = ((c & 8u) ? -m : m) * sf * scale;
  }
}

// One row of a pool part (K or V of a page and head): stores x (one rounding, from fp32) and replaces it by the
// values the stored row stands for.
template <int D, int FMT>
__device__ __forceinline__ void store_row(uint8_t* part, int off, int lane, float scale, float (&x)[D / 32]) {
  constexpr int H2 = Lane<D>::H2;
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    const int e0 = hh * (D / 2) + lane * H2;
    if constexpr (FMT == kKvBf16) {
      using T = typename Raw<2 * H2>::T;
      T raw;
      __nv_bfloat16* e = reinterpret_cast<__nv_bfloat16*>(&raw);
#pragma unroll
      for (int j = 0; j < H2; ++j) {
        e[j] = __float2bfloat16(x[hh * H2 + j]);
        x[hh * H2 + j] = __bfloat162float(e[j]);
      }
      *reinterpret_cast<T*>(part + off * 2 * D + kv_swizzle_byte(2 * e0, off, 2 * D)) = raw;
    } else if constexpr (FMT == kKvFp8) {
      using T = typename Raw<H2>::T;
      T raw;
      uint8_t* e = reinterpret_cast<uint8_t*>(&raw);
#pragma unroll
      for (int j = 0; j < H2; ++j) {
        e[j] = float_to_e4m3(x[hh * H2 + j] / scale);
        x[hh * H2 + j] = e4m3_to_float(e[j]) * scale;
      }
      *reinterpret_cast<T*>(part + off * D + kv_swizzle_byte(e0, off, D)) = raw;
    } else {
      constexpr int LPB = 16 / H2;       // lanes per 16-value block
      using T = typename Raw<(H2 / 2 > 0 ? H2 / 2 : 1)>::T;
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < H2; ++j) {
        x[hh * H2 + j] /= scale;
        amax = fmaxf(amax, fabsf(x[hh * H2 + j]));
      }
#pragma unroll
      for (int o = 1; o < LPB; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const uint8_t s8 = nvfp4_block_scale(amax);
      const float sf = e4m3_to_float(s8);
      if ((lane % LPB) == 0) part[kPage * (D / 2) + off * (D / 16) + e0 / 16] = s8;
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < H2; ++j) word |= e2m1_code(x[hh * H2 + j] / sf) << (4 * j);
      *reinterpret_cast<T*>(part + off * (D / 2) + kv_swizzle_byte(e0 / 2, off, D / 2)) = static_cast<T>(word);
      widen_e2m1<H2>(word, sf, scale, &x[hh * H2]);
    }
  }
}

template <int D, int FMT>
__device__ __forceinline__ void load_row(const uint8_t* part, int off, int lane, float scale, float (&x)[D / 32]) {
  constexpr int H2 = Lane<D>::H2;
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    const int e0 = hh * (D / 2) + lane * H2;
    if constexpr (FMT == kKvBf16) {
      using T = typename Raw<2 * H2>::T;
      const T raw = *reinterpret_cast<const T*>(part + off * 2 * D + kv_swizzle_byte(2 * e0, off, 2 * D));
      const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&raw);
#pragma unroll
      for (int j = 0; j < H2; ++j) x[hh * H2 + j] = __bfloat162float(e[j]);
    } else if constexpr (FMT == kKvFp8) {
      using T = typename Raw<H2>::T;
      const T raw = *reinterpret_cast<const T*>(part + off * D + kv_swizzle_byte(e0, off, D));
      const uint8_t* e = reinterpret_cast<const uint8_t*>(&raw);
#pragma unroll
      for (int j = 0; j < H2; ++j) x[hh * H2 + j] = e4m3_to_float(e[j]) * scale;
    } else {
      using T = typename Raw<(H2 / 2 > 0 ? H2 / 2 : 1)>::T;
      const float sf = e4m3_to_float(part[kPage * (D / 2) + off * (D / 16) + e0 / 16]);
      const T raw = *reinterpret_cast<const T*>(part + off * (D / 2) + kv_swizzle_byte(e0 / 2, off, D / 2));
      widen_e2m1<H2>(raw, sf, scale, &x[hh * H2]);
    }
  }
}

// Norm (per head, optional) and rotation in fp32; nothing is rounded in between.
template <int D>
__device__ __forceinline__ void norm_rope(float (&x)[D / 32], const __nv_bfloat16* w, float eps, bool plus_one,
                                          const float* cs, int lane) {
  constexpr int H2 = Lane<D>::H2, E = Lane<D>::E;
  if (w) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) ss += x[j] * x[j];
    const float inv = rsqrtf(warp_sum(ss) / D + eps);
    float g[E];
    load_bf16<D>(w, lane, g);
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = x[j] * inv * (plus_one ? 1.f + g[j] : g[j]);
  }
#pragma unroll
  for (int j = 0; j < H2; ++j) {
    const float c = cs[lane * H2 + j], s = cs[D / 2 + lane * H2 + j];
    const float a = x[j], b = x[H2 + j];
    x[j] = a * c - b * s;
    x[H2 + j] = b * c + a * s;
  }
}

// Running bound of the rows seen by this lane, and the CTA-wide end of it: codes and scale of one page and head.
template <int D>
struct Bound {
  float lo[D / 32], hi[D / 32];
  bool bad;                             // a key was not finite
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) { lo[j] = INFINITY; hi[j] = -INFINITY; }
    bad = false;
  }
  __device__ __forceinline__ void add(const float (&x)[D / 32]) {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      lo[j] = fminf(lo[j], x[j]);
      hi[j] = fmaxf(hi[j], x[j]);
      bad |= !(fabsf(x[j]) < INFINITY);
    }
  }
};

constexpr int kWarps = 4;

template <int D>
__device__ void finish_bound(const Bound<D>& bd, int8_t* codes, __nv_bfloat16* scale, float* smem) {
  constexpr int H2 = Lane<D>::H2;
  const int lane = lane_id(), warp = warp_id();
  float* slo = smem;                    // [kWarps][D]
  float* shi = smem + kWarps * D;
  __shared__ float smax[kWarps];
  __shared__ int sbad;
  if (threadIdx.x == 0) sbad = 0;
  __syncthreads();
#pragma unroll
  for (int hh = 0; hh < 2; ++hh)
#pragma unroll
    for (int j = 0; j < H2; ++j) {
      slo[warp * D + hh * (D / 2) + lane * H2 + j] = bd.lo[hh * H2 + j];
      shi[warp * D + hh * (D / 2) + lane * H2 + j] = bd.hi[hh * H2 + j];
    }
  if (bd.bad) sbad = 1;
  __syncthreads();
  constexpr int PER = D / (kWarps * 32);
  float c[PER], w[PER], amax = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = threadIdx.x * PER + i;
    float lo = slo[d], hi = shi[d];
#pragma unroll
    for (int k = 1; k < kWarps; ++k) { lo = fminf(lo, slo[k * D + d]); hi = fmaxf(hi, shi[k * D + d]); }
    c[i] = (lo + hi) * 0.5f;
    w[i] = (hi - lo) * 0.5f;
    amax = fmaxf(amax, fmaxf(fabsf(c[i]), w[i]));
  }
  amax = warp_max(amax);
  if (lane == 0) smax[warp] = amax;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kWarps; ++k) amax = fmaxf(amax, smax[k]);
  const bool bad = sbad != 0 || !(amax < INFINITY);     // (lo + hi or hi - lo may overflow)
  const int e = code_exp(amax);
  const float inv = pow2(-e);
  using T = typename Raw<PER>::T;
  T rc, rw;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    reinterpret_cast<int8_t*>(&rc)[i] = static_cast<int8_t>(bad ? 0 : code8(c[i], inv));
    reinterpret_cast<int8_t*>(&rw)[i] = static_cast<int8_t>(bad ? 0 : code8(w[i], inv));
  }
  reinterpret_cast<T*>(codes)[threadIdx.x] = rc;
  reinterpret_cast<T*>(codes + D)[threadIdx.x] = rw;
  if (threadIdx.x == 0) *scale = __float2bfloat16(bad ? INFINITY : pow2(e));
  __syncthreads();                      // smem is used again by the next run
}

// ------------------------------------------------------------------------------------------ append
// Grid: x = slabs of `slab` rows; y < Hk: the K vectors of kv head y, else four of the Hq + Hk q and v vectors.
// A K CTA owns the page runs that start in its slab (consecutive rows at consecutive slots of one page): its warps
// share the run's rows, and when the run ends at the page's last row the CTA also reads the rows written by earlier
// calls and writes the page's bound, so the bound costs no launch and no second pass over the new keys.
__device__ __forceinline__ int row_slot(const BlockAppendArgs& a, int t) {
  const int s = a.slot[t], p = a.pos[t];
  return (s < 0 || s >= a.slots || p < 0 || p >= a.max_pos) ? -1 : s;
}

template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32) block_append_kernel(const BlockAppendArgs a) {
  __shared__ float red[2 * kWarps * D];
  const int warp = warp_id(), lane = lane_id();
  const int t0 = blockIdx.x * a.slab, t1 = min(a.T, t0 + a.slab);
  const __nv_bfloat16* qkv = reinterpret_cast<const __nv_bfloat16*>(a.qkv);
  const int part = gqa_block_bytes(FMT, D, kPage) / 2;
  float x[D / 32];
  if (static_cast<int>(blockIdx.y) >= a.Hk) {
    const int v = (blockIdx.y - a.Hk) * kWarps + warp;
    if (v >= a.Hq + a.Hk) return;
    const bool is_q = v < a.Hq;
    for (int t = t0; t < t1; ++t) {
      const int src = is_q ? v : v + a.Hk;
      load_bf16<D>(qkv + static_cast<size_t>(t) * a.qkv_stride + static_cast<size_t>(src) * D, lane, x);
      if (is_q) {
        const int p = a.pos[t];
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.q_out) + (static_cast<size_t>(t) * a.Hq + v) * D;
        if (p >= 0 && p < a.max_pos) {
          norm_rope<D>(x, reinterpret_cast<const __nv_bfloat16*>(a.q_norm), a.eps, a.plus_one,
                       a.cos_sin + static_cast<size_t>(p) * D, lane);
        } else {
#pragma unroll
          for (int j = 0; j < D / 32; ++j) x[j] = 0.f;
        }
        store_bf16<D>(dst, lane, x);
      } else {
        const int s = row_slot(a, t);
        if (s < 0) continue;
        uint8_t* base = a.pool + (static_cast<size_t>(s / kPage) * a.Hk + (v - a.Hq)) * (2 * part) + part;
        store_row<D, FMT>(base, s % kPage, lane, a.v_scale, x);
      }
    }
    return;
  }
  const int h = blockIdx.y;
  for (int t = t0; t < t1; ++t) {
    const int s = row_slot(a, t);
    if (s < 0) continue;
    if (t > 0 && (s % kPage) != 0 && row_slot(a, t - 1) == s - 1) continue;      // inside a run that began before
    int n = 1;                            // rows of the run (at most a page)
    while (s % kPage + n < kPage && t + n < a.T && row_slot(a, t + n) == s + n) ++n;
    const int page = s / kPage, off = s % kPage;
    const bool last = off + n == kPage;
    uint8_t* base = a.pool + (static_cast<size_t>(page) * a.Hk + h) * (2 * part);
    Bound<D> bd;
    bd.reset();
    for (int i = warp; i < n; i += kWarps) {
      load_bf16<D>(qkv + static_cast<size_t>(t + i) * a.qkv_stride + static_cast<size_t>(a.Hq + h) * D, lane, x);
      norm_rope<D>(x, reinterpret_cast<const __nv_bfloat16*>(a.k_norm), a.eps, a.plus_one,
                   a.cos_sin + static_cast<size_t>(a.pos[t + i]) * D, lane);
      store_row<D, FMT>(base, off + i, lane, a.k_scale, x);
      bd.add(x);
    }
    if (!last) continue;
    for (int i = warp; i < off; i += kWarps) {
      load_row<D, FMT>(base, i, lane, a.k_scale, x);
      bd.add(x);
    }
    const size_t ph = static_cast<size_t>(page) * a.Hk + h;
    finish_bound<D>(bd, a.codes + ph * 2 * D, reinterpret_cast<__nv_bfloat16*>(a.scale) + ph, red);
  }
}

// Bounds of whole pages from their stored keys: one CTA per (page of the list, kv head).
template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32) block_summarize_kernel(const BlockAppendArgs a, const int* pages) {
  __shared__ float red[2 * kWarps * D];
  const int page = pages[blockIdx.x], h = blockIdx.y;
  if (page < 0 || page >= a.slots / kPage) return;
  const int part = gqa_block_bytes(FMT, D, kPage) / 2;
  const uint8_t* base = a.pool + (static_cast<size_t>(page) * a.Hk + h) * (2 * part);
  Bound<D> bd;
  bd.reset();
  float x[D / 32];
#pragma unroll 4
  for (int i = warp_id(); i < kPage; i += kWarps) {
    load_row<D, FMT>(base, i, lane_id(), a.k_scale, x);
    bd.add(x);
  }
  const size_t ph = static_cast<size_t>(page) * a.Hk + h;
  finish_bound<D>(bd, a.codes + ph * 2 * D, reinterpret_cast<__nv_bfloat16*>(a.scale) + ph, red);
}

// ------------------------------------------------------------------------------------------ select
constexpr int kSelThreads = 256;

// m16n8k32, 8-bit codes, 32-bit sums.
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// fp32 -> unsigned key of the same order (the scores are never NaN).
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One CTA per (group, kv head).  Scores: the 16 query rows' codes [q8 | |q8|] are the A operand (shared memory, rows
// padded by 64 bytes: conflict-free 16-byte reads), 8 pages' records of 2 D codes the B operand, read once from
// global memory, 16 bytes a thread; the products' k order is permuted alike on both sides so that a thread's 16 bytes are
// two instructions' fragments.  Then a radix selection over the scores' order keys in shared memory.
template <int D>
__global__ void __launch_bounds__(kSelThreads) block_select_kernel(const BlockSelectArgs a) {
  constexpr int RS = 2 * D + 64;        // bytes between query rows
  extern __shared__ __align__(16) uint8_t dyn[];
  int8_t* qs = reinterpret_cast<int8_t*>(dyn);                     // [16][RS]
  uint32_t* keys = reinterpret_cast<uint32_t*>(dyn + 16 * RS);     // [N]
  __shared__ float rscale[16];
  __shared__ int hist[256];
  __shared__ int wsum[kSelThreads / 32];
  __shared__ int sdigit, sneed;
  const int b = blockIdx.x, h = blockIdx.y;
  const int tid = threadIdx.x, warp = warp_id(), lane = lane_id();
  const int row = a.req_idx ? a.req_idx[b] : b;
  const int G = a.Hq / a.Hk, R = a.n_q * G;
  int* out = a.blocks + (static_cast<size_t>(b) * a.Hk + h) * a.budget;
  const int len = (row < 0 || row >= a.rows) ? 0 : min(a.kv_len[b], a.pt_stride * kPage);
  const int npages = len > 0 ? (len + kPage - 1) / kPage : 0;
  const int take = min(npages, a.budget);
  if (tid == 0) a.count[static_cast<size_t>(b) * a.Hk + h] = take;
  if (npages <= a.budget) {               // every page fits: nothing to rank
    for (int j = tid; j < a.budget; j += kSelThreads) out[j] = j < npages ? j : -1;
    return;
  }
  const int first_local = max(0, max(0, len - a.n_q) / kPage - (a.local - 1));
  const int lo = a.sink, n = first_local - a.sink;                   // candidates [lo, lo + n)
  const int want = a.budget - (npages - n);                          // how many of them are taken
  // ---- query codes: one warp per row
  for (int r = warp; r < 16; r += kSelThreads / 32) {
    float amax = 0.f;
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) +
                             static_cast<size_t>(b * a.n_q + r / G) * a.q_stride + (h * G + r % G) * D;
    constexpr int V = D / 32;
    float x[V];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      x[j] = r < R ? __bfloat162float(q[lane * V + j]) : 0.f;
      amax = fmaxf(amax, fabsf(x[j]));
      bad |= !(fabsf(x[j]) < INFINITY);
    }
    amax = warp_max(amax);
    bad = __any_sync(0xffffffffu, bad);
    const int e = code_exp(amax);
    const float inv = pow2(-e);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = bad ? 0 : code8(x[j], inv);
      qs[r * RS + lane * V + j] = static_cast<int8_t>(c);
      qs[r * RS + D + lane * V + j] = static_cast<int8_t>(abs(c));
    }
    if (lane == 0) rscale[r] = (r < R && !bad) ? pow2(e) : -1.f;
  }
  __syncthreads();
  // ---- scores: each warp 8 pages at a time
  const int g = lane >> 2, j4 = lane & 3;
  const float s0 = rscale[g], s1 = rscale[g + 8];
  const int* pt = a.page_table + static_cast<size_t>(row) * a.pt_stride;
  for (int p0 = warp * 8; p0 < n; p0 += kSelThreads / 32 * 8) {
    const int mine = min(p0 + g, n - 1);
    int phys = pt[lo + mine];
    const bool ok = phys >= 0 && phys < a.pages;
    if (!ok) phys = 0;
    const size_t ph = static_cast<size_t>(phys) * a.Hk + h;
    const uint4* rec = reinterpret_cast<const uint4*>(a.codes + ph * 2 * D) + j4;
    int c[4] = {0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < 2 * D / 64; ++u) {
      const uint4 bv = rec[4 * u];
      const uint4 x = *reinterpret_cast<const uint4*>(qs + g * RS + 64 * u + 16 * j4);
      const uint4 y = *reinterpret_cast<const uint4*>(qs + (g + 8) * RS + 64 * u + 16 * j4);
      mma_s8(c, x.x, y.x, x.y, y.y, bv.x, bv.y);
      mma_s8(c, x.z, y.z, x.w, y.w, bv.z, bv.w);
    }
    float m0 = -INFINITY, m1 = -INFINITY;           // pages p0 + 2 j4, p0 + 2 j4 + 1
    if (s0 > 0.f) { m0 = static_cast<float>(c[0]) * s0; m1 = static_cast<float>(c[1]) * s0; }
    if (s1 > 0.f) { m0 = fmaxf(m0, static_cast<float>(c[2]) * s1); m1 = fmaxf(m1, static_cast<float>(c[3]) * s1); }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
      m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
    }
    float sc = ok ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.scale)[ph]) : -1.f;
    const float sc0 = __shfl_sync(0xffffffffu, sc, 8 * j4), sc1 = __shfl_sync(0xffffffffu, sc, 8 * j4 + 4);
    if (g == 0) {
      const int p = p0 + 2 * j4;
      // a page whose keys are not finite ranks first, one outside the pool last
      const float v0 = sc0 < 0.f ? -INFINITY : sc0 == INFINITY ? INFINITY : m0 * sc0;
      const float v1 = sc1 < 0.f ? -INFINITY : sc1 == INFINITY ? INFINITY : m1 * sc1;
      if (p < n) keys[p] = order_key(v0);
      if (p + 1 < n) keys[p + 1] = order_key(v1);
    }
  }
  // ---- radix selection of the `want` largest keys, eight bits at a time
  uint32_t prefix = 0, mask = 0;
  int need = want;                                 // of the keys equal to the prefix so far
  if (want == 0) prefix = 0xffffffffu;             // above every key: nothing is taken
  for (int shift = want > 0 ? 24 : -8; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSelThreads) {
      const uint32_t k = keys[i];
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (warp == 0) {
      int own = 0, cnt[8];                         // lane l: digits 255 - 8 l .. 248 - 8 l
#pragma unroll
      for (int i = 0; i < 8; ++i) { cnt[i] = hist[255 - 8 * lane - i]; own += cnt[i]; }
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
          if (acc < need && need <= acc + cnt[i]) { sdigit = 255 - 8 * lane - i; sneed = need - acc; }
          acc += cnt[i];
        }
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(sdigit) << shift;
    mask |= 255u << shift;
    need = sneed;
  }
  __syncthreads();
  // ---- compaction in page order: thread t owns a contiguous run of candidates
  const int per = (n + kSelThreads - 1) / kSelThreads;
  const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
  int gt = 0, eq = 0;
  for (int i = i0; i < i1; ++i) {
    gt += keys[i] > prefix;
    eq += keys[i] == prefix;
  }
  // exclusive prefixes of both counts over the CTA (n < 2^16: packed in one word)
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
  for (int w = 0; w < kSelThreads / 32; ++w)
    if (w < warp) base += wsum[w];
  int gt_before = base >> 16, eq_before = base & 0xffff;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = keys[i];
    const bool sel = k > prefix || (k == prefix && eq_before < need);
    if (sel) out[a.sink + gt_before + min(eq_before, need)] = lo + i;
    gt_before += k > prefix;
    eq_before += k == prefix;
  }
  for (int i = tid; i < a.sink; i += kSelThreads) out[i] = i;
  for (int i = first_local + tid; i < npages; i += kSelThreads) out[a.sink + want + (i - first_local)] = i;
}

template <int D, int FMT>
cudaError_t append_launch(const BlockAppendArgs& a, cudaStream_t s) {
  const dim3 grid((a.T + a.slab - 1) / a.slab, a.Hk + (a.Hq + a.Hk + kWarps - 1) / kWarps);
  block_append_kernel<D, FMT><<<grid, kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}
template <int D, int FMT>
cudaError_t summarize_launch(const BlockAppendArgs& a, const int* pages, int n, cudaStream_t s) {
  block_summarize_kernel<D, FMT><<<dim3(n, a.Hk), kWarps * 32, 0, s>>>(a, pages);
  return cudaGetLastError();
}
template <int D>
cudaError_t select_launch(const BlockSelectArgs& a, cudaStream_t s) {
  const int smem = 16 * (2 * D + 64) + 4 * a.pt_stride;
  if (smem > 48 * 1024)
    IOB_CUDA_CHECK(cudaFuncSetAttribute(block_select_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  block_select_kernel<D><<<dim3(a.B, a.Hk), kSelThreads, smem, s>>>(a);
  return cudaGetLastError();
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
  // A decode step (few rows, each its own page) wants a CTA per row; a prefill wants fewer, longer CTAs.
  a.slab = a.T <= 256 ? 1 : 16;
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
