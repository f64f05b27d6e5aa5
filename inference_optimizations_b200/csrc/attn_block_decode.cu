// Attention over a list of cache pages: one group of query rows (n_q consecutive tokens x the G heads of one kv head,
// at most 16 rows) against the listed 64-token pages of its request, softmax over the visible positions of those
// pages, output and log-sum-exp.
//
// One cluster of C CTAs per (group, kv head).  The list is cut into tiles of ST tokens, dealt out in turn to the warps
// of the cluster; every warp runs a streaming softmax over its tiles by itself (one pass, running maximum m, sum l
// and output O in fp32 registers, no barrier) and the partial results are joined at the end, over distributed shared
// memory between CTAs, so a list is one launch whatever its split.  A warp's K and V tiles arrive by bulk copies in a
// ring of slots of its own.
//
// Both products have the cache on the M side of mma.sync m16n8k16: S^T = K Q^T (16 tokens x 8 rows) and
// O^T = V^T P^T (16 values x 8 rows), so a list of up to 8 query rows wastes no tensor row and holds half the
// registers that rows on the M side would take (D = 512: 128 of output and 64 of Q).  P goes from the accumulator
// layout to the operand layout by a register transpose.  The contraction index of a product may be permuted freely:
// a thread's 4 consecutive bytes of K (E4M3: 4 values, E2M1: 8) are used as the fragment they arrive in, with Q's
// columns permuted alike, and V's values as the row order of O^T they arrive in, undone when O is stored.  8-bit and
// 4-bit values are widened to f16 (exactly, block scales included) between shared memory and the fragments.
//
// Bound by the listed pages' bytes over bf16 and E4M3 caches (16 x 16 lists of 32 pages of D = 512, bf16: 143 us, 6.7
// TB/s; 64 x 8 lists of D = 128, E4M3: 49.5 us, 5.4 TB/s).  Over FP4 caches by latency that 8 warps an SM do not hide, no
// pipe being full (32 x 16 lists of 64 pages of D = 512: 266 us, 4.3 TB/s; issue slots and ALU under 50 %), for one user by
// launch and load latency (8 lists of 32 pages of D = 128: 7.9 us), for a prefill's groups by the path from L2 and the
// products (512 x 8 lists of 32 pages, 4.3 GB, of a 35k-token request: 375 us, 440 once the power cap takes the clock down).
#include "common.cuh"
#include "kernels.h"

namespace iob {
namespace {

constexpr int kPage = 64;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
// The running maximum may lag behind the true one by kLag in the base-2 exponentials: floating point keeps its relative
// precision, and the output is hardly ever rescaled after the first tiles.  P is rounded for the second product.  To 11
// bits (f16) over 8-bit and 4-bit caches: f16 has 2^-14 as its smallest normal number, so P carries 2^kUp there (at most
// 2^15 with the lag), weights down to 2^-26 of the largest keep their 11 bits, smaller ones are off by at most 2^-37 of it.
// Over a bf16 cache both operands are bf16, whose 8 bits would be the coarsest rounding of the whole kernel: P goes in
// as its leading 8 bits and what those left (kTerms products), 16 bits together.  Both terms of a weight that is not 0
// are positive, so that an infinite V stays what it is.
template <bool BF>
struct Weights {
  static constexpr float kLag = BF ? 8.f : 3.f, kUp = BF ? 0.f : 12.f;
  static constexpr int kTerms = BF ? 2 : 1;
};

template <int D_, int FMT_, int NR_, bool GROUP_>
struct Cfg {
  static constexpr int D = D_, FMT = FMT_, NR = NR_;       // NR: groups of 8 query rows
  // Several tokens of a request in one list: a row of V may be seen by some of the query rows only.  A form of its own,
  // because the little that it adds costs the other one its schedule (D = 512, FP4, 32 x 16 x 64 pages: 264 / 275 us).
  static constexpr bool GROUP = GROUP_;
  static constexpr bool BF = FMT == kKvBf16;
  static constexpr int RB = BF ? 2 * D : FMT == kKvFp8 ? D : D / 2;       // bytes of a row
  static constexpr int SC = FMT == kKvNvfp4 ? D / 16 : 0;                 // block scale bytes of a row
  // Bytes of a tile (at least 16 tokens, at most a page) and CTAs of an SM, which the registers bound (Q and O take
  // D / 8 * NR + D / 4 * NR of a thread's).  Larger tiles spread a step's fixed cost, more CTAs hide latencies.
  // Measured, 8 KB with 3 CTAs against 4 KB with 4 (D = 128, one column group): bf16 32 x 8 x 32 pages 43.4 / 45.4 us,
  // E4M3 64 x 8 x 32 pages 59.0 / 49.5 us, FP4 the same lists 46.6 / 40.9 us; two column groups, bf16 512 x 8 x 32
  // pages 375 / 478 us.  D = 512, FP4, 32 x 16 x 64 pages: 8 KB 266 us, 4 KB 306 us.
  static constexpr bool SMALL = D == 128 && NR == 1 && !BF;
  static constexpr int TB = SMALL ? 4096 : 8192;
  static constexpr int ST = TB / RB < 16 ? 16 : TB / RB < 64 ? TB / RB : 64;
  static constexpr int SUB = ST / 16;
  static constexpr int TPP = kPage / ST;                   // tiles of a page
  static constexpr int SLOT = ST * (RB + SC);              // K or V of a tile
  static constexpr int PART = kPage * (RB + SC);           // K or V of a page
  static constexpr int NCH = RB / 16 < 8 ? RB / 16 : 8;    // chunk swizzle span of a row
  static constexpr int NX = NCH / 2;
  static constexpr int KK = D / 16;                        // k16 steps of Q K^T
  static constexpr int MT = D / 16;                        // 16-value tiles of O^T
  static constexpr int DP = D + 4;                         // floats between rows of a partial output
  // Over FP4 caches Q's operand registers stay in shared memory where O takes 128 of a thread's: 64 more would leave
  // too few to overlap the conversions (D = 512, 32 x 16 x 64 pages: 266 against 280 us; over 8-bit and 16-bit caches,
  // bound by their bytes, registers are better: when it was chosen, D = 512, bf16, 16 x 16 x 32 pages 151 against 144 us).
  static constexpr bool QSM = D * NR >= 512 && FMT == kKvNvfp4;
  static constexpr int QB = QSM ? KK * NR * 256 : 0;       // bytes of it
  static constexpr int RES = SLOT > 12000 ? 1 : D * NR >= 512 ? 2 : SMALL ? 4 : 3;
  static constexpr int SMEM = 227 * 1024 / RES - 3584 - QB;     // of a CTA's rings, beside its static part and a list of 64
  static constexpr int NS = SMEM / (kWarps * SLOT) < 6 ? SMEM / (kWarps * SLOT) : 6;     // slots of a warp
  static constexpr int RING = NS * SLOT;
  static_assert(NS >= 2 && RING >= 8 * NR * DP * 4, "a warp's partial output takes the place of its ring");
  static constexpr int off_q = kWarps * RING;
  static constexpr int off_list = off_q + QB;
  static constexpr int smem(int cap) { return off_list + 8 * cap; }
};

template <bool BF>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  if constexpr (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Exact conversions to f16 pairs, free to be scheduled.
__device__ __forceinline__ uint32_t e4m3x2(uint32_t w) {            // low two bytes
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(w)));
  return r;
}
__device__ __forceinline__ void e4m3x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = e4m3x2(w);
  hi = e4m3x2(w >> 16);
}
__device__ __forceinline__ void e2m1x8(uint32_t w, uint32_t (&o)[4]) {      // byte k's two values -> o[k]
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}\n"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}
template <class C>
__device__ __forceinline__ uint32_t swz(int row, int chunk) {       // byte offset of a row's 16-byte chunk
  return row * C::RB + ((((chunk ^ row) & (C::NCH - 1)) | (chunk & ~(C::NCH - 1))) << 4);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (BF) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// Two query values as one register of an operand (bf16 as they are; f16 after the row's power of two).
template <bool BF>
__device__ __forceinline__ uint32_t q_pair(const __nv_bfloat16* q, float f) {
  if (!q) return 0u;
  const uint32_t raw = *reinterpret_cast<const uint32_t*>(q);
  if constexpr (BF) return raw;
  return pack16<false>(__uint_as_float(raw << 16) * f, __uint_as_float(raw & 0xffff0000u) * f);
}

// Words of stored V rows (block scales for an FP4 cache): the value with everything that is not finite cleared.
template <int FMT>
__device__ __forceinline__ uint32_t finite_word(uint32_t w) {
  if constexpr (FMT == kKvBf16) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
  } else {                                       // E4M3: NaN only
    w &= ~(__vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu));
  }
  return w;
}
// Clears what is not finite in the V rows [lo, hi) of a tile (one warp; a call, so that the main loop's registers and
// schedule do not depend on it).
template <class C>
__device__ __noinline__ void clear_odd(uint8_t* tile, int lo, int hi, int* found) {
  constexpr int ZB = C::FMT == kKvNvfp4 ? C::SC : C::RB;
  uint8_t* z = tile + (C::FMT == kKvNvfp4 ? C::ST * C::RB : 0);
  for (int i = max(0, lo) * ZB + 4 * lane_id(); i < min(C::ST, hi) * ZB; i += 128) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(z + i), f = finite_word<C::FMT>(w);
    if (w != f) {
      *reinterpret_cast<uint32_t*>(z + i) = f;
      *found = 1;
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}
// Value d of V row `row` of a page if it is not finite, else 0.
template <class C>
__device__ __forceinline__ float not_finite(const uint8_t* part, int row, int d) {
  if constexpr (C::BF) {
    const uint32_t v = *reinterpret_cast<const uint16_t*>(part + swz<C>(row, d / 8) + 2 * (d % 8));
    return (v & 0x7f80u) == 0x7f80u ? __uint_as_float(v << 16) : 0.f;
  } else {
    const uint8_t v = C::FMT == kKvFp8 ? part[swz<C>(row, d / 16) + d % 16] : part[kPage * C::RB + row * C::SC + d / 16];
    return (v & 0x7fu) == 0x7fu ? NAN : 0.f;
  }
}

// The list entries of one unit that name a page of the request and the pool, by one warp: logical pages in s_blk,
// physical pages in s_phys; returns their number.
__device__ __forceinline__ int valid_pages(const BlockDecodeArgs& a, int unit, int prow, int len, int* s_blk,
                                           int* s_phys) {
  const int lane = lane_id();
  const int* list = a.blocks + static_cast<size_t>(unit) * a.budget;
  int cnt = 0;
  for (int i0 = 0; i0 < a.budget; i0 += 32) {
    const int i = i0 + lane;
    const int blk = i < a.budget ? list[i] : -1;
    int phys = -1;
    if (blk >= 0 && blk < a.pt_stride && blk * kPage < len)
      phys = a.page_table[static_cast<size_t>(prow) * a.pt_stride + blk];
    const bool ok = phys >= 0 && phys < a.pages;
    const uint32_t m = __ballot_sync(0xffffffffu, ok);
    if (ok) {
      const int at = cnt + __popc(m & ((1u << lane) - 1));
      s_blk[at] = blk;
      s_phys[at] = phys;
    }
    cnt += __popc(m);
  }
  return cnt;
}

// Power of two that brings a query row's largest value into [2^14, 2^15), f16's last octave but one (one warp): values
// down to 2^-31 of the largest keep bf16's 8 bits.
template <int D>
__device__ __forceinline__ float row_pow2(const __nv_bfloat16* q) {
  float amax = 0.f;
  if (q)
    for (int d = 2 * lane_id(); d < D; d += 64) {
      const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(q + d);
      amax = fmaxf(amax, fmaxf(fabsf(__low2float(v)), fabsf(__high2float(v))));
    }
  amax = warp_max(amax);
  int x = 0;
  if (amax > 0.f && amax < INFINITY) frexpf(amax, &x);
  x = max(-126, x - 15);                         // (at most 128 - 15)
  return __int_as_float((x + 127) << 23);
}

template <class C>
__global__ void __launch_bounds__(kThreads, C::RES) block_decode_kernel(const BlockDecodeArgs a, const int csize,
                                                                        const int cap, const int rgroups) {
  using W = Weights<C::BF>;
  constexpr int NR = C::NR, ROWS = 8 * NR;
  extern __shared__ __align__(1024) uint8_t sm[];
  __shared__ __align__(8) uint64_t full[kWarps][C::NS];
  __shared__ float s_wm[kWarps][ROWS], s_wl[kWarps][ROWS], s_m[ROWS], s_l[ROWS], s_qf[ROWS], s_f[8][ROWS];
  __shared__ int s_cnt, s_abort, s_odd, s_odd_any;
  int* s_blk = reinterpret_cast<int*>(sm + C::off_list);
  int* s_phys = s_blk + cap;
  const int tid = threadIdx.x, warp = warp_id(), lane = lane_id();
  const int rank = blockIdx.x % csize, ur = blockIdx.x / csize;
  const int unit = ur / rgroups, r0 = (ur % rgroups) * ROWS;      // list, first query row of this cluster
  const int b = unit / a.Hk, h = unit % a.Hk;
  const int G = a.Hq / a.Hk, R = min(a.n_q * G - r0, ROWS);
  const int prow = a.req_idx ? a.req_idx[b] : b;
  const int len = (prow < 0 || prow >= a.rows) ? 0 : min(a.kv_len[b], a.pt_stride * kPage);
  const int q0 = len - a.n_q;                    // position of the group's first token (may be negative)
  auto q_row = [&](int r) -> const __nv_bfloat16* {
    if (r >= R) return nullptr;
    return reinterpret_cast<const __nv_bfloat16*>(a.q) + static_cast<size_t>(b * a.n_q + (r0 + r) / G) * a.q_stride +
           static_cast<size_t>(h * G + (r0 + r) % G) * C::D;
  };
  if (tid == 0) {
    s_abort = s_odd = s_odd_any = 0;
    for (int i = 0; i < kWarps * C::NS; ++i) mbar_init(&full[0][0] + i, 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    const int cnt = valid_pages(a, unit, prow, len, s_blk, s_phys);
    if (lane == 0) s_cnt = cnt;
  } else if constexpr (!C::BF) {
    for (int r = warp - 1; r < ROWS; r += kWarps - 1) {
      const float f = row_pow2<C::D>(q_row(r));
      if (lane == 0) s_qf[r] = f;
    }
  }
  __syncthreads();
  // ---- this warp's tiles: t0, t0 + step, ...; slot q of its ring sequence holds K (q even) or V of tile q / 2
  const int ntiles = s_cnt * C::TPP;
  const int step = csize * kWarps, t0 = warp * csize + rank;
  const int nk = ntiles > t0 ? (ntiles - t0 + step - 1) / step : 0;
  uint8_t* ring = sm + warp * C::RING;
  int itile = t0;                                // lane 0: the next tile to fetch, its K's place, which part is next
  const uint8_t* isrc = nullptr;
  bool ival = false;
  auto issue = [&](int slot) {
    uint8_t* dst = ring + slot * C::SLOT;
    mbar_expect_tx(&full[warp][slot], C::SLOT + a.never_bytes);
    const int in = itile % C::TPP;
    if (!ival) {
      isrc = a.pool + (static_cast<size_t>(s_phys[itile / C::TPP]) * a.Hk + h) * (2 * C::PART) + in * (C::ST * C::RB);
    } else {
      isrc += C::PART;
      itile += step;
    }
    ival = !ival;
    bulk_g2s(dst, isrc, C::SC == 0 || C::TPP == 1 ? C::SLOT : C::ST * C::RB, &full[warp][slot]);
    if constexpr (C::SC != 0 && C::TPP != 1)
      bulk_g2s(dst + C::ST * C::RB, isrc + kPage * C::RB - in * (C::ST * (C::RB - C::SC)), C::ST * C::SC,
               &full[warp][slot]);
  };
  if (lane == 0)
    for (int q = 0; q < C::NS && q < 2 * nk; ++q) issue(q);

  const int g = lane >> 2, j4 = lane & 3, mi = lane >> 3, ri = lane & 7;
  // ---- Q: column n of an operand is query row 8 n + g
  uint32_t qf[C::QSM ? 1 : C::KK][NR][2];
  uint2* s_q = reinterpret_cast<uint2*>(sm + C::off_q) + lane;      // [KK][NR][32]
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const __nv_bfloat16* q = q_row(8 * n + g);
    const float f = C::BF ? 1.f : 1.f / s_qf[8 * n + g];
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) {
      if (C::QSM && kk % kWarps != warp) continue;                  // shared: each warp prepares its part
      int d0, d1;
      if constexpr (C::BF) { d0 = 16 * kk + 2 * j4; d1 = d0 + 8; }
      else if constexpr (C::FMT == kKvFp8) { d0 = 16 * kk + 4 * j4; d1 = d0 + 2; }
      else { d0 = 32 * (kk / 2) + 8 * j4 + 4 * (kk % 2); d1 = d0 + 2; }
      const uint32_t x = q_pair<C::BF>(q ? q + d0 : nullptr, f), y = q_pair<C::BF>(q ? q + d1 : nullptr, f);
      if constexpr (C::QSM) {
        s_q[(kk * NR + n) * 32] = make_uint2(x, y);
      } else {
        qf[kk][n][0] = x;
        qf[kk][n][1] = y;
      }
    }
  }
  if constexpr (C::QSM) __syncthreads();
  auto q_at = [&](int kk, int n, uint32_t (&o)[2]) {
    if constexpr (C::QSM) {
      const uint2 v = s_q[(kk * NR + n) * 32];
      o[0] = v.x;
      o[1] = v.y;
    } else {
      o[0] = qf[kk][n][0];
      o[1] = qf[kk][n][1];
    }
  };
  // ---- softmax state of this thread's rows 8 n + 2 j4 + e (shared by the 8 lanes of equal j4)
  float scale[2 * NR], m[2 * NR], l[2 * NR];
#pragma unroll
  for (int i = 0; i < 2 * NR; ++i) {
    const int r = 8 * (i >> 1) + 2 * j4 + (i & 1);
    scale[i] = a.sm_scale * kLog2e * (C::BF ? 1.f : a.k_scale * s_qf[r]);
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  float acc[C::MT][NR][4];
#pragma unroll
  for (int t = 0; t < C::MT; ++t)
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[t][n][k] = 0.f;
  // Offsets of this lane's fragment rows: the chunk swizzle leaves NX of them (a load takes a pair of chunks), further
  // pairs lie at constant distances.
  uint32_t klane[C::NX], vlane[C::NX];
#pragma unroll
  for (int i = 0; i < C::NX; ++i) {
    klane[i] = swz<C>((mi & 1) * 8 + ri, 2 * i + (mi >> 1));
    vlane[i] = swz<C>((mi >> 1) * 8 + ri, 2 * i + (mi & 1));
  }

  int slot = 0, phase = 0;
  for (int k = 0; k < nk; ++k) {
    const int tile = t0 + k * step;
    const int base = s_blk[tile / C::TPP] * kPage + (tile % C::TPP) * C::ST;
    // ---- S^T = K Q^T
    if (!mbar_wait(&full[warp][slot], phase, &s_abort, a.status, kTimeoutProducer)) s_abort = 1;
    float s[C::SUB][NR][4];
    {
      const uint8_t* kp = ring + slot * C::SLOT;
      const uint32_t kb = smem_u32(kp);
#pragma unroll
      for (int u = 0; u < C::SUB; ++u)
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][n][e] = 0.f;
      if constexpr (C::BF) {
#pragma unroll
        for (int u = 0; u < C::SUB; ++u)
#pragma unroll
          for (int kk = 0; kk < C::KK; ++kk) {
            uint32_t r[4];
            ldsm4(r, kb + u * 16 * C::RB + klane[kk % C::NX] + kk / C::NX * (C::NCH * 16));
#pragma unroll
            for (int n = 0; n < NR; ++n) mma<true>(s[u][n], r, qf[kk][n]);
          }
      } else if constexpr (C::FMT == kKvFp8) {
#pragma unroll
        for (int u = 0; u < C::SUB; ++u)
#pragma unroll
          for (int i = 0; i < C::KK / 2; ++i) {
            uint32_t r[4];
            ldsm4(r, kb + u * 16 * C::RB + klane[i % C::NX] + i / C::NX * (C::NCH * 16));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t f[4];
              e4m3x4(r[2 * e], f[0], f[2]);
              e4m3x4(r[2 * e + 1], f[1], f[3]);
#pragma unroll
              for (int n = 0; n < NR; ++n) mma<false>(s[u][n], f, qf[2 * i + e][n]);
            }
          }
      } else {
        // block scales of the two tokens u * 16 + g (+ 8): of each pair of a chunk's bytes this thread uses one
        const uint8_t* ksc = kp + C::ST * C::RB + g * C::SC;
        const uint32_t selp = (j4 >> 1) | (2 + (j4 >> 1)) << 4;
        constexpr int NP = C::KK / 4;                        // pairs of 32-value chunks
        uint32_t q[4][NR][2];                                // (shared Q: read once for all the tile's tokens)
#pragma unroll
        for (int it = 0; it < NP * C::SUB; ++it) {
          const int u = C::QSM ? it % C::SUB : it / NP, i = C::QSM ? it / C::SUB : it % NP;
          if (!C::QSM || u == 0) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
              for (int n = 0; n < NR; ++n) q_at(4 * i + x, n, q[x][n]);
          }
          uint32_t r[4], sw[2];
          sw[0] = *reinterpret_cast<const uint32_t*>(ksc + u * 16 * C::SC + 4 * i);
          sw[1] = *reinterpret_cast<const uint32_t*>(ksc + (u * 16 + 8) * C::SC + 4 * i);
          ldsm4(r, kb + u * 16 * C::RB + klane[i % C::NX] + i / C::NX * (C::NCH * 16));
          const uint32_t sp[2] = {e4m3x2(prmt(sw[0], 0u, selp)), e4m3x2(prmt(sw[1], 0u, selp))};      // both chunks'
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t v[2][4];
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const uint32_t s2 = prmt(sp[o], 0u, e ? 0x3232u : 0x1010u);
              e2m1x8(r[2 * e + o], v[o]);
#pragma unroll
              for (int x = 0; x < 4; ++x) v[o][x] = hmul2_u32(v[o][x], s2);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const uint32_t f[4] = {v[0][2 * t], v[1][2 * t], v[0][2 * t + 1], v[1][2 * t + 1]};
#pragma unroll
              for (int n = 0; n < NR; ++n) mma<false>(s[u][n], f, q[2 * e + t][n]);
            }
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0 && 2 * k + C::NS < 2 * nk && !s_abort) issue(slot);
    if (++slot == C::NS) { slot = 0; phase ^= 1; }
    // ---- softmax over the tile's tokens u * 16 + g (+ 8)
    if (base + C::ST - 1 > q0) {                 // some row does not see all of them
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int vis = min(len, q0 + (r0 + 8 * n + 2 * j4 + e) / G + 1) - base - g;
#pragma unroll
          for (int u = 0; u < C::SUB; ++u) {
            if (16 * u >= vis) s[u][n][e] = -INFINITY;
            if (16 * u + 8 >= vis) s[u][n][2 + e] = -INFINITY;
          }
        }
    }
    float mt[2 * NR];
    bool over = false;
#pragma unroll
    for (int i = 0; i < 2 * NR; ++i) {
      float x = -INFINITY;
#pragma unroll
      for (int u = 0; u < C::SUB; ++u) x = fmaxf(x, fmaxf(s[u][i >> 1][i & 1], s[u][i >> 1][2 + (i & 1)]));
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
      mt[i] = x;
      over |= (x - m[i]) * scale[i] > W::kLag;      // (m = -inf: any finite score; a score of -inf never)
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int i = 0; i < 2 * NR; ++i) {
        const float mn = fmaxf(m[i], mt[i]);
        const float al = mn == -INFINITY ? 1.f : ex2((m[i] - mn) * scale[i]);
        m[i] = mn;
        l[i] *= al;
#pragma unroll
        for (int t = 0; t < C::MT; ++t) {
          acc[t][i >> 1][i & 1] *= al;
          acc[t][i >> 1][2 + (i & 1)] *= al;
        }
      }
    }
    uint32_t p[C::SUB][NR][W::kTerms][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const float c0 = m[2 * n] == -INFINITY ? 0.f : W::kUp - m[2 * n] * scale[2 * n];
      const float c1 = m[2 * n + 1] == -INFINITY ? 0.f : W::kUp - m[2 * n + 1] * scale[2 * n + 1];
#pragma unroll
      for (int u = 0; u < C::SUB; ++u) {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const float p0 = ex2(fmaf(s[u][n][2 * o], scale[2 * n], c0));
          const float p1 = ex2(fmaf(s[u][n][2 * o + 1], scale[2 * n + 1], c1));
          l[2 * n] += p0;
          l[2 * n + 1] += p1;
          const uint32_t b0 = __float_as_uint(p0), b1 = __float_as_uint(p1);
          const uint32_t w = C::BF ? prmt(b0, b1, 0x7632u) : pack16<C::BF>(p0, p1);
          p[u][n][0][o] = transpose8x8(w);                       // rows 8 n + g, tokens 2 j4, 2 j4 + 1 of the octet
          if constexpr (W::kTerms == 2) {
            constexpr float kLeast = 0x1p-40f;
            p[u][n][W::kTerms - 1][o] =
                transpose8x8(pack16<C::BF>(fmaxf(p0 - __uint_as_float(b0 & 0xffff0000u), p0 * kLeast),
                                           fmaxf(p1 - __uint_as_float(b1 & 0xffff0000u), p1 * kLeast)));
          }
        }
      }
    }
    // ---- O^T += V^T P^T
    if (!mbar_wait(&full[warp][slot], phase, &s_abort, a.status, kTimeoutProducer)) s_abort = 1;
    uint8_t* vp = ring + slot * C::SLOT;
    if (base + C::ST > len) {                    // rows past the cache's end may hold anything: cleared
      constexpr int ZB = C::FMT == kKvNvfp4 ? C::SC : C::RB;      // (an FP4 row is zero when its scales are)
      uint8_t* z = vp + (C::FMT == kKvNvfp4 ? C::ST * C::RB : 0);
      for (int i = max(0, len - base) * ZB + 4 * lane; i < C::ST * ZB; i += 128) *reinterpret_cast<uint32_t*>(z + i) = 0u;
      fence_proxy_async_smem();
      __syncwarp();
    }
    // A row of V that later tokens of the group see and earlier ones do not meets weights of 0 in this product, and 0 x inf
    // is NaN: values that are not finite are taken out here and added at the end, to the rows that see them.
    if constexpr (C::GROUP)
      if (base + C::ST - 1 > q0) clear_odd<C>(vp, q0 + 1 - base, len - base, &s_odd);
    const uint32_t vb = smem_u32(vp);
#pragma unroll
    for (int u = 0; u < C::SUB; ++u) {
      const uint32_t vt = vb + u * 16 * C::RB;
      if constexpr (C::BF) {
#pragma unroll
        for (int t = 0; t < C::MT; ++t) {
          uint32_t r[4];
          ldsm4t(r, vt + vlane[t % C::NX] + t / C::NX * (C::NCH * 16));
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int x = 0; x < W::kTerms; ++x) mma<true>(acc[t][n], r, p[u][n][x]);
        }
      } else if constexpr (C::FMT == kKvFp8) {
#pragma unroll
        for (int i = 0; i < C::MT / 2; ++i) {
          uint32_t r[4];
          ldsm4t(r, vt + vlane[i % C::NX] + i / C::NX * (C::NCH * 16));
#pragma unroll
          for (int e = 0; e < 2; ++e) {          // a 16-byte chunk: values 2 g (rows g) and 2 g + 1 (rows g + 8)
            uint32_t f[4];
            e4m3x4(prmt(r[e], 0u, 0x3120u), f[0], f[1]);
            e4m3x4(prmt(r[2 + e], 0u, 0x3120u), f[2], f[3]);
#pragma unroll
            for (int n = 0; n < NR; ++n) mma<false>(acc[2 * i + e][n], f, p[u][n][0]);
          }
        }
      } else {
        const uint8_t* vsc = vp + C::ST * C::RB + (u * 16 + 2 * j4) * C::SC;
#pragma unroll
        for (int i = 0; i < C::MT / 4; ++i) {
          uint32_t r[4], sv[2][2];               // [octet][token 2 j4, 2 j4 + 1]: scale bytes of the chunk pair
#pragma unroll
          for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int e = 0; e < 2; ++e) sv[o][e] = *reinterpret_cast<const uint32_t*>(vsc + (8 * o + e) * C::SC + 4 * i);
          ldsm4t(r, vt + vlane[i % C::NX] + i / C::NX * (C::NCH * 16));
          // scales of this lane's block in the two chunks, as pairs of the two tokens
          const uint32_t pr[2] = {prmt(sv[0][0], sv[0][1], 0x6240u + (lane >> 4) * 0x1111u),
                                  prmt(sv[1][0], sv[1][1], 0x6240u + (lane >> 4) * 0x1111u)};
#pragma unroll
          for (int e = 0; e < 2; ++e) {          // a chunk of 32 values: 4 g + {0 .. 3}
            uint32_t v[2][4];
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const uint32_t s2 = e4m3x2(e ? pr[o] >> 16 : pr[o]);
              uint32_t w[4];                     // (0, 1) (2, 3) of token 2 j4, then of 2 j4 + 1
              e2m1x8(r[2 * o + e], w);
              v[o][0] = prmt(w[0], w[2], 0x5410u);
              v[o][1] = prmt(w[0], w[2], 0x7632u);
              v[o][2] = prmt(w[1], w[3], 0x5410u);
              v[o][3] = prmt(w[1], w[3], 0x7632u);
#pragma unroll
              for (int x = 0; x < 4; ++x) v[o][x] = hmul2_u32(v[o][x], s2);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const uint32_t f[4] = {v[0][2 * t], v[0][2 * t + 1], v[1][2 * t], v[1][2 * t + 1]};
#pragma unroll
              for (int n = 0; n < NR; ++n) mma<false>(acc[4 * i + 2 * e + t][n], f, p[u][n][0]);
            }
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0 && 2 * k + 1 + C::NS < 2 * nk && !s_abort) issue(slot);
    if (++slot == C::NS) { slot = 0; phase ^= 1; }
  }
  // A wait that ran out in some warp: this one may have copies under way that it did not wait for.  It waits for the last
  // of each slot, with the same limit, before anything takes their place or the CTA ends; the group's result is NaN.
  const bool lost = __any_sync(0xffffffffu, *const_cast<volatile int*>(&s_abort));
  bool idle = true;
  if (lost) {
    const int issued = __shfl_sync(0xffffffffu, 2 * ((itile - t0) / step) + (ival ? 1 : 0), 0);
    for (int q = max(0, issued - C::NS); idle && q < issued; ++q)
      idle = __all_sync(0xffffffffu, mbar_wait(&full[warp][q % C::NS], (q / C::NS) & 1, nullptr, a.status, kTimeoutProducer));
  }
  // ---- partial result of the warp in place of its ring, which is idle
  float* wO = reinterpret_cast<float*>(ring);                     // [ROWS][DP]
#pragma unroll
  for (int i = 0; i < 2 * NR; ++i) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    const int r = 8 * (i >> 1) + 2 * j4 + (i & 1);
    if (g == 0) {
      s_wm[warp][r] = m[i] * scale[i] - W::kUp;
      s_wl[warp][r] = lost ? NAN : l[i];
    }
    if (r < R && idle) {
#pragma unroll
      for (int t = 0; t < C::MT; ++t) {
        int d, dn;                               // values of rows g, g + 8 of the tile
        if constexpr (C::BF) { d = 16 * t + g; dn = 8; }
        else if constexpr (C::FMT == kKvFp8) { d = 16 * t + 2 * g; dn = 1; }
        else { d = 32 * (t >> 1) + 4 * g + 2 * (t & 1); dn = 1; }
        wO[r * C::DP + d] = acc[t][i >> 1][i & 1];
        wO[r * C::DP + d + dn] = acc[t][i >> 1][2 + (i & 1)];
      }
    }
  }
  __syncthreads();
  // ---- the CTA's partial result, in place of warp 0's
  if (tid < ROWS) {
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_wm[w][tid]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(s_wm[w][tid] - (M == -INFINITY ? 0.f : M));
      s_f[w][tid] = f;
      L += f * s_wl[w][tid];
    }
    s_m[tid] = M;
    s_l[tid] = L;
  }
  __syncthreads();
  for (int i = tid; i < R * (C::D / 4); i += kThreads) {
    const int row = i / (C::D / 4), at = 4 * (row * C::DP + 4 * (i % (C::D / 4)));
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_f[w][row];
      const float4 v = *reinterpret_cast<const float4*>(sm + w * C::RING + at);
      if (f != 0.f) {
        o.x += f * v.x;
        o.y += f * v.y;
        o.z += f * v.z;
        o.w += f * v.w;
      }
    }
    *reinterpret_cast<float4*>(sm + at) = o;
  }
  // ---- join of the cluster: every CTA finishes its share of the R x D outputs
  if (csize > 1) cluster_sync_all();
  else __syncthreads();
  // (the CTAs' statistics are fetched by as many threads, the outputs' parts all before their sum: one remote latency
  // each, not one per CTA)
  const uint32_t ao = smem_u32(sm);
  static_assert(8 * ROWS <= kThreads && 8 * ROWS * 4 <= C::RING, "a thread per CTA and row");
  float(*s_cl)[ROWS] = reinterpret_cast<float(*)[ROWS]>(sm + C::RING);      // (the second warp's ring is free by now)
  if (tid < csize * ROWS) {
    const int c = tid / ROWS, r = tid % ROWS;
    const uint32_t vm = ld_cluster_u32(mapa_shared(smem_u32(&s_m[r]), c));
    const uint32_t vl = ld_cluster_u32(mapa_shared(smem_u32(&s_l[r]), c));
    const uint32_t odd = C::GROUP ? ld_cluster_u32(mapa_shared(smem_u32(&s_odd), c)) : 0u;
    s_f[c][r] = __uint_as_float(vm);
    s_cl[c][r] = __uint_as_float(vl);
    if (odd != 0u) s_odd_any = 1;
  }
  __syncthreads();
  if (tid < ROWS) {
    float M = -INFINITY, L = 0.f;
    for (int c = 0; c < csize; ++c) M = fmaxf(M, s_f[c][tid]);
    const float ms = M == -INFINITY ? 0.f : M;
    for (int c = 0; c < csize; ++c) {
      const float f = ex2(s_f[c][tid] - ms);
      s_f[c][tid] = f;
      L += f * s_cl[c][tid];
    }
    const float inv = L == 0.f ? 0.f : (C::BF ? 1.f : a.v_scale) / L;
    for (int c = 0; c < csize; ++c) s_f[c][tid] *= inv;
    if (rank == 0 && tid < R)
      a.lse[static_cast<size_t>(b * a.n_q + (r0 + tid) / G) * a.Hq + h * G + (r0 + tid) % G] =
          L == 0.f ? -INFINITY : 0.6931471805599453f * (M + log2f(L));
  }
  __syncthreads();
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out);
  for (int i = rank * kThreads + tid; i < R * (C::D / 4); i += csize * kThreads) {
    const int row = i / (C::D / 4), d = 4 * (i % (C::D / 4));
    float4 v[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < csize) v[c] = ld_cluster_f4(mapa_shared(ao + 4 * (row * C::DP + d), c));
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float f = c < csize ? s_f[c][row] : 0.f;
      if (f != 0.f) {
        o.x += f * v[c].x;
        o.y += f * v[c].y;
        o.z += f * v[c].z;
        o.w += f * v[c].w;
      }
    }
    if (C::GROUP && s_odd_any) {                           // V that is not finite, of the group's own tokens up to this row's
      const int last = min(len - 1, q0 + (r0 + row) / G);
      for (int pos = max(0, q0 + 1); pos <= last; ++pos)
        for (int j = 0; j < s_cnt; ++j)
          if (s_blk[j] == pos / kPage) {
            const uint8_t* part = a.pool + (static_cast<size_t>(s_phys[j]) * a.Hk + h) * (2 * C::PART) + C::PART;
            o.x += not_finite<C>(part, pos % kPage, d);
            o.y += not_finite<C>(part, pos % kPage, d + 1);
            o.z += not_finite<C>(part, pos % kPage, d + 2);
            o.w += not_finite<C>(part, pos % kPage, d + 3);
          }
    }
    uint2 raw;
    raw.x = pack16<true>(o.x, o.y);
    raw.y = pack16<true>(o.z, o.w);
    *reinterpret_cast<uint2*>(out + (static_cast<size_t>(b * a.n_q + (r0 + row) / G) * a.Hq + h * G + (r0 + row) % G) *
                                        C::D + d) = raw;
  }
  if (csize > 1) cluster_sync_all();             // a CTA's partial results are read until here
}

template <class C>
cudaError_t launch_c(const BlockDecodeArgs& a, int rgroups, cudaStream_t s) {
  // Few lists: each is split over a cluster, as far as the SMs have room for all its CTAs at once and a CTA keeps two
  // pages.
  const int units = a.B * a.Hk * rgroups;
  int cs = 1;
  while (cs < 8 && units * (cs + 1) <= 148 * C::RES && a.budget >= 2 * (cs + 1)) ++cs;
  // (the limit is the longest list's, the same in every call: calls of several host threads do not lower it)
  static_assert(C::smem(kBlockMaxList) + 4096 <= 227 * 1024, "the longest list fits beside the rings");
  auto k = block_decode_kernel<C>;
  IOB_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem(kBlockMaxList)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(units) * cs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::smem(a.budget);
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
    cfg.gridDim.x = static_cast<unsigned>(units) * cs;
  }
  return cudaLaunchKernelEx(&cfg, k, a, cs, a.budget, rgroups);
}

template <int D, int FMT, int NR>
cudaError_t launch_r(const BlockDecodeArgs& a, int rgroups, cudaStream_t s) {
  return a.n_q > 1 ? launch_c<Cfg<D, FMT, NR, true>>(a, rgroups, s) : launch_c<Cfg<D, FMT, NR, false>>(a, rgroups, s);
}

template <int D, int FMT>
cudaError_t launch(const BlockDecodeArgs& a, cudaStream_t s) {
  // Up to 8 query rows: one column group.  More: two, or for D = 512, where a warp has no registers for two, two
  // clusters that read the same pages.
  const int rows = a.n_q * (a.Hq / a.Hk);
  if (rows <= 8) return launch_r<D, FMT, 1>(a, 1, s);
  if constexpr (D == 512) return launch_r<D, FMT, 1>(a, 2, s);
  else return launch_r<D, FMT, 2>(a, 1, s);
}

}  // namespace

cudaError_t block_decode(const BlockDecodeArgs& a, cudaStream_t s) {
  if (a.B == 0) return cudaSuccess;
  if (a.Hk < 1 || a.Hq % a.Hk || a.n_q < 1 || a.n_q * (a.Hq / a.Hk) > 16 || a.budget < 1 || a.budget > kBlockMaxList ||
      !(a.sm_scale > 0.f) || (a.fmt != kKvBf16 && !(a.k_scale > 0.f)))
    return cudaErrorInvalidValue;
  switch (a.D * 4 + a.fmt) {
    case 128 * 4 + kKvBf16: return launch<128, kKvBf16>(a, s);
    case 128 * 4 + kKvFp8: return launch<128, kKvFp8>(a, s);
    case 128 * 4 + kKvNvfp4: return launch<128, kKvNvfp4>(a, s);
    case 256 * 4 + kKvBf16: return launch<256, kKvBf16>(a, s);
    case 256 * 4 + kKvFp8: return launch<256, kKvFp8>(a, s);
    case 256 * 4 + kKvNvfp4: return launch<256, kKvNvfp4>(a, s);
    case 512 * 4 + kKvBf16: return launch<512, kKvBf16>(a, s);
    case 512 * 4 + kKvFp8: return launch<512, kKvFp8>(a, s);
    case 512 * 4 + kKvNvfp4: return launch<512, kKvNvfp4>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace iob
