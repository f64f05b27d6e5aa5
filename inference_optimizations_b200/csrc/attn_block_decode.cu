// Attention over a list of cache pages: one group of query rows (n_q consecutive tokens x the G heads of one kv head,
// at most 16 rows) against the listed 64-token pages of its request, softmax over the visible positions of those
// pages, output and log-sum-exp.
//
// One cluster of C CTAs per (group, kv head); the CTAs share the list, each runs a streaming softmax over its pages
// (running maximum m, sum l and output O in fp32, one pass), and the partial results are joined over distributed
// shared memory, so a list is one launch whatever its split.  A page's K and V arrive as one bulk copy into a ring of
// stages.  Per tile: S = Q K^T (warps split the tokens, and from D = 256 on also the head dim), scores through shared
// memory to a row-wise softmax, P back as the A operand, O += P V (warps split the head dim).
//
// mma.sync m16n8k16 carries both products: a list of single-token queries has at most 16 rows, so the tensor work is
// small against the bytes, and register operands let a page's 8-bit and 4-bit values be widened (exactly, to f16) on
// their way from shared memory into the fragments.  K order inside a product is free, so a thread's 4 consecutive
// bytes (E4M3: 4 values, E2M1: 8) are used as the fragment they arrive in, with Q's columns permuted alike.
#include "common.cuh"
#include "kernels.h"

namespace iob {
namespace {

constexpr int kPage = 64;
constexpr int kRows = 16;

template <int D_, int FMT_>
struct Cfg {
  static constexpr int D = D_, FMT = FMT_;
  static constexpr bool BF = FMT == kKvBf16;
  static constexpr int NW = D == 128 ? 4 : 8;              // warps
  static constexpr int NT = NW * 32;
  static constexpr int DS = NW / 4;                        // head-dim splits of Q K^T (four token groups)
  static constexpr int TT = (BF && D == 512) ? 32 : 64;    // tokens per tile
  static constexpr int RB = BF ? 2 * D : FMT == kKvFp8 ? D : D / 2;
  static constexpr int SC = FMT == kKvNvfp4 ? D / 16 : 0;  // scale bytes per row
  static constexpr int PART = TT * (RB + SC);              // one of K, V of a tile
  static constexpr int STAGE = 2 * PART;
  static constexpr int NS = STAGE <= 20480 ? 4 : FMT == kKvNvfp4 ? 2 : 3;
  static constexpr int NCH = RB / 16 < 8 ? RB / 16 : 8;    // chunk swizzle span of a row
  static constexpr int SST = TT + (DS == 1 ? 8 : 16);      // floats between score rows
  static constexpr int PST = TT + 8;                       // 16-bit values between P rows
  static constexpr int KK = D / DS / 16;                   // k16 steps of a warp's share of Q K^T
  static constexpr int N8 = TT / 32;                       // 8-token tiles of a token group
  static constexpr int DW = D / NW;                        // output columns of a warp
  static constexpr int NO = DW / 8;
  static constexpr int off_s = NS * STAGE;
  static constexpr int off_p = off_s + DS * kRows * SST * 4;
  static constexpr int off_list = off_p + kRows * PST * 2;
  static constexpr int smem(int cap) { return off_list + 8 * cap; }
  // CTAs that share an SM: by shared memory, at most 4
  static constexpr int RES = 230000 / (off_list + 3072) < 4 ? 230000 / (off_list + 3072) : 4;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// Four E4M3 bytes -> (bytes 0, 1) and (bytes 2, 3) as f16x2.
__device__ __forceinline__ void e4m3x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = e4m3x2_to_f16x2(static_cast<uint16_t>(w));
  hi = e4m3x2_to_f16x2(static_cast<uint16_t>(w >> 16));
}
template <class C>
__device__ __forceinline__ uint32_t swz(int row, int chunk) {       // byte offset of a row's 16-byte chunk in a part
  return row * C::RB + ((((chunk ^ row) & (C::NCH - 1)) | (chunk & ~(C::NCH - 1))) << 4);
}

// Two query values as one register of the A operand (bf16 as they are; f16 after the row's power of two).
template <bool BF>
__device__ __forceinline__ uint32_t q_pair(const __nv_bfloat16* q, float f) {
  if (!q) return 0u;
  const uint32_t raw = *reinterpret_cast<const uint32_t*>(q);
  if constexpr (BF) return raw;
  const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&raw);
  const __half2 h = __floats2half2_rn(__low2float(v) * f, __high2float(v) * f);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <class C>
__global__ void __launch_bounds__(C::NT, C::RES) block_decode_kernel(const BlockDecodeArgs a, const int csize, const int cap) {
  extern __shared__ __align__(1024) uint8_t sm[];
  __shared__ __align__(8) uint64_t full[C::NS];
  __shared__ float s_alpha[kRows], s_m[kRows], s_l[kRows], s_qf[kRows], s_f[8][kRows];
  __shared__ int s_cnt, s_abort;
  float* sS = reinterpret_cast<float*>(sm + C::off_s);
  uint16_t* sP = reinterpret_cast<uint16_t*>(sm + C::off_p);
  int* s_blk = reinterpret_cast<int*>(sm + C::off_list);
  int* s_phys = s_blk + cap;

  const int tid = threadIdx.x, warp = warp_id(), lane = lane_id();
  const int unit = blockIdx.x / csize, rank = blockIdx.x % csize;
  const int b = unit / a.Hk, h = unit % a.Hk;
  const int G = a.Hq / a.Hk, R = a.n_q * G;
  const int prow = a.req_idx ? a.req_idx[b] : b;
  const int len = (prow < 0 || prow >= a.rows) ? 0 : min(a.kv_len[b], a.pt_stride * kPage);
  const int q0 = len - a.n_q;                    // position of the group's first token (may be negative)

  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < C::NS; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  // ---- this CTA's pages: list entries rank, rank + csize, ...; entries outside the request or the pool drop out
  if (warp == 0) {
    const int* list = a.blocks + static_cast<size_t>(unit) * a.budget;
    int cnt = 0;
    for (int i0 = rank; i0 < a.budget; i0 += 32 * csize) {
      const int i = i0 + lane * csize;
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
    if (lane == 0) s_cnt = cnt;
  } else if constexpr (!C::BF) {
    // ---- powers of two that bring every query row into f16's range
    for (int r = warp - 1; r < kRows; r += C::NW - 1) {
      float amax = 0.f;
      if (r < R) {
        const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) +
                                 static_cast<size_t>(b * a.n_q + r / G) * a.q_stride + (h * G + r % G) * C::D;
        for (int d = lane; d < C::D; d += 32) amax = fmaxf(amax, fabsf(__bfloat162float(q[d])));
      }
      amax = warp_max(amax);
      int x = 0;
      if (amax > 0.f && amax < INFINITY) frexpf(amax, &x);
      x = max(-100, min(100, x));
      if (lane == 0) s_qf[r] = __int_as_float((x + 127) << 23);
    }
  }
  __syncthreads();
  constexpr int TPP = kPage / C::TT;             // tiles per page
  const int ntiles = s_cnt * TPP;
  auto issue = [&](int tile) {                   // one thread
    const int st = tile % C::NS;
    const uint8_t* src = a.pool + (static_cast<size_t>(s_phys[tile / TPP]) * a.Hk + h) * (C::STAGE * TPP);
    uint8_t* dst = sm + st * C::STAGE;
    mbar_expect_tx(&full[st], C::STAGE);
    if constexpr (TPP == 1) {
      bulk_g2s(dst, src, C::STAGE, &full[st]);
    } else {
      src += (tile % TPP) * C::PART;
      bulk_g2s(dst, src, C::PART, &full[st]);
      bulk_g2s(dst + C::PART, src + TPP * C::PART, C::PART, &full[st]);
    }
  };
  if (tid == 0)
    for (int i = 0; i < C::NS && i < ntiles; ++i) issue(i);

  // ---- Q fragments of this warp's head-dim share
  const int g = lane >> 2, j4 = lane & 3;
  const int tg = warp & 3, dh = warp >> 2;
  uint32_t qf[C::KK][4];
  {
    const __nv_bfloat16* qr[2];
    float f[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = g + 8 * k;
      qr[k] = r < R ? reinterpret_cast<const __nv_bfloat16*>(a.q) +
                          static_cast<size_t>(b * a.n_q + r / G) * a.q_stride + (h * G + r % G) * C::D +
                          dh * (C::D / C::DS)
                    : nullptr;
      f[k] = C::BF ? 1.f : 1.f / s_qf[r];
    }
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) {
      int d0, d1;
      if constexpr (C::BF) { d0 = 16 * kk + 2 * j4; d1 = d0 + 8; }
      else if constexpr (C::FMT == kKvFp8) { d0 = 16 * kk + 4 * j4; d1 = d0 + 2; }
      else { d0 = 32 * (kk / 2) + 8 * j4 + 4 * (kk % 2); d1 = d0 + 2; }
      qf[kk][0] = q_pair<C::BF>(qr[0] ? qr[0] + d0 : nullptr, f[0]);
      qf[kk][1] = q_pair<C::BF>(qr[1] ? qr[1] + d0 : nullptr, f[1]);
      qf[kk][2] = q_pair<C::BF>(qr[0] ? qr[0] + d1 : nullptr, f[0]);
      qf[kk][3] = q_pair<C::BF>(qr[1] ? qr[1] + d1 : nullptr, f[1]);
    }
  }
  // ---- softmax state: row srow is shared by TPR consecutive threads
  constexpr int TPR = C::NT / kRows;
  const int srow = tid / TPR, sc0 = 2 * (tid % TPR);
  const int st_tok = srow < R ? srow / G : 0;
  const float ks = C::BF ? 1.f : a.k_scale * s_qf[srow];
  const float s_scale = a.sm_scale * ks * 1.4426950408889634f;
  float m_run = -INFINITY, l_run = 0.f;
  float acc[C::NO][4];
#pragma unroll
  for (int i = 0; i < C::NO; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[i][k] = 0.f;
  const uint32_t smb = smem_u32(sm);

  for (int tile = 0; tile < ntiles; ++tile) {
    const int st = tile % C::NS;
    if (!mbar_wait(&full[st], (tile / C::NS) & 1, &s_abort, a.status, kTimeoutProducer)) s_abort = 1;
    const uint32_t kb = smb + st * C::STAGE, vb = kb + C::PART;
    const int base = s_blk[tile / TPP] * kPage + (tile % TPP) * C::TT;
    // ---- S = Q K^T
    float s[C::N8][4];
#pragma unroll
    for (int n = 0; n < C::N8; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[n][k] = 0.f;
    {
      const int c0 = dh * (C::RB / 16 / C::DS);
      const int mi = lane >> 3, ri = lane & 7;
      if constexpr (C::BF) {
#pragma unroll
        for (int kk = 0; kk < C::KK; kk += 2 / C::N8) {
          uint32_t r[4];
          if constexpr (C::N8 == 2) {
            ldsm4(r, kb + swz<C>(tg * 16 + (mi >> 1) * 8 + ri, c0 + 2 * kk + (mi & 1)));
            mma_bf16(s[0], qf[kk], r[0], r[1]);
            mma_bf16(s[1], qf[kk], r[2], r[3]);
          } else {
            ldsm4(r, kb + swz<C>(tg * 8 + ri, c0 + 2 * kk + mi));
            mma_bf16(s[0], qf[kk], r[0], r[1]);
            mma_bf16(s[0], qf[kk + 1], r[2], r[3]);
          }
        }
      } else if constexpr (C::FMT == kKvFp8) {
#pragma unroll
        for (int kk = 0; kk < C::KK; kk += 2) {
          uint32_t r[4], lo, hi;
          ldsm4(r, kb + swz<C>(tg * 16 + (mi >> 1) * 8 + ri, c0 + kk + (mi & 1)));
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              e4m3x4(r[2 * n + k], lo, hi);
              mma_f16(s[n], qf[kk + k], lo, hi);
            }
        }
      } else {
        const uint8_t* ksc = sm + st * C::STAGE + kPage * C::RB;
#pragma unroll
        for (int cc = 0; cc < C::KK / 2; cc += 2) {
          uint32_t r[4], v[4];
          ldsm4(r, kb + swz<C>(tg * 16 + (mi >> 1) * 8 + ri, c0 + cc + (mi & 1)));
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t sb = ksc[(tg * 16 + n * 8 + g) * C::SC + 2 * (c0 + cc + k) + (j4 >> 1)];
              const uint32_t s2 = e4m3x2_to_f16x2(static_cast<uint16_t>(sb | (sb << 8)));
              e2m1x8_to_f16x2x4(r[2 * n + k], v);
              mma_f16(s[n], qf[2 * (cc + k)], hmul2_u32(v[0], s2), hmul2_u32(v[1], s2));
              mma_f16(s[n], qf[2 * (cc + k) + 1], hmul2_u32(v[2], s2), hmul2_u32(v[3], s2));
            }
        }
      }
    }
    float* srowp = sS + dh * kRows * C::SST;
#pragma unroll
    for (int n = 0; n < C::N8; ++n) {
      const int col = (tg * C::N8 + n) * 8 + 2 * j4;
      *reinterpret_cast<float2*>(srowp + g * C::SST + col) = make_float2(s[n][0], s[n][1]);
      *reinterpret_cast<float2*>(srowp + (g + 8) * C::SST + col) = make_float2(s[n][2], s[n][3]);
    }
    __syncthreads();
    // ---- softmax of the tile's scores; value rows past the cache's end are cleared (they may hold anything)
    {
      constexpr int NI = C::TT / (2 * TPR);
      float2 x[NI];
      float mt = -INFINITY;
      const int vis = srow < R ? min(len, q0 + st_tok + 1) - base : 0;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int col = sc0 + i * 2 * TPR;
        x[i] = *reinterpret_cast<const float2*>(sS + srow * C::SST + col);
        if constexpr (C::DS == 2) {
          const float2 y = *reinterpret_cast<const float2*>(sS + (kRows + srow) * C::SST + col);
          x[i].x += y.x;
          x[i].y += y.y;
        }
        x[i].x = col < vis ? x[i].x * s_scale : -INFINITY;
        x[i].y = col + 1 < vis ? x[i].y * s_scale : -INFINITY;
        mt = fmaxf(mt, fmaxf(x[i].x, x[i].y));
      }
#pragma unroll
      for (int o = 1; o < TPR; o <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
      const float m_new = fmaxf(m_run, mt);
      const float ms = m_new == -INFINITY ? 0.f : m_new;
      const float al = ex2(m_run - ms);
      m_run = m_new;
      l_run *= al;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const float p0 = ex2(x[i].x - ms), p1 = ex2(x[i].y - ms);
        l_run += p0 + p1;
        uint32_t raw;
        if constexpr (C::BF) {
          const __nv_bfloat162 v = __floats2bfloat162_rn(p0, p1);
          raw = *reinterpret_cast<const uint32_t*>(&v);
        } else {
          const __half2 v = __floats2half2_rn(p0, p1);
          raw = *reinterpret_cast<const uint32_t*>(&v);
        }
        *reinterpret_cast<uint32_t*>(sP + srow * C::PST + sc0 + i * 2 * TPR) = raw;
      }
      if (tid % TPR == 0) s_alpha[srow] = al;
      if (base + C::TT > len) {
        uint8_t* v = sm + st * C::STAGE + C::PART;
        constexpr int ZB = C::FMT == kKvNvfp4 ? C::SC : C::RB;      // an FP4 row is zero when its scales are
        uint8_t* z = v + (C::FMT == kKvNvfp4 ? C::TT * C::RB : 0);
        for (int i = max(0, len - base) * ZB + 4 * tid; i < C::TT * ZB; i += 4 * C::NT)
          *reinterpret_cast<uint32_t*>(z + i) = 0u;
        fence_proxy_async_smem();
      }
    }
    __syncthreads();
    // ---- O = alpha O + P V
    {
      const float al0 = s_alpha[g], al1 = s_alpha[g + 8];
#pragma unroll
      for (int i = 0; i < C::NO; ++i) {
        acc[i][0] *= al0;
        acc[i][1] *= al0;
        acc[i][2] *= al1;
        acc[i][3] *= al1;
      }
      const uint32_t pb = smem_u32(sP) + ((lane & 15) * C::PST + (lane >> 4) * 8) * 2;
      const int mi = lane >> 3, ri = lane & 7;
      if constexpr (C::BF) {
        const int c0 = warp * (C::DW / 8);
#pragma unroll
        for (int kt = 0; kt < C::TT / 16; ++kt) {
          uint32_t p[4], r[4];
          ldsm4(p, pb + kt * 32);
#pragma unroll
          for (int c = 0; c < C::NO; c += 2) {
            ldsm4t(r, vb + swz<C>(kt * 16 + (mi & 1) * 8 + ri, c0 + c + (mi >> 1)));
            mma_bf16(acc[c], p, r[0], r[1]);
            mma_bf16(acc[c + 1], p, r[2], r[3]);
          }
        }
      } else {
        const int c0 = warp * (C::DW * C::RB / C::D / 16);
        const uint8_t* vsc = sm + st * C::STAGE + C::PART + kPage * C::RB;
        (void)vsc;
#pragma unroll
        for (int kt = 0; kt < C::TT / 32; ++kt) {
          uint32_t p[2][4], r[4];
          ldsm4(p[0], pb + kt * 64);
          ldsm4(p[1], pb + kt * 64 + 32);
#pragma unroll
          for (int c = 0; c < C::DW * C::RB / C::D / 16; ++c) {
            ldsm4t(r, vb + swz<C>(kt * 32 + mi * 8 + ri, c0 + c));
            if constexpr (C::FMT == kKvFp8) {
              uint32_t e[4], o[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) e4m3x4(prmt(r[k], 0u, 0x3120u), e[k], o[k]);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                mma_f16(acc[2 * c], p[k], e[2 * k], e[2 * k + 1]);
                mma_f16(acc[2 * c + 1], p[k], o[2 * k], o[2 * k + 1]);
              }
            } else {
              uint32_t v[4][4];                    // [token octet][value of the 4]
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int t0 = kt * 32 + k * 8 + 2 * j4, blk = 2 * (c0 + c) + (lane >> 4);
                const uint32_t sb = vsc[t0 * C::SC + blk] | (static_cast<uint32_t>(vsc[(t0 + 1) * C::SC + blk]) << 8);
                const uint32_t s2 = e4m3x2_to_f16x2(static_cast<uint16_t>(sb));
                // nibbles of tokens t0 (low half) and t0 + 1 (high half) -> bytes of one value's token pair, in
                // the low halves of two bit selections
                const uint32_t ev = (r[k] & 0x0f0f0f0fu) | ((r[k] >> 12) & 0xf0f0f0f0u);       // values 0, 2
                const uint32_t od = ((r[k] >> 4) & 0x0f0f0f0fu) | ((r[k] >> 16) & 0xf0f0f0f0u); // values 1, 3
                uint32_t w[4];
                e2m1x8_to_f16x2x4(prmt(ev, od, 0x5410u), w);                                    // 0, 2, 1, 3
                v[k][0] = hmul2_u32(w[0], s2);
                v[k][2] = hmul2_u32(w[1], s2);
                v[k][1] = hmul2_u32(w[2], s2);
                v[k][3] = hmul2_u32(w[3], s2);
              }
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) mma_f16(acc[4 * c + e], p[k], v[2 * k][e], v[2 * k + 1][e]);
            }
          }
        }
      }
    }
    __syncthreads();
    if (tid == 0 && tile + C::NS < ntiles && !s_abort) issue(tile + C::NS);
  }
  // ---- partial results to shared memory (the ring is idle: every issued copy was waited for)
  float* sO = reinterpret_cast<float*>(sm);            // [16][D]
#pragma unroll
  for (int o = 1; o < TPR; o <<= 1) l_run += __shfl_xor_sync(0xffffffffu, l_run, o);
  if (tid % TPR == 0) {
    s_m[srow] = m_run;
    s_l[srow] = s_abort ? NAN : l_run;
  }
#pragma unroll
  for (int i = 0; i < C::NO; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = g + 8 * (k >> 1), e = k & 1;
      int d;
      if constexpr (C::BF) d = 8 * i + 2 * j4 + e;
      else if constexpr (C::FMT == kKvFp8) d = 16 * (i / 2) + 4 * j4 + 2 * e + (i & 1);
      else d = 32 * (i / 4) + 8 * j4 + 4 * e + (i & 3);
      sO[row * C::D + warp * C::DW + d] = acc[i][k];
    }
  }
  if (csize > 1) cluster_sync_all();
  else __syncthreads();
  // ---- join: every CTA finishes its share of the R x D outputs
  const uint32_t am = smem_u32(s_m), al = smem_u32(s_l), ao = smem_u32(sO);
  if (tid < kRows) {
    float M = -INFINITY;
    for (int c = 0; c < csize; ++c)
      M = fmaxf(M, __uint_as_float(ld_cluster_u32(mapa_shared(am + 4 * tid, c))));
    const float ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    for (int c = 0; c < csize; ++c) {
      const float f = ex2(__uint_as_float(ld_cluster_u32(mapa_shared(am + 4 * tid, c))) - ms);
      s_f[c][tid] = f;
      L += f * __uint_as_float(ld_cluster_u32(mapa_shared(al + 4 * tid, c)));
    }
    const float inv = L == 0.f ? 0.f : (C::BF ? 1.f : a.v_scale) / L;
    for (int c = 0; c < csize; ++c) s_f[c][tid] *= inv;
    if (rank == 0 && tid < R)
      a.lse[static_cast<size_t>(b * a.n_q + tid / G) * a.Hq + h * G + tid % G] =
          L == 0.f ? -INFINITY : 0.6931471805599453f * (M + log2f(L));
  }
  __syncthreads();
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out);
  for (int i = rank * C::NT + tid; i < R * (C::D / 4); i += csize * C::NT) {
    const int row = i / (C::D / 4), d = 4 * (i % (C::D / 4));
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < csize; ++c) {
      const float f = s_f[c][row];
      const float4 v = ld_cluster_f4(mapa_shared(ao + 4 * (row * C::D + d), c));
      if (f != 0.f) {
        o.x += f * v.x;
        o.y += f * v.y;
        o.z += f * v.z;
        o.w += f * v.w;
      }
    }
    const __nv_bfloat162 lo = __floats2bfloat162_rn(o.x, o.y), hi = __floats2bfloat162_rn(o.z, o.w);
    uint2 raw;
    raw.x = *reinterpret_cast<const uint32_t*>(&lo);
    raw.y = *reinterpret_cast<const uint32_t*>(&hi);
    *reinterpret_cast<uint2*>(out + (static_cast<size_t>(b * a.n_q + row / G) * a.Hq + h * G + row % G) * C::D + d) = raw;
  }
  if (csize > 1) cluster_sync_all();             // a CTA's partial results are read until here
}

template <int D, int FMT>
cudaError_t launch(const BlockDecodeArgs& a, cudaStream_t s) {
  using C = Cfg<D, FMT>;
  // Few lists: each is split over a cluster until every SM holds the CTAs it has room for, as long as a CTA keeps
  // two pages.
  const int units = a.B * a.Hk;
  int cs = 1;
  while (cs < 8 && units * cs * 2 <= 148 * C::RES && a.budget >= 4 * cs) cs *= 2;
  const int cap = (a.budget + cs - 1) / cs;
  const int smem = C::smem(cap);
  auto k = block_decode_kernel<C>;
  IOB_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(units) * cs);
  cfg.blockDim = dim3(C::NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, a, cs, cap);
}

}  // namespace

cudaError_t block_decode(const BlockDecodeArgs& a, cudaStream_t s) {
  if (a.B == 0) return cudaSuccess;
  if (a.Hk < 1 || a.Hq % a.Hk || a.n_q < 1 || a.n_q * (a.Hq / a.Hk) > kRows || a.budget < 1 ||
      a.budget > kBlockMaxList)
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
