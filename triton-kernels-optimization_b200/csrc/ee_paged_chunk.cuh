// ee_paged_chunk.cuh - attention of a chunk of new tokens over the paged cache on tcgen05.
//
// A unit (ee_paged.cuh) is two tiles of 128 query rows: TQ / 2 tokens each, every token with
// the unit's query heads of one KV head, so that a key is fetched and converted once for all
// of them.  Per tile of 128 keys: S = Q K^T (fp32 in TMEM), the online softmax with the row's
// entropy, O += P V.  One CTA per SM, 512 threads:
//   warps 0-1   UMMA issuers, one thread each, warp w for query tile w: S_0 | S_j+1, P_j V_j | ..
//               (the next S runs under the softmax of the current one);
//   warps 4-7   the keys: a page's values come from HBM in the order they are kept, are
//               converted to fp16 in registers (8-bit codes exactly: the scales stay out) and
//               stored as the K-major SW128 operands K [128 keys, D] and V^T [D, 128 keys].  Each
//               unit of 16 bytes is replaced by the next tile's as soon as it is used, so a
//               tile's loads are in flight during the tile before;
//   warps 8-15  warpgroup w = query tile w, one row per thread: scores from TMEM, row
//               maximum, P = 2^(x - m) as fp16 into shared memory, l and t, and at the end
//               O / l (or the part's O, l, t, m for the join).
// The orders inside K and V^T follow the pages' own (no shuffles): 16-byte column q4 2 + c of
// block `piece` of K's rows is dimensions q4 D/4 + 16 piece + 8 c .. (Q is stored alike); row
// 8 i + gq of V^T is dimension gq D/8 + i; column chunk 2 q4 + pi of V^T's 64-key block vb is keys
// 64 vb + 32 pi + 2 q4 + {0, 1, 8, 9, 16, 17, 24, 25} (P is stored alike).
// Scales: K's multiplies S in fp32 with the softmax scale; V's raises the exponent of P
// (v_shift), so P is rounded to fp16 once, with it.
// Every wait is bounded; on expiry the CTA records the error word, drains its MMAs, frees
// TMEM and exits.
//
// Included once, by ee_paged.cu, after ee_paged.cuh.
#pragma once

#include <climits>

namespace ee {

constexpr int kChunkThreads = 512;
// registers per thread at launch: 128 (512 threads, one CTA per SM), dealt out again by
// warpgroup: issuers, keys, 2 x softmax
constexpr int kChunkIssueRegs = 56, kChunkKeyRegs = 88, kChunkSoftmaxRegs = 184;
static_assert(kChunkIssueRegs + kChunkKeyRegs + 2 * kChunkSoftmaxRegs <= 4 * 128, "register split above the launch budget");
constexpr int kChunkTile = 128;                  // query rows per tile, keys per tile
constexpr int kChunkBox = kChunkTile * 128;      // one SW128 block of 128 rows: 16 KB
constexpr int kChunkMeta = 4;                    // tiles of scales held

template <int D>
struct ChunkCfg {
  static constexpr int KB = D / 64;                       // 128-byte column blocks of Q and K rows
  static constexpr int kQBytes = KB * kChunkBox;          // a Q tile, a K tile
  static constexpr int kVBytes = 2 * D * 128;             // V^T: D rows, two blocks of 64 keys
  static constexpr int kPBytes = 2 * kChunkBox;
  static constexpr int NS = 2, NV = D == 64 ? 2 : 1;      // ring depths of K and V
  static constexpr int kBarBytes = 256, kMetaBytes = kChunkMeta * 8 * 16;
  static constexpr size_t kSmem = 1024 + 2 * size_t(kQBytes) + NS * size_t(kQBytes) + NV * size_t(kVBytes) +
                                  2 * size_t(kPBytes) + kMetaBytes + kBarBytes;
  static_assert(kSmem <= 227 * 1024, "chunk attention above the 227 KB of shared memory per CTA");
  static constexpr uint32_t kTmemS = 0, kTmemO = 2 * kChunkTile;
  // a part's results: (m, l, t, then the D columns in V^T's row order) x 256 rows
  static constexpr int64_t kRec = int64_t(D + 3) * 256;
};

// 32 lanes x 16 columns of TMEM
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void fence_proxy_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// masked scores: far below any score, and their product with a scale (1e-25 at least) far below
// any reference, but finite, so that 0 times their distance is 0
constexpr float kMasked = -1e33f;

// tiles of a part that query tile w takes part in
template <int D>
struct ChunkPart {
  int n[2], nmax;  // key tiles of query tile 0 / 1, of the part
  int tq;          // tokens of query tile 0
};
__device__ __forceinline__ int chunk_tiles(int64_t reach) { return static_cast<int>((reach + kChunkTile - 1) / kChunkTile); }
template <int D>
__device__ __forceinline__ ChunkPart<D> chunk_part(const PagedPlan& pl, const PagedPart& u) {
  ChunkPart<D> p;
  const int half = pl.TQ / 2;
  p.tq = u.ntok < half ? u.ntok : half;
  const int t0 = chunk_tiles(u.s.start + u.tok0 + p.tq);
  const int e0 = t0 < u.tile1 ? t0 : u.tile1;
  p.n[0] = e0 > u.tile0 ? e0 - u.tile0 : 0;
  p.n[1] = u.ntok > half && u.tile1 > u.tile0 ? u.tile1 - u.tile0 : 0;
  p.nmax = p.n[0] > p.n[1] ? p.n[0] : p.n[1];
  return p;
}

template <int D, int TIER>
__global__ void __launch_bounds__(kChunkThreads, 1)
    paged_chunk_kernel(const PagedArgs c, const PagedStepArgs st, const PagedPlan pl, const PagedRows q, int heads,
                       float scale, __half* __restrict__ out, int64_t ldo, float* __restrict__ H,
                       float* __restrict__ part) {
  using Cfg = ChunkCfg<D>;
  constexpr int NS = Cfg::NS, NV = Cfg::NV, T = kChunkTile;
  extern __shared__ uint8_t chunk_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(chunk_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * Cfg::kQBytes;
  uint8_t* sV = sK + NS * Cfg::kQBytes;
  uint8_t* sP = sV + NV * Cfg::kVBytes;
  float4* sMeta = reinterpret_cast<float4*>(sP + 2 * Cfg::kPBytes);  // [kChunkMeta][8 groups]: K factor, V shift, 2^-shift
  uint64_t* bars = reinterpret_cast<uint64_t*>(sP + 2 * Cfg::kPBytes + Cfg::kMetaBytes);
  uint64_t* q_full = bars;            // [2] Q tile stored (4 warps)
  uint64_t* k_full = q_full + 2;      // [NS] K tile stored (4 warps)
  uint64_t* k_empty = k_full + NS;    // [NS] both issuers' S MMAs done
  uint64_t* v_full = k_empty + NS;    // [NV]
  uint64_t* v_empty = v_full + NV;    // [NV]
  uint64_t* s_full = v_empty + NV;    // [2] S_w ready
  uint64_t* s_free = s_full + 2;      // [2] S_w in registers (4 warps)
  uint64_t* p_full = s_free + 2;      // [2] P_w stored, O_w corrected (4 warps)
  uint64_t* o_done = p_full + 2;      // [2] P_w V done
  uint64_t* o_free = o_done + 2;      // [2] O_w read out (4 warps)
  uint64_t* drain = o_free + 2;       // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int64_t* s_share = reinterpret_cast<int64_t*>(tmem_slot + 2);
  static_assert((2 + 2 * NS + 2 * NV + 12) * 8 + 8 + 24 <= Cfg::kBarBytes, "barrier region overflows");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&k_empty[i], 2);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_free[i], 4);
      mbar_init(&drain[i], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  griddep_wait();
  PagedWalk walk = paged_begin(c, st, pl, blockIdx.x, gridDim.x, s_share);
  if (walk.left <= 0) return;
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  auto give_up = [&]() {
    if (lane == 0) {
      atomicOr(&g_paged_error, kErrWaitTimeout);
      *abort_flag = 1;
    }
  };

  PagedPart u;
  if (warp < 4) {
    warpgroup_reg_dealloc<kChunkIssueRegs>();
    if (warp < 2) {
      // ------------------------------------------------------------ UMMA issuers
      constexpr uint32_t idesc_s = make_idesc(1u, 0u, T, T);
      constexpr uint32_t idesc_o = make_idesc(1u, 0u, T, D);
      const int w = warp;
      bool ok = true;
      uint32_t kt = 0, vt = 0, g = 0, loads = 0;  // K / V tiles, tiles and parts of query tile w so far
      auto issue_s = [&](uint32_t kidx, uint32_t gidx) -> bool {
        const int s = kidx % NS;
        if (!mbar_wait_warp(&k_full[s], (kidx / NS) & 1u, abort_flag) ||
            !mbar_wait_warp(&s_free[w], (gidx & 1u) ^ 1u, abort_flag))
          return false;
        tc_fence_after();
        if (lane == 0) {
          for (int kb = 0; kb < Cfg::KB; ++kb) {
            const uint64_t da = sdesc_k_sw128(smem_u32(sQ + w * Cfg::kQBytes + kb * kChunkBox));
            const uint64_t db = sdesc_k_sw128(smem_u32(sK + s * Cfg::kQBytes + kb * kChunkBox));
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc_mma<kKindF16>(tmem_base + Cfg::kTmemS + w * T, da + 2u * k, db + 2u * k, idesc_s, kb || k ? 1u : 0u);
          }
          tc_commit(&s_full[w]);
        }
        __syncwarp();
        return true;
      };
      auto issue_pv = [&](uint32_t vidx, uint32_t gidx, bool first) -> bool {
        const int s = vidx % NV;
        if (!mbar_wait_warp(&v_full[s], (vidx / NV) & 1u, abort_flag) ||
            !mbar_wait_warp(&p_full[w], gidx & 1u, abort_flag))
          return false;
        tc_fence_after();
        if (lane == 0) {
          for (int vb = 0; vb < 2; ++vb) {
            const uint64_t da = sdesc_k_sw128(smem_u32(sP + w * Cfg::kPBytes + vb * kChunkBox));
            const uint64_t db = sdesc_k_sw128(smem_u32(sV + s * Cfg::kVBytes + vb * (D * 128)));
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc_mma<kKindF16>(tmem_base + Cfg::kTmemO + w * D, da + 2u * k, db + 2u * k, idesc_o,
                               first && !vb && !k ? 0u : 1u);
          }
          tc_commit(&o_done[w]);
        }
        __syncwarp();
        return true;
      };
      while (ok && paged_next<T>(c, st, pl, walk, u)) {
        const ChunkPart<D> cp = chunk_part<D>(pl, u);
        const int n = cp.n[w];
        if (n > 0) ok = mbar_wait_warp(&q_full[w], loads & 1u, abort_flag);
        for (int j = -1; ok && j < cp.nmax; ++j) {
          if (j + 1 < cp.nmax) {  // S of tile j + 1 (or its share of the K stage's release)
            const uint32_t kn = kt + j + 1;
            ok = j + 1 < n ? issue_s(kn, g + j + 1) : mbar_wait_warp(&k_full[kn % NS], (kn / NS) & 1u, abort_flag);
            if (ok && lane == 0) tc_commit(&k_empty[kn % NS]);
            __syncwarp();
          }
          if (ok && j >= 0) {  // P V of tile j
            const uint32_t vn = vt + j;
            if (j < n) {
              // the part's first P V overwrites O_w: the part before must be read out
              if (j == 0 && loads > 0) ok = mbar_wait_warp(&o_free[w], (loads - 1) & 1u, abort_flag);
              ok = ok && issue_pv(vn, g + j, j == 0);
            } else {
              ok = mbar_wait_warp(&v_full[vn % NV], (vn / NV) & 1u, abort_flag);
            }
            if (ok && lane == 0) tc_commit(&v_empty[vn % NV]);
            __syncwarp();
          }
        }
        kt += cp.nmax;
        vt += cp.nmax;
        g += n;
        loads += n > 0;
      }
      if (!ok) {
        give_up();
        if (lane == 0) tc_commit(&drain[w]);
        __syncwarp();
        (void)mbar_wait(&drain[w], 0u, nullptr);
      }
    }
  } else if (warp < 8) {
    warpgroup_reg_dealloc<kChunkKeyRegs>();
    // -------------------------------------------------------------- keys
    // Warp kw takes keys 32 kw .. + 31 of every tile: groups 2 kw, 2 kw + 1 of 16.
    const int kw = warp - 4, gq = lane >> 2, q4 = lane & 3;
    const float to2 = scale * 1.4426950408889634f;
    const int pg = c.page_shift - 4;
    uint32_t kt = 0, vt = 0;
    bool ok = true;
    // K row of group ga, half hf: 16 (2 kw + ga) + 8 hf + gq, so row & 7 = gq
    auto k_at = [&](uint8_t* tile, int ga, int hf, int piece, int cc) -> uint4* {
      return reinterpret_cast<uint4*>(tile + piece * kChunkBox + (32 * kw + 16 * ga + 8 * hf + gq) * 128 +
                                      (((2 * q4 + cc) ^ gq) << 4));
    };
    auto v_at = [&](uint8_t* tile, int i) -> uint4* {  // dimension gq D/8 + i
      return reinterpret_cast<uint4*>(tile + (kw >> 1) * (D * 128) + (8 * i + gq) * 128 + (((2 * q4 + (kw & 1)) ^ gq) << 4));
    };
    while (ok && paged_next<T>(c, st, pl, walk, u)) {
      const ChunkPart<D> cp = chunk_part<D>(pl, u);
      const PagedSeq& s = u.s;
      const int64_t full = TIER == kFP16 ? c.max_pages : s.length >> c.page_shift;  // blocks in pages
      const int32_t* table = c.table + s.seq * c.max_pages;
      const float log2_vref = __log2f(paged_vref(c, s, u.h));
      // where a group's values are: nowhere (a hole, or past the tokens), in a page, in the open block
      auto lookup = [&](int j, int (&pgs)[2]) {
#pragma unroll
        for (int ga = 0; ga < 2; ++ga) {
          const int64_t g = static_cast<int64_t>(u.tile0 + j) * 8 + 2 * kw + ga, blk = g >> pg;
          int p = -1;
          if (j < cp.nmax && g * 16 < s.length) {
            if (blk >= full) {
              p = INT_MAX;  // open
            } else {
              p = table[blk];
              p = p >= 0 && p < c.num_pages ? p : -1;
            }
          }
          pgs[ga] = p;
        }
      };
      auto meta_of = [&](int p) -> float4 {
        if (p < 0) return make_float4(1e-25f, kMasked, 1.f, 0.f);
        float2 sc = make_float2(1.f, 1.f);
        if (TIER != kFP16 && p != INT_MAX)
          sc = *reinterpret_cast<const float2*>(c.scale + (static_cast<int64_t>(p) * c.kv_heads + u.h) * 2);
        const float lv = v_shift(sc.y, log2_vref);
        return make_float4(fmaxf(to2 * sc.x, 1e-25f), lv, ex2_approx(-lv), 0.f);
      };
      for (int j = -1; ok && j < cp.nmax; ++j) {
        // K of tile j + 1, then V of tile j
        const bool k_now = j + 1 < cp.nmax;
        for (int which = 0; which < 2 && ok; ++which) {
          if (which == 0 ? !k_now : j < 0) continue;
          const int tile_j = which == 0 ? j + 1 : j;
          int pgs[2];
          lookup(tile_j, pgs);
          const uint32_t idx = which == 0 ? kt + tile_j : vt + tile_j;
          const int stage = which == 0 ? idx % NS : idx % NV;
          uint64_t* empty = which == 0 ? &k_empty[stage] : &v_empty[stage];
          const uint32_t par = ((which == 0 ? idx / NS : idx / NV) & 1u) ^ 1u;
          uint8_t* dst = which == 0 ? sK + stage * Cfg::kQBytes : sV + stage * Cfg::kVBytes;
          const int64_t g0 = static_cast<int64_t>(u.tile0 + tile_j) * 8 + 2 * kw;
          const bool wide0 = TIER == kFP16 || pgs[0] == INT_MAX, wide1 = TIER == kFP16 || pgs[1] == INT_MAX;
          auto base = [&](int ga) -> const uint8_t* {
            const int64_t g = g0 + ga, off = (g & ((1 << pg) - 1)) * 16 * D;
            if (pgs[ga] == INT_MAX)
              return reinterpret_cast<const uint8_t*>(paged_open(c, s.seq, full, u.h, which) + off) + lane * 16;
            return paged_block(c, pgs[ga], u.h, which) + off * (TIER == kFP16 ? 2 : 1) + lane * 16;
          };
          if (which == 0) {
            float4 m = make_float4(0.f, 0.f, 0.f, 0.f);
            if (lane < 2) m = meta_of(lane == 0 ? pgs[0] : pgs[1]);
            uint4 x[2][D / 32];
            if constexpr (TIER != kFP16) {
#pragma unroll
              for (int ga = 0; ga < 2; ++ga)
#pragma unroll
                for (int i = 0; i < D / 32; ++i)
                  x[ga][i] = pgs[ga] >= 0 && !(ga ? wide1 : wide0)
                                 ? __ldg(reinterpret_cast<const uint4*>(base(ga) + i * 512))
                                 : make_uint4(0, 0, 0, 0);
            }
            ok = mbar_wait_warp(empty, par, abort_flag);
            if (!ok) break;
            if (lane < 2) sMeta[(idx % kChunkMeta) * 8 + 2 * kw + lane] = m;
#pragma unroll
            for (int ga = 0; ga < 2; ++ga) {
              if (ga ? wide1 : wide0) {
                const uint4* src = reinterpret_cast<const uint4*>(pgs[ga] >= 0 ? base(ga) : nullptr);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                  const uint4 y = pgs[ga] >= 0 ? src[i * 32] : make_uint4(0, 0, 0, 0);
                  const int hf = i / (D / 32), p8 = i % (D / 32);
                  *k_at(dst, ga, hf, p8 >> 1, p8 & 1) = y;
                }
              } else if constexpr (TIER != kFP16) {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                  const int hf = i / (D / 64), piece = i % (D / 64);
                  uint4 a, b;
                  if (pgs[ga] >= 0) {
                    codes_to_h2<TIER>(x[ga][i].x, a.x, a.y);
                    codes_to_h2<TIER>(x[ga][i].y, a.z, a.w);
                    codes_to_h2<TIER>(x[ga][i].z, b.x, b.y);
                    codes_to_h2<TIER>(x[ga][i].w, b.z, b.w);
                  } else {
                    a = b = make_uint4(0, 0, 0, 0);
                  }
                  *k_at(dst, ga, hf, piece, 0) = a;
                  *k_at(dst, ga, hf, piece, 1) = b;
                }
              }
            }
          } else {
            uint4 x[2][D / 32];
            if constexpr (TIER != kFP16) {
#pragma unroll
              for (int ga = 0; ga < 2; ++ga)
#pragma unroll
                for (int i = 0; i < D / 32; ++i)
                  x[ga][i] = pgs[ga] >= 0 && !(ga ? wide1 : wide0)
                                 ? __ldg(reinterpret_cast<const uint4*>(base(ga) + i * 512))
                                 : make_uint4(0, 0, 0, 0);
            }
            ok = mbar_wait_warp(empty, par, abort_flag);
            if (!ok) break;
            uint32_t keep[2][2];  // tokens past the sequence's are no numbers to multiply by
#pragma unroll
            for (int ga = 0; ga < 2; ++ga)
#pragma unroll
              for (int th = 0; th < 2; ++th) {
                const int64_t t0 = (g0 + ga) * 16 + 2 * q4 + 8 * th;
                keep[ga][th] = pgs[ga] < 0 ? 0u : ((t0 < s.length ? 0xffffu : 0u) | (t0 + 1 < s.length ? 0xffff0000u : 0u));
              }
            const uint8_t* b0 = pgs[0] >= 0 ? base(0) : nullptr;
            const uint8_t* b1 = pgs[1] >= 0 ? base(1) : nullptr;
#pragma unroll
            for (int mb = 0; mb < D / 16; ++mb) {
              uint4 lo, hi;  // dimensions 2 mb, 2 mb + 1: keys of group 0 (two pairs), of group 1
#pragma unroll
              for (int ga = 0; ga < 2; ++ga) {
                uint32_t j0t0, j1t0, j0t1, j1t1;
                if (ga ? wide1 : wide0) {
                  const uint4 y = pgs[ga] >= 0 ? reinterpret_cast<const uint4*>(ga ? b1 : b0)[mb * 32] : make_uint4(0, 0, 0, 0);
                  j0t0 = y.x;
                  j1t0 = y.y;
                  j0t1 = y.z;
                  j1t1 = y.w;
                } else {
                  const uint4 y = x[ga][TIER != kFP16 ? mb >> 1 : 0];
                  codes_to_h2<TIER == kFP16 ? kINT8 : TIER>(mb & 1 ? y.z : y.x, j0t0, j1t0);
                  codes_to_h2<TIER == kFP16 ? kINT8 : TIER>(mb & 1 ? y.w : y.y, j0t1, j1t1);
                }
                j0t0 &= keep[ga][0];
                j1t0 &= keep[ga][0];
                j0t1 &= keep[ga][1];
                j1t1 &= keep[ga][1];
                (ga ? lo.z : lo.x) = j0t0;
                (ga ? lo.w : lo.y) = j0t1;
                (ga ? hi.z : hi.x) = j1t0;
                (ga ? hi.w : hi.y) = j1t1;
              }
              *v_at(dst, 2 * mb) = lo;
              *v_at(dst, 2 * mb + 1) = hi;
            }
          }
          fence_proxy_async_shared();  // the stores, visible to the tensor core
          __syncwarp();
          if (lane == 0) mbar_arrive(which == 0 ? &k_full[stage] : &v_full[stage]);
        }
      }
      kt += cp.nmax;
      vt += cp.nmax;
    }
    if (!ok) give_up();
  } else {
    warpgroup_reg_alloc<kChunkSoftmaxRegs>();
    // -------------------------------------------------------------- softmax, entropy, output
    const int w = (warp - 8) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem_base + Cfg::kTmemS + w * T + lane_off;
    const uint32_t t_o = tmem_base + Cfg::kTmemO + w * D + lane_off;
    uint8_t* pbuf = sP + w * Cfg::kPBytes + row * 128;
    uint8_t* qbuf = sQ + w * Cfg::kQBytes + row * 128;
    const int rx = row & 7;
    bool ok = true;
    uint32_t kt = 0, g = 0;
    while (ok && paged_next<T>(c, st, pl, walk, u)) {
      const ChunkPart<D> cp = chunk_part<D>(pl, u);
      const int n = cp.n[w];
      // this row: token and query head
      const int half = pl.TQ / 2, tok = row / pl.Gc + w * half, hd = u.hg * pl.Gc + row % pl.Gc;
      const bool real = row < half * pl.Gc && tok < u.ntok && hd < pl.G;
      const int64_t qrow = u.s.row0 + u.tok0 + (real ? tok : 0);
      const int head = u.h * pl.G + (real ? hd : 0);
      float m = kNegInf, l = 0.f, t = 0.f;
      if (n > 0) {
        // Q: the S MMAs of the part before have read the old one (their last S was waited for)
        const uint4* src = reinterpret_cast<const uint4*>(q.p + qrow * q.ld + head * D);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint4 x = real ? src[i] : make_uint4(0, 0, 0, 0);
          const int q4 = i / (D / 32), r = i % (D / 32);  // dimensions 8 i ..: piece r / 2, chunk 2 q4 + r % 2
          *reinterpret_cast<uint4*>(qbuf + (r >> 1) * kChunkBox + (((2 * q4 + (r & 1)) ^ rx) << 4)) = x;
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[w]);
      }
      for (int j = 0; j < n; ++j) {
        const uint32_t gj = g + j;
        ok = mbar_wait_warp(&s_full[w], gj & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const int64_t key0 = static_cast<int64_t>(u.tile0 + j) * T;
        const int64_t seen = u.s.start + u.tok0 + tok + 1 - key0;
        const int lim = !real || seen > T ? T : (seen < 0 ? 0 : static_cast<int>(seen));
        uint32_t r[4][32];
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) tmem_ld32(t_s + 32 * k, r[k]);
        tmem_ld_wait(r[0]);
        regs_after_wait(r[1]);
        regs_after_wait(r[2]);
        regs_after_wait(r[3]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[w]);  // S_w is in registers: the next S may land
        auto S = [&](int i) -> float { return __uint_as_float(r[i >> 5][i & 31]); };
        if (!__all_sync(0xffffffffu, lim >= T)) {
#pragma unroll
          for (int i = 0; i < T; ++i)
            if (i >= lim) r[i >> 5][i & 31] = __float_as_uint(kMasked);
        }
        const float4* meta = sMeta + ((kt + j) % kChunkMeta) * 8;
        float mt = kNegInf;
#pragma unroll
        for (int gr = 0; gr < 8; ++gr) {
          float a = fmaxf(S(16 * gr), S(16 * gr + 1)), b = fmaxf(S(16 * gr + 2), S(16 * gr + 3));
#pragma unroll
          for (int i = 4; i < 16; i += 4) {
            a = fmaxf(a, fmaxf(S(16 * gr + i), S(16 * gr + i + 1)));
            b = fmaxf(b, fmaxf(S(16 * gr + i + 2), S(16 * gr + i + 3)));
          }
          const float4 f = meta[gr];
          mt = fmaxf(mt, fmaf(fmaxf(a, b), f.x, f.y));
        }
        if (lim <= 0 || mt < 0.1f * kMasked) mt = kNegInf;  // sees no key of this tile
        float alpha = 1.f;
        const float m_old = m;
        if (m == kNegInf) {
          m = mt;
        } else if (mt > m + 8.f) {
          alpha = ex2_approx(m - mt);
          m = mt;
        }
        const bool rescale = __any_sync(0xffffffffu, alpha != 1.f);
        if (j > 0) {  // P_w V_{j-1} done: P_w may be written again, O_w stands still
          ok = mbar_wait_warp(&o_done[w], (gj - 1u) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
        }
        if (rescale) {
#pragma unroll
          for (int c0 = 0; c0 < D; c0 += 16) {
            uint32_t o[16];
            __syncwarp();
            tmem_ld16(t_o + c0, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st16(t_o + c0, o);
          }
          tmem_st_wait();
          if (alpha != 1.f) {
            t = alpha * (t + l * (m_old - m));
            l = alpha * l;
          }
        }
        const float mu = m == kNegInf ? 0.f : m;
#pragma unroll
        for (int sp = 0; sp < 4; ++sp) {
          uint32_t pk[2][8];
#pragma unroll
          for (int ga = 0; ga < 2; ++ga) {
            const int c0 = 32 * sp + 16 * ga;
            const float4 f = meta[2 * sp + ga];
            const float2 ks2 = make_float2(f.x, f.x), nb2 = make_float2(f.y - mu, f.y - mu);
            float2 sum = make_float2(0.f, 0.f), dot = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 d = __ffma2_rn(make_float2(S(c0 + 2 * i), S(c0 + 2 * i + 1)), ks2, nb2);
              const float2 p = make_float2(ex2_approx(d.x), ex2_approx(d.y));
              sum = __fadd2_rn(sum, p);
              dot = __ffma2_rn(p, d, dot);
              pk[ga][i] = pack2(p.x, p.y);
            }
            const float sm = sum.x + sum.y;
            l = fmaf(f.z, sm, l);
            t = fmaf(f.z, fmaf(-f.y, sm, dot.x + dot.y), t);
          }
          uint8_t* dst = pbuf + (sp >> 1) * kChunkBox;
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<uint4*>(dst + (((2 * q4 + (sp & 1)) ^ rx) << 4)) =
                make_uint4(pk[0][q4], pk[0][q4 + 4], pk[1][q4], pk[1][q4 + 4]);
        }
        fence_proxy_async_shared();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[w]);
      }
      if (ok && n > 0) ok = mbar_wait_warp(&o_done[w], (g + n - 1) & 1u, abort_flag);
      if (!ok) break;
      float* rec = part + (2 * static_cast<int64_t>(blockIdx.x) + (u.first ? 1 : 0)) * Cfg::kRec + w * T + row;
      if (n > 0) {
        tc_fence_after();
        const float vref = paged_vref(c, u.s, u.h);
        const float f = l != 0.f ? vref / l : 0.f;  // a row that sees no key: zeros
        __half* dst = out + qrow * ldo + head * D;
#pragma unroll
        for (int hh = 0; hh < D / 64; ++hh) {  // columns 64 hh ..: dimensions 8 hh .. of each gq's
          uint32_t a[32], b[32];
          __syncwarp();
          tmem_ld32(t_o + 64 * hh, a);
          tmem_ld32(t_o + 64 * hh + 32, b);
          tmem_ld_wait(a);
          regs_after_wait(b);
          if (u.whole) {
            if (real) {
#pragma unroll
              for (int gq = 0; gq < 8; ++gq) {
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const uint32_t x0 = k < 2 ? a[16 * k + gq] : b[16 * (k - 2) + gq];
                  const uint32_t x1 = k < 2 ? a[16 * k + 8 + gq] : b[16 * (k - 2) + 8 + gq];
                  o[k] = pack2(l != 0.f ? __uint_as_float(x0) * f : 0.f, l != 0.f ? __uint_as_float(x1) * f : 0.f);
                }
                *reinterpret_cast<uint4*>(dst + gq * (D / 8) + 8 * hh) = make_uint4(o[0], o[1], o[2], o[3]);
              }
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              rec[(3 + 64 * hh + k) * 256] = __uint_as_float(a[k]);
              rec[(3 + 64 * hh + 32 + k) * 256] = __uint_as_float(b[k]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[w]);
      }
      if (u.whole) {
        if (real && H != nullptr) H[qrow * heads + head] = l != 0.f ? 0.69314718055994531f * (__log2f(l) - t / l) : 0.f;
        if (real && n == 0) {
          for (int i = 0; i < D / 8; ++i) *reinterpret_cast<uint4*>(out + qrow * ldo + head * D + 8 * i) = make_uint4(0, 0, 0, 0);
        }
      } else {
        rec[0] = m;
        rec[256] = l;
        rec[512] = t;
      }
      kt += cp.nmax;
      g += n;
    }
    if (!ok) give_up();
    tc_fence_before();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

// The units that several CTAs shared: block (x, y) joins rows 32 y .. of the unit that begins in CTA
// x's share and runs past it, its parts in the order of the keys.  Warp gq sums the dimensions
// gq D/8 .. of a row per lane.
template <int D>
__global__ void __launch_bounds__(256)
    paged_join_kernel(const PagedArgs c, const PagedStepArgs st, const PagedPlan pl, int heads, __half* __restrict__ out,
                      int64_t ldo, float* __restrict__ H, const float* __restrict__ part) {
  using Cfg = ChunkCfg<D>;
  __shared__ int64_t s_share[3];
  griddep_wait();
  griddep_launch_dependents();
  PagedWalk walk = paged_begin(c, st, pl, blockIdx.x, gridDim.x, s_share);
  PagedPart u;
  bool found = false;
  while (paged_next<kChunkTile>(c, st, pl, walk, u))
    if (u.first && !u.whole) {
      found = true;
      break;
    }
  if (!found) return;
  const int lane = threadIdx.x & 31, gq = threadIdx.x >> 5;
  const int r = blockIdx.y * 32 + lane, w = r >> 7, row = r & 127;
  const int half = pl.TQ / 2, tok = row / pl.Gc + w * half, hd = u.hg * pl.Gc + row % pl.Gc;
  const bool real = row < half * pl.Gc && tok < u.ntok && hd < pl.G;
  if (!real) return;
  auto rec_of = [&](int64_t k) { return part + (2 * k + (k == u.cta0 ? 1 : 0)) * Cfg::kRec + r; };
  float M = kNegInf;
  for (int64_t k = u.cta0; k <= u.cta1; ++k) M = fmaxf(M, rec_of(k)[0]);
  float L = 0.f, T = 0.f, o[D / 8];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i] = 0.f;
  for (int64_t k = u.cta0; k <= u.cta1; ++k) {
    const float* rec = rec_of(k);
    const float m = rec[0], l = rec[256];
    if (m == kNegInf && l == 0.f) continue;  // a part that saw no key of the row
    const float a = m == kNegInf ? 1.f : ex2_approx(m - M);
    L = fmaf(a, l, L);
    T = fmaf(a, rec[512] + (m == kNegInf ? 0.f : l * (m - M)), T);
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i] = fmaf(a, rec[(3 + 8 * i + gq) * 256], o[i]);
  }
  const int64_t qrow = u.s.row0 + u.tok0 + tok;
  const int head = u.h * pl.G + hd;
  const float f = L != 0.f ? paged_vref(c, u.s, u.h) / L : 0.f;
#pragma unroll
  for (int i = 0; i < D / 8; i += 8) {
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = pack2(o[i + 2 * k] * f, o[i + 2 * k + 1] * f);
    *reinterpret_cast<uint4*>(out + qrow * ldo + head * D + gq * (D / 8) + i) = make_uint4(x[0], x[1], x[2], x[3]);
  }
  if (gq == 0 && H != nullptr) H[qrow * heads + head] = L != 0.f ? 0.69314718055994531f * (__log2f(L) - T / L) : 0.f;
}

}  // namespace ee
