// Attention of chunks of new tokens over the 8-bit paged cache, on the 5th-generation tensor cores.
//
// A CTA takes 256 query rows of one (sequence, key/value head): two MMA tiles of 128, tokens x the query heads that share the head. It walks
// the keys 64 at a time; with few CTAs the keys are shared out over grid.z and a second kernel joins the parts.
//
//   warp 0        producer: codes and exponents of 64 tokens (bulk copies, the rows of a page and head lie together) into a ring
//   warps 12-15   codes to f16, into operand tiles with the 128-byte swizzle. Within a tile a row's scale is applied relative to the largest
//                 of the tile (a power of two: exact unless it is 2^-20 of that), so the tile has one scale left over, for K and for V
//   warp 1        MMA issuer: S_g = Q_g . K^T of the next keys into the other of two buffers, then O_g += P_g . V (P from TMEM)
//   warps 4-11    softmax, a query row per thread (as attention_tc.cu). The tile's scale of K is part of the score's factor; that of V, 2^E, goes
//                 into the exponent, 2^(t + E - m), and the denominator adds the tile's sum times 2^-E
//
// The MMAs of 64 keys take 1024 cycles, the exponentials as many, the conversion 16 K codes; all operands pass through shared memory.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/api.h"
#include "../common/launch.h"
#include "../common/ptx.cuh"
#include "attention_fp8.cuh"

namespace mb {
namespace a8 {

constexpr int kRing = 3;                // stages of codes
constexpr int kThreads = 512;
constexpr int kMaxSplits = 16;
constexpr int kHeadroom = 6;            // the tile's largest scale becomes 2^6: codes reach 2^15 of f16

struct ChunkParams {
  MbFp8Attention a;
  MbFp8Cache c;
  float* ws;                            // [split][T * n_q][HD + 2]: O, m, l
  int splits, box;
};

struct TileInfo {
  float k, v;                           // factor of a score, exponent of the values
};
struct ChunkBars {
  uint64_t full[kRing], empty[kRing];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t info_full[4];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], o_done[2];       // [query tile][buffer]
  TileInfo info[4];
  uint32_t qmax;
  uint32_t tmem_base;
  int abort_word;
};

template <int HD>
struct Shape {
  static constexpr int NC = HD / 64;                              // 64-column chunks of a row
  static constexpr int kQTile = NC * 128 * 128;
  static constexpr int kCodes = 64 * HD;
  static constexpr int kStage = 2 * kCodes;
  static constexpr int kTile16 = NC * 64 * 128;                   // an operand tile
  static constexpr size_t kSmem = 2 * kQTile + 4 * kTile16 + kRing * (kStage + 128) + sizeof(ChunkBars);
};

// MN-major operand with 128B swizzle: see attention_tc.cu
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(const void* smem_tile, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_u32(smem_tile) & 0x3ffff) >> 4);
  d |= static_cast<uint64_t>(lbo_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(sbo_bytes >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 2^x as f16 in both halves, x <= 6; zero below the smallest subnormal
__device__ __forceinline__ uint32_t pow2_f16x2(int x) {
  const uint32_t h = x >= -14 ? static_cast<uint32_t>(x + 15) << 10 : x >= -24 ? 1u << (x + 24) : 0u;
  return h | (h << 16);
}

// What a CTA works on. Plan tiles hold 64 / G tokens; a CTA takes up to four of them in a row.
struct Work {
  int seq, tq0, qs, ql, kl, tok, last_tq, kv_hi;
};
__device__ __forceinline__ bool work_of(const MbFp8Attention& a, int at, Work& w) {
  const int G = a.n_q / a.n_kv, n = a.n_tiles, lead = (n + 3) >> 2;
  // first the tiles that surely have work (where a sequence begins at a multiple of four), later ones of a prompt, which see more keys, first
  const int k = at - lead, tile = at < lead ? 4 * (lead - 1 - at) : k / 3 * 4 + k % 3 + 1;
  w.tok = 64 / G;
  w.seq = a.tile_seq[tile];
  if (w.seq < 0) return false;
  w.tq0 = a.tile_q0[tile];
  if (w.tq0 % (4 * w.tok) != 0) return false;       // covered by the CTA of a tile before it
  w.qs = a.q_start[w.seq]; w.ql = a.q_len[w.seq]; w.kl = a.kv_len[w.seq];
  w.last_tq = min(w.tq0 + 4 * w.tok, w.ql);
  w.kv_hi = max(0, min(w.kl, w.kl - w.ql + w.last_tq));
  return w.tq0 < w.ql;
}

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(const __grid_constant__ ChunkParams p) {
  using Sh = Shape<HD>;
  constexpr int NC = Sh::NC;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if (smem_u32(smem_raw) & 1023u) {                 // (no static shared memory: the window starts aligned)
    if (threadIdx.x == 0 && p.a.err) atomicCAS(p.a.err, 0, 759);
    return;
  }
  uint8_t* sQ = smem_raw;                           // [tile][chunk][128 rows x 128 B]
  uint8_t* sK = sQ + 2 * Sh::kQTile;                // [buffer][chunk][64 rows x 128 B]
  uint8_t* sV = sK + 2 * Sh::kTile16;
  uint8_t* sRing = sV + 2 * Sh::kTile16;            // [stage][K codes | V codes]
  uint8_t* sScale = sRing + kRing * Sh::kStage;     // [stage][K 64 | V 64]
  ChunkBars* bars = reinterpret_cast<ChunkBars*>(sScale + kRing * 128);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x, G = p.a.n_q / p.a.n_kv;
  pdl_wait();
  Work w;
  if (!work_of(p.a, blockIdx.y, w)) return;
  const int half_tok = 2 * w.tok;                   // tokens of an MMA tile
  const bool two = w.tq0 + half_tok < w.ql;
  const int all_tiles = (w.kv_hi + 63) / 64;
  const int t0 = static_cast<int>(static_cast<int64_t>(all_tiles) * blockIdx.z / p.splits);
  const int nt = static_cast<int>(static_cast<int64_t>(all_tiles) * (blockIdx.z + 1) / p.splits) - t0;

  if (tid == 0) {
    for (int s = 0; s < kRing; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 4); }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->k_full[b], 4); mbar_init(&bars->k_empty[b], 1);
      mbar_init(&bars->v_full[b], 4); mbar_init(&bars->v_empty[b], 1);
      for (int g = 0; g < 2; ++g) { mbar_init(&bars->s_full[g][b], 1); mbar_init(&bars->p_full[g][b], 4); mbar_init(&bars->pv_done[g][b], 1); }
      mbar_init(&bars->o_done[b], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bars->info_full[i], 1);
    bars->qmax = 0;
    bars->abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  __syncthreads();
  // query rows: the largest value first, then f16 with the 128-byte swizzle; a thread takes its own row
  const int g = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
  const int tq = w.tq0 + g * half_tok + r / G, head = kvh * G + r % G;
  const bool softmax_warp = warp >= 4 && warp < 12;
  const bool valid = softmax_warp && r < half_tok * G && tq < w.ql && w.qs + tq < p.a.T;
  const T* src = static_cast<const T*>(p.a.q) + static_cast<int64_t>(valid ? w.qs + tq : 0) * p.a.ldq + static_cast<int64_t>(head) * HD;
  if (softmax_warp) {
    float big = 0.f;
#pragma unroll
    for (int c = 0; c < HD; c += 16) {
      float x[16];
      load16(src + c, x, valid);
#pragma unroll
      for (int k = 0; k < 16; ++k) big = fmaxf(big, finite_abs(x[k]));
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
    if (lane == 0) atomicMax(&bars->qmax, top);
  }
  __syncthreads();
  const int qe = f16_shift(__uint_as_float(bars->qmax));
  if (softmax_warp) {
    const float mul = pow2f(qe);
#pragma unroll
    for (int c = 0; c < HD; c += 16) {
      float x[16];
      load16(src + c, x, valid);
      uint32_t h[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) h[k] = pack_f16(x[2 * k] * mul, x[2 * k + 1] * mul);
      uint8_t* row = sQ + g * Sh::kQTile + (c >> 6) * 16384 + r * 128;
      const int piece = (c & 63) >> 3;
      *reinterpret_cast<uint4*>(row + ((piece ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(row + (((piece + 1) ^ (r & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  volatile int* abort_word = &bars->abort_word;

  // 512 x 128 registers at launch = 128 x (48 + 192 + 192 + 80)
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- producer
      const int32_t* bt = p.a.block_table + static_cast<int64_t>(w.seq) * p.a.bt_stride;
      int s = 0;
      uint32_t ph = 0;
      for (int t = 0; t < nt; ++t) {
        const int kv0 = (t0 + t) * 64, boxes = (min(64, w.kv_hi - kv0) + p.box - 1) / p.box;
        int page[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          page[b] = 0;
          if (b >= boxes) continue;
          const int nth = (kv0 + b * p.box) / p.c.page_size;
          page[b] = nth < p.a.bt_stride ? bt[nth] : -1;
          if (page[b] < 0 || page[b] >= p.c.pages) {               // reported; some page stands in for it
            if (p.a.err) atomicCAS(p.a.err, 0, 731);
            page[b] = 0;
          }
        }
        if (!mbar_wait(&bars->empty[s], ph ^ 1, abort_word, p.a.err, 751)) break;
        mbar_arrive_expect_tx(&bars->full[s], static_cast<uint32_t>(boxes) * p.box * (2 * HD + 2));
        uint8_t* dst = sRing + s * Sh::kStage;
        uint8_t* sc = sScale + s * 128;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (b >= boxes) continue;
          const int64_t pg = page[b], off = (kv0 + b * p.box) % p.c.page_size;
          bulk_load(dst + b * p.box * HD, static_cast<const uint8_t*>(p.c.k) + pg * p.c.k_page + kvh * p.c.k_head + off * HD, p.box * HD, &bars->full[s]);
          bulk_load(dst + Sh::kCodes + b * p.box * HD, static_cast<const uint8_t*>(p.c.v) + pg * p.c.v_page + kvh * p.c.v_head + off * HD, p.box * HD, &bars->full[s]);
          bulk_load(sc + b * p.box, p.c.ks + pg * p.c.ks_page + kvh * p.c.ks_head + off, p.box, &bars->full[s]);
          bulk_load(sc + 64 + b * p.box, p.c.vs + pg * p.c.vs_page + kvh * p.c.vs_head + off, p.box, &bars->full[s]);
        }
        if (++s == kRing) { s = 0; ph ^= 1; }
      }
    } else if (warp == 1 && lane == 0) {
      // ---------------------------------------------------------------- MMA issuer
      const uint32_t idesc_s = umma_idesc(128, 64, 0, 0), idesc_pv = umma_idesc(128, HD, 0, 0) | (1u << 16);    // V is MN-major
      const int last = two ? 1 : 0;
      bool ok = true;
      auto scores = [&](int t) {
        const int b = t & 1;
        ok = ok && mbar_wait(&bars->k_full[b], (t >> 1) & 1, abort_word, p.a.err, 752);
        if (!ok) return;
        tc_fence_after();
        for (int q = 0; q <= last; ++q) {
#pragma unroll
          for (int k = 0; k < NC * 4; ++k) {
            const uint64_t da = umma_desc_sw128(sQ + q * Sh::kQTile + (k >> 2) * 16384) + static_cast<uint64_t>((k & 3) * 2);
            const uint64_t db = umma_desc_sw128(sK + b * Sh::kTile16 + (k >> 2) * 8192) + static_cast<uint64_t>((k & 3) * 2);
            umma_bf16(tmem_base + q * 128 + b * 64, da, db, idesc_s, k > 0 ? 1u : 0u);
          }
          tc_commit(&bars->s_full[q][b]);
        }
        tc_commit(&bars->k_empty[b]);
      };
      if (nt > 0) scores(0);
      for (int t = 0; t < nt && ok; ++t) {
        const int b = t & 1;
        if (t + 1 < nt) scores(t + 1);              // the product that read P of that buffer was issued before
        ok = ok && mbar_wait(&bars->v_full[b], (t >> 1) & 1, abort_word, p.a.err, 753);
        for (int q = 0; q <= last && ok; ++q) {
          ok = mbar_wait(&bars->p_full[q][b], (t >> 1) & 1, abort_word, p.a.err, 754);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16_ts(tmem_base + 256 + q * 128, tmem_base + q * 128 + b * 64 + k * 8, umma_desc_mn_sw128(sV + b * Sh::kTile16 + k * 2048, 8192, 1024),
                        idesc_pv, (t > 0 || k > 0) ? 1u : 0u);
          tc_commit(&bars->pv_done[q][b]);
          if (q == last) tc_commit(&bars->v_empty[b]);
          if (t + 1 == nt) tc_commit(&bars->o_done[q]);
        }
      }
    }
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    // ------------------------------------------------------------------ codes to f16
    const int cw = warp - 12, lo = lane & 3, up = (lane >> 2) & 1, quarter = lane >> 3;
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = 0; t < nt && ok; ++t) {
      const int b = t & 1, n = min(64, w.kv_hi - (t0 + t) * 64);       // rows behind the last key become zeros
      if (!__all_sync(0xffffffffu, mbar_wait(&bars->full[s], ph, abort_word, p.a.err, 755))) break;
      const uint8_t* sc = sScale + s * 128;
      int top[2];
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t two_bytes = *reinterpret_cast<const uint16_t*>(sc + kv * 64 + 2 * lane);
        const uint32_t x = 2 * lane < n ? two_bytes & 255u : 0u, y = 2 * lane + 1 < n ? two_bytes >> 8 : 0u;
        top[kv] = static_cast<int>(__reduce_max_sync(0xffffffffu, max(x, y)));
      }
      top[1] = min(max(top[1], kLeastByte), kMostByte);
      if (warp == 12 && lane == 0) {
        bars->info[t & 3].k = score_factor(p.a.scale * kLog2e, top[0] - 127 - kHeadroom - qe);
        bars->info[t & 3].v = static_cast<float>(top[1] - 127);
        mbar_arrive(&bars->info_full[t & 3]);
      }
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        ok = __all_sync(0xffffffffu, mbar_wait(kv == 0 ? &bars->k_empty[b] : &bars->v_empty[b], ((t >> 1) & 1) ^ 1, abort_word, p.a.err, 756));
        if (!ok) break;
        const uint8_t* from = sRing + s * Sh::kStage + kv * Sh::kCodes;
        uint8_t* to = (kv == 0 ? sK : sV) + b * Sh::kTile16;
        // 16 rows a warp. A quarter-warp reads 128 bytes together; lanes of the row's second half (HD 128) write their two pieces in the other
        // order, so that the eight meet no bank twice
#pragma unroll
        for (int it = 0; it < NC * 2; ++it) {
          const int row = cw * 16 + (NC == 2 ? it * 4 + quarter : it * 8 + quarter * 2 + up), chunk = NC == 2 ? (lane & 7) : lo;
          uint4 c = *reinterpret_cast<const uint4*>(from + row * HD + chunk * 16);
          uint32_t f = pow2_f16x2(static_cast<int>(sc[kv * 64 + row]) - top[kv] + kHeadroom);
          if (row >= n) { c = make_uint4(0, 0, 0, 0); f = 0; }
          const __half2 f2 = *reinterpret_cast<const __half2*>(&f);
          const uint32_t words[4] = {c.x, c.y, c.z, c.w};
          uint32_t h[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t x[2];
            codes_f16(words[k], x[0], x[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&x[e]), f2);
              h[2 * k + e] = *reinterpret_cast<const uint32_t*>(&y);
            }
          }
          uint8_t* dst = to + (chunk >> 2) * 8192 + row * 128;
          const int piece = 2 * (chunk & 3), swap = NC == 2 ? (chunk >> 2) : 0;
          const uint4 a = make_uint4(h[0], h[1], h[2], h[3]), z = make_uint4(h[4], h[5], h[6], h[7]);
          *reinterpret_cast<uint4*>(dst + (((piece + swap) ^ (row & 7)) << 4)) = swap ? z : a;
          *reinterpret_cast<uint4*>(dst + (((piece + 1 - swap) ^ (row & 7)) << 4)) = swap ? a : z;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(kv == 0 ? &bars->k_full[b] : &bars->v_full[b]);
      }
      if (!ok) break;
      if (lane == 0) mbar_arrive(&bars->empty[s]);
      if (++s == kRing) { s = 0; ph ^= 1; }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ------------------------------------------------------------------ softmax
    const int quad = warp & 3;
    const int limit = valid ? w.kl - w.ql + tq : 0x7fffffff;       // (queries that are not there are zeros: nothing to mask)
    const bool idle = quad * 32 >= half_tok * G || w.tq0 + g * half_tok + quad * 32 / G >= w.ql;      // no row of this warp is in use
    const uint32_t s_tile = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + g * 128, o_addr = s_tile + 256;
    float m = 0.f, l = 0.f;                          // weights and l are relative to m, a lagging running maximum
    bool ok = true, unset = true;                    // unset: no key has been visible to the row yet
    const int mine = g == 0 || two ? nt : 0;
    for (int t = 0; t < mine; ++t) {
      const int b = t & 1;
      const uint32_t s_addr = s_tile + b * 64;
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[g][b], (t >> 1) & 1, abort_word, p.a.err, 757));
      if (!ok) break;
      if (!idle) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->info_full[t & 3], (t >> 2) & 1, abort_word, p.a.err, 758));
        if (!ok) break;
        const float kf = bars->info[t & 3].k, ev = bars->info[t & 3].v;
        tc_fence_after();
        uint32_t sr[2][32];
        tmem_ld_32x32(s_addr, sr[0]);
        tmem_ld_32x32(s_addr + 32, sr[1]);
        tc_wait_ld();
        const int kv0 = (t0 + t) * 64;
        if (kv0 + 63 > limit) {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (kv0 + c > limit) sr[c >> 5][c & 31] = __float_as_uint(-INFINITY);
        }
        float mxa[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 64; ++c) mxa[c & 3] = fmaxf(mxa[c & 3], __uint_as_float(sr[c >> 5][c & 31]));
        const float mx = fmaf(fmaxf(fmaxf(mxa[0], mxa[1]), fmaxf(mxa[2], mxa[3])), kf, ev);       // kf > 0
        bool grow = false;
        if (unset) {
          unset = mx == -INFINITY;
          m = unset ? 0.f : mx;
        } else {
          grow = mx - m > 8.0f;
        }
        if (__any_sync(0xffffffffu, grow)) {
          ok = t == 0 || mbar_wait(&bars->pv_done[g][(t - 1) & 1], ((t - 1) >> 1) & 1, abort_word, p.a.err, 760);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const float factor = grow ? exp2f(m - mx) : 1.0f;
          if (grow) { m = mx; l *= factor; }
#pragma unroll
          for (int q4 = 0; q4 < HD / 32; ++q4) {
            uint32_t tr[32];
            tmem_ld_32x32(o_addr + q4 * 32, tr);
            tc_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) tr[c] = __float_as_uint(__uint_as_float(tr[c]) * factor);
            tmem_st_32x32(o_addr + q4 * 32, tr);
          }
        }
        float la[4] = {0.f, 0.f, 0.f, 0.f};
        const float shift = ev - m + kShift;
        uint32_t pk[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float p0 = ex2(fmaf(__uint_as_float(sr[j >> 4][2 * (j & 15)]), kf, shift));
          const float p1 = ex2(fmaf(__uint_as_float(sr[j >> 4][2 * (j & 15) + 1]), kf, shift));
          la[j & 3] += p0 + p1;
          pk[j] = pack_f16(p0, p1);
        }
        tmem_st_32x32(s_addr, pk);
        l = fmaf((la[0] + la[1]) + (la[2] + la[3]), pow2f(-static_cast<int>(ev)), l);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(&bars->p_full[g][b]);
    }
    if (ok && mine > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_done[g], 0, abort_word, p.a.err, 761));
    if (ok && (g == 0 || two)) {
      tc_fence_after();
      const float back = 1.f / (1 << kHeadroom);
      const int64_t out_row = valid ? w.qs + tq : 0;
      const float f = p.splits > 1 ? back : (l == 0.f ? 0.f : back / l);
      T* orow = static_cast<T*>(p.a.out) + out_row * p.a.ldo + static_cast<int64_t>(head) * HD;
      float* part = p.ws + ((static_cast<int64_t>(blockIdx.z) * p.a.T + out_row) * p.a.n_q + head) * (HD + 4);
#pragma unroll
      for (int q4 = 0; q4 < HD / 32; ++q4) {
        uint32_t ta[32];
        if (mine > 0) {
          tmem_ld_32x32(o_addr + q4 * 32, ta);      // warp-collective
          tc_wait_ld();
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) ta[c] = 0;
        }
        if (valid) {
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 v = make_float4(__uint_as_float(ta[c]), __uint_as_float(ta[c + 1]), __uint_as_float(ta[c + 2]), __uint_as_float(ta[c + 3]));
            if (p.splits == 1) store4(orow + q4 * 32 + c, v, f);
            else *reinterpret_cast<float4*>(part + q4 * 32 + c) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
          }
        }
      }
      if (valid && p.splits > 1) { part[HD] = unset ? kNoMax : m; part[HD + 1] = l; }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// The parts of each row, added up: a block per (plan tile, head), a warp per row in turn.
template <int HD, typename T>
__global__ void __launch_bounds__(256) chunk_join_kernel(const __grid_constant__ ChunkParams p) {
  pdl_wait();
  const MbFp8Attention& a = p.a;
  const int G = a.n_q / a.n_kv, tok = 64 / G, tile = blockIdx.y, kvh = blockIdx.x;
  const int seq = a.tile_seq[tile];
  if (seq < 0) return;
  const int tq0 = a.tile_q0[tile], ql = a.q_len[seq], qs = a.q_start[seq];
  const int rows = (min(tq0 + tok, ql) - tq0) * G, lane = threadIdx.x & 31;
  constexpr int PER = HD / 32;
  for (int r = threadIdx.x >> 5; r < rows; r += 8) {
    const int64_t row = qs + tq0 + r / G;
    if (row >= a.T) continue;
    const int head = kvh * G + r % G;
    const float* part = p.ws + (row * a.n_q + head) * (HD + 4);
    const int64_t step = static_cast<int64_t>(a.T) * a.n_q * (HD + 4);
    float m = kNoMax;
    for (int z = 0; z < p.splits; ++z) m = fmaxf(m, part[z * step + HD]);
    float l = 0.f, o[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = 0.f;
    for (int z = 0; z < p.splits; ++z) {
      const float* q = part + z * step;
      const float f = exp2f(q[HD] - m);
      l = fmaf(q[HD + 1], f, l);
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] = fmaf(q[lane * PER + i], f, o[i]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* dst = static_cast<T*>(a.out) + row * a.ldo + static_cast<int64_t>(head) * HD + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) dst[i] = static_cast<T>(o[i] * inv);
  }
}

// Parts per CTA's keys: as many as give every SM a CTA. A sequence of the plan has one CTA per head at least, four plan tiles at most share one.
static int chunk_splits(const MbFp8Attention& a, int num_sms) {
  const int ctas = max((a.n_tiles + 3) / 4, min(a.n_tiles, a.B - a.n_decode)) * a.n_kv;
  return max(1, min(kMaxSplits, num_sms / max(1, ctas)));
}

size_t chunk_workspace(const MbFp8Attention& a, int num_sms) {
  const int s = a.n_tiles > 0 ? chunk_splits(a, num_sms) : 1;
  return s > 1 ? static_cast<size_t>(s) * a.T * a.n_q * (a.head_dim + 4) * sizeof(float) : 0;
}

template <int HD, typename T>
static int launch(const MbFp8Attention& a, const MbFp8Cache& c, int num_sms, cudaStream_t stream) {
  static PerDeviceOnce configured;
  auto kern = chunk_kernel<HD, T>;
  if (configured.needed()) {
    // the register split inside the kernel adds up to what 512 threads of 128 registers bring along
    cudaFuncAttributes at;
    if (cudaFuncGetAttributes(&at, kern) != cudaSuccess || at.numRegs != 128) return MB_ERR_LAUNCH;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<HD>::kSmem)) != cudaSuccess) return MB_ERR_LAUNCH;
    configured.done();
  }
  ChunkParams p = {};
  p.a = a;
  p.c = c;
  p.ws = static_cast<float*>(a.ws);
  p.splits = chunk_splits(a, num_sms);
  p.box = c.page_size % 64 == 0 ? 64 : c.page_size % 32 == 0 ? 32 : 16;
  if (launch_k(kern, dim3(a.n_kv, a.n_tiles, p.splits), dim3(kThreads), Shape<HD>::kSmem, stream, p) != cudaSuccess) return MB_ERR_LAUNCH;
  if (p.splits > 1 && launch_k(chunk_join_kernel<HD, T>, dim3(a.n_kv, a.n_tiles), dim3(256), 0, stream, p) != cudaSuccess) return MB_ERR_LAUNCH;
  return MB_OK;
}

int chunk_attention(const MbFp8Attention& a, const MbFp8Cache& c, int num_sms, cudaStream_t stream) {
  if (a.n_tiles <= 0) return MB_OK;
  if (a.n_tiles > 65535) return MB_ERR_TOO_LARGE;
  if (a.ws_bytes < chunk_workspace(a, num_sms)) return MB_ERR_TOO_LARGE;
  if (a.head_dim == 128) return a.dtype == 0 ? launch<128, __nv_bfloat16>(a, c, num_sms, stream) : launch<128, __half>(a, c, num_sms, stream);
  return a.dtype == 0 ? launch<64, __nv_bfloat16>(a, c, num_sms, stream) : launch<64, __half>(a, c, num_sms, stream);
}

}  // namespace a8
}  // namespace mb
