// Attention of sequences of few rows (single tokens, up to 16 query rows per key/value head) over the 8-bit paged cache.
//
// What bounds it is reading the cache: 2 (HD + 1) bytes a token and head, and 24 codes a cycle and SM to unpack on the way.
//
//   * The 64-token tiles of all sequences are one line of work per head, cut into equal shares (two tiles at least) for as many CTAs
//     as the SMs hold. A sequence inside one share is finished there; the pieces of one that is cut go to the workspace and
//     join_kernel puts them together, in the order of the shares.
//   * A CTA is a producer warp (TMA: K and V boxes, bulk copies of the exponents, a ring of stages) and two pairs of warps that take the tiles in
//     turn, 32 tokens a warp, for all query rows (the 16 rows of one mma.sync m16n8k16, f16 operands, fp32 sums).
//   * Codes become f16 in registers, exactly and without their scale. A lane's 16 bytes of a key are the operands of four k-steps (the order of
//     k is free as long as the queries, loaded once, have the same). Values come through ldmatrix.trans as byte pairs, one permutation
//     and one conversion per two values; even and odd columns are separate MMA columns.
//   * Scales are whole powers of two and ride on the exponents of the softmax: with t_j = log2(e) scale q.k_j 2^ek_j + ev_j the numerator
//     weights are 2^(t_j - m) <= 2^8, which are P for the raw codes of V, and the denominator adds 2^(t_j - m) 2^-ev_j. So a row of small
//     values beside one of large values loses nothing. m lags: it moves when a weight would exceed 2^8, and P carries 2^7 more, so that
//     weights down to 2^-21 keep all bits of f16.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/api.h"
#include "../common/launch.h"
#include "../common/ptx.cuh"
#include "attention_fp8.cuh"
#include "gemm_common.h"

namespace mb {
namespace a8 {

constexpr int kDecStages = 6;
constexpr int kDecCtas = 2;             // per SM
constexpr int kMinShare = 2;            // tiles
constexpr int kDecThreads = 160;
constexpr int kMaxDecode = 4096;        // sequences of a launch (their tile counts wait in shared memory)

struct DecParams {
  MbFp8Attention a;
  MbFp8Cache c;
  float* ws;
  int box, GX, rows_alloc;   // rows of a box; CTAs of a head; query rows kept in a partial result
};

struct DecBars {
  uint64_t full[kDecStages];
  uint64_t empty[kDecStages];
  int abort_word;
  int warp_sum[5];
};

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// tiles of sequence i of the decode list
__device__ __forceinline__ int tiles_of(const MbFp8Attention& a, int i) {
  const int seq = a.decode_seq[i];
  if (seq < 0) return 0;
  return (max(a.kv_len[seq], 0) + 63) >> 6;
}
// share of CTA g: [U g / G, U (g + 1) / G) with G the CTAs that get at least kMinShare tiles
__device__ __forceinline__ int shares_of(int U, int GX) { return max(1, min(GX, U / kMinShare)); }
__device__ __forceinline__ int share_start(int U, int G, int g) { return static_cast<int>(static_cast<int64_t>(U) * g / G); }
__device__ __forceinline__ int share_holding(int U, int G, int u) { return static_cast<int>(((static_cast<int64_t>(u) + 1) * G - 1) / U); }

// A partial result: fp32 O [rows][HD], then m [16], l [16]; two slots per CTA (its first and its last sequence)
template <int HD>
__host__ __device__ constexpr int slot_floats(int rows) { return rows * HD + 32; }

// Rows g and g + 8 of a warp's state, columns 16 c + 4 t4 + {0, 2} of the even and {1, 3} of the odd MMA columns of chunk c
template <int HD>
struct RowState {
  float o[HD / 8][4];
  float m[2], l[2];
};

// Token order inside a group of 8: with 128-byte rows tokens 0, 4, 1, 5, .. alternate between the halves of the swizzle, so that the eight lanes
// of a quarter-warp read from all banks.
template <int HD>
__device__ __forceinline__ int order(int n) { return HD == 128 ? (n >> 1) + (n & 1) * 4 : n; }

// 32 tokens from key k0 on, rows row0 and up of the tile. sE: exponent bytes of the keys, those of the values 64 bytes behind. Four groups of eight
// tokens side by side: one group's products wait for one another.
template <int HD, bool EDGE>
__device__ __forceinline__ void walk32(RowState<HD>& st, const uint32_t (&qf)[HD / 16][4], uint32_t sK, uint32_t sV, uint32_t sE, float sc, int row0,
                                       int lane, int k0, int kl, const int (&limit)[2]) {
  const int g = lane >> 2, t4 = lane & 3;
  // ---- scores of 4 x 8 tokens
  float c[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
#pragma unroll
  for (int n = 0; n < HD / 64; ++n) {
    uint4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = row0 + j * 8 + order<HD>(g), chunk = n * 4 + t4;
      w[j] = lds128(sK + (HD == 128 ? row * 128 + ((chunk ^ (row & 7)) << 4) : row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4)));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t lo, hi;
        codes_f16(k == 0 ? w[j].x : k == 1 ? w[j].y : k == 2 ? w[j].z : w[j].w, lo, hi);
        mma_f16(c[j], qf[n * 4 + k], lo, hi);
      }
  }
  // ---- weights: column 2 t4 + e of group j is token 8 j + order(2 t4 + e). Its byte becomes a float's exponent (the scale of K), a float (the
  // exponent of V, as the low bits of 2^23) and an exponent again (the way back).
  float back[4][2];
  bool grow = false;
  float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int jj = 0; jj < 2; ++jj) {
    const uint4 kb4 = lds128(sE + jj * 16), vb4 = lds128(sE + 64 + jj * 16);
    const uint32_t kb[4] = {kb4.x, kb4.y, kb4.z, kb4.w}, vb[4] = {vb4.x, vb4.y, vb4.z, vb4.w};
#pragma unroll
    for (int j2 = 0; j2 < 2; ++j2)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = jj * 2 + j2, tok = j * 8 + order<HD>(2 * t4 + e);
        // HD 128: tokens t4, 4 + t4 of group j, byte t4 of a word each; HD 64: tokens 2 t4 and 2 t4 + 1
        const uint32_t sel = HD == 128 ? t4 : 2 * (t4 & 1) + e;
        const uint32_t kw = HD == 128 ? kb[2 * j2 + e] : (t4 < 2 ? kb[2 * j2] : kb[2 * j2 + 1]);
        const uint32_t vw = HD == 128 ? vb[2 * j2 + e] : (t4 < 2 ? vb[2 * j2] : vb[2 * j2 + 1]);
        const float ak = __uint_as_float(__byte_perm(kw, 0, 0x4440 | sel) << 23) * sc;
        const uint32_t vbyte = __byte_perm(vw, 0x4B000000u, 0x7440 | sel);       // 2^23 + byte
        const float ev = fmaxf(__uint_as_float(vbyte) - 8388735.f, -100.f);
        back[j][e] = fminf(__uint_as_float((0x4B0000FEu - vbyte) << 23), 1.2676506e30f);        // 2^-ev, 2^100 at most
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x = fmaf(c[j][2 * h + e], ak, ev);
          if (EDGE) x = k0 + tok <= limit[h] ? x : -INFINITY;
          c[j][2 * h + e] = x;
          top[h] = fmaxf(top[h], x);
        }
      }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) grow |= top[h] > st.m[h] + 8.f;
  if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(st.m[h], mx), f = exp2f(st.m[h] - mn);
      st.m[h] = mn;
      st.l[h] *= f;
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) { st.o[d][2 * h] *= f; st.o[d][2 * h + 1] *= f; }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float ref = st.m[h] - kShift;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float pv = ex2(c[j][2 * h + e] - ref);
        c[j][2 * h + e] = pv;
        // (the byte of a key that is not there may be anything)
        st.l[h] = fmaf(pv, EDGE && pv == 0.f ? 0.f : back[j][e], st.l[h]);
      }
  }
  // ---- values. Rows behind the last key are zeroed: they may hold anything, NaN among it
#pragma unroll
  for (int jj = 0; jj < 2; ++jj) {
    const uint32_t pa[4] = {pack_f16(c[2 * jj][0], c[2 * jj][1]), pack_f16(c[2 * jj][2], c[2 * jj][3]), pack_f16(c[2 * jj + 1][0], c[2 * jj + 1][1]),
                            pack_f16(c[2 * jj + 1][2], c[2 * jj + 1][3])};
    uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
    if (EDGE) {
      const int valid = kl - k0 - jj * 16;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        keep[j] = (j * 8 + order<HD>(2 * t4) < valid ? 0xffffu : 0u) | (j * 8 + order<HD>(2 * t4 + 1) < valid ? 0xffff0000u : 0u);
    }
    const int row = row0 + jj * 16 + ((lane >> 3) & 1) * 8 + order<HD>(lane & 7);
#pragma unroll
    for (int cp = 0; cp < HD / 32; ++cp) {
      const int chunk = 2 * cp + (lane >> 4);
      uint32_t r[4];
      ldsm_x4_t(r, sV + (HD == 128 ? row * 128 + ((chunk ^ (row & 7)) << 4) : row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4)));
      if (EDGE) { r[0] &= keep[0]; r[1] &= keep[1]; r[2] &= keep[0]; r[3] &= keep[1]; }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t even[2], odd[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) codes_f16(__byte_perm(r[2 * k + j], 0, 0x3120), even[j], odd[j]);
        mma_f16(st.o[(2 * cp + k) * 2], pa, even[0], even[1]);
        mma_f16(st.o[(2 * cp + k) * 2 + 1], pa, odd[0], odd[1]);
      }
    }
  }
}

template <int HD, typename T>
__global__ void __launch_bounds__(kDecThreads, kDecCtas)
decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ DecParams p) {
  constexpr int kCodes = 64 * HD, kStage = 2 * kCodes;
  constexpr int NH = HD / 64;                       // 64-column halves of a row
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {                     // (no static shared memory: the window starts aligned)
    if (threadIdx.x == 0 && p.a.err) atomicCAS(p.a.err, 0, 749);
    return;
  }
  uint8_t* sScale = smem + kDecStages * kStage;     // [stage][K 64 | V 64]
  float* sO = reinterpret_cast<float*>(sScale + kDecStages * 128);        // [16][HD + 4]: the four warps' results joined
  float* sML = sO + 16 * (HD + 4);                                         // [warp][m 16 | l 16]
  DecBars& bars = *reinterpret_cast<DecBars*>(sML + 128);
  int* prefix = reinterpret_cast<int*>(&bars + 1);                         // [n_decode + 1]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.y, nd = p.a.n_decode, G = p.a.n_q / p.a.n_kv;
  if (tid == 0) {
    for (int s = 0; s < kDecStages; ++s) { mbar_init(&bars.full[s], 1); mbar_init(&bars.empty[s], 2); }
    bars.abort_word = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  pdl_wait();
  // running sums of the tile counts
  int run = 0;
  for (int base = 0; base < nd; base += kDecThreads) {
    const int i = base + tid;
    int v = i < nd ? tiles_of(p.a, i) : 0, mine = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += w;
    }
    if (lane == 31) bars.warp_sum[warp] = v;
    __syncthreads();
    int before = run;
    for (int w = 0; w < warp; ++w) before += bars.warp_sum[w];
    if (i < nd) prefix[i] = before + v - mine;
    for (int w = 0; w < 5; ++w) run += bars.warp_sum[w];
    __syncthreads();
  }
  if (tid == 0) prefix[nd] = run;
  __syncthreads();
  const int U = run, GE = shares_of(U, p.GX), gx = blockIdx.x;
  if (gx == 0) {
    // rows of sequences without keys
    for (int i = 0; i < nd; ++i) {
      if (prefix[i + 1] != prefix[i]) continue;
      const int seq = p.a.decode_seq[i];
      if (seq < 0) continue;
      const int qs = p.a.q_start[seq], n = min(p.a.q_len[seq] * G, 16);
      for (int k = tid; k < n * HD; k += kDecThreads) {
        const int r = k / HD, row = qs + r / G;
        if (row < p.a.T) static_cast<T*>(p.a.out)[static_cast<int64_t>(row) * p.a.ldo + (kvh * G + r % G) * HD + k % HD] = static_cast<T>(0.f);
      }
    }
  }
  if (gx >= GE || U == 0) { pdl_trigger(); return; }
  const int u0 = share_start(U, GE, gx), u1 = share_start(U, GE, gx + 1);
  int first;                                        // the sequence that holds tile u0: the last i with prefix[i] <= u0
  {
    int lo = 0, hi = nd - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= u0) lo = mid; else hi = mid - 1;
    }
    first = lo;
  }
  volatile int* abort_word = &bars.abort_word;

  if (warp == 4) {
    // ---------------------------------------------------------------- producer: 32 lanes fetch page numbers, lane 0 issues
    const int per = 64 / p.box;                     // boxes of a tile
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int i = first, u = u0; u < u1 && ok; ++i) {
      const int fu = prefix[i], t1 = min(prefix[i + 1], u1) - fu;
      if (t1 <= u - fu) continue;
      const int seq = p.a.decode_seq[i], kl = p.a.kv_len[seq];
      const int32_t* bt = p.a.block_table + static_cast<int64_t>(seq) * p.a.bt_stride;
      int page_lane = 0, have = 0, at = 0;          // pages of the next 32 boxes
      for (int t = u - fu; t < t1 && ok; ++t) {
        const int left = kl - t * 64, boxes = min(per, (left + p.box - 1) / p.box);
        ok = mbar_wait(&bars.empty[s], ph ^ 1, abort_word, p.a.err, 741);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        uint8_t* dst = smem + s * kStage;
        if (lane == 0) mbar_arrive_expect_tx(&bars.full[s], static_cast<uint32_t>(boxes) * p.box * (2 * HD + 2));
        for (int b = 0; b < boxes; ++b, ++at) {
          if (at == have) {
            at = 0;
            have = 32;
            const int tok = t * 64 + (b + lane) * p.box, nth = tok / p.c.page_size;
            page_lane = 0;
            if (tok < kl) {
              page_lane = nth < p.a.bt_stride ? bt[nth] : -1;
              if (page_lane < 0 || page_lane >= p.c.pages) {       // reported; some page stands in for it
                if (p.a.err) atomicCAS(p.a.err, 0, 731);
                page_lane = 0;
              }
            }
          }
          const int page = __shfl_sync(0xffffffffu, page_lane, at);
          if (lane == 0) {
            const int off = (t * 64 + b * p.box) % p.c.page_size;
            tma_load_4d(dst + b * p.box * HD, &tmK, &bars.full[s], 0, off, kvh, page);
            tma_load_4d(dst + kCodes + b * p.box * HD, &tmV, &bars.full[s], 0, off, kvh, page);
            bulk_load(sScale + s * 128 + b * p.box, p.c.ks + page * p.c.ks_page + kvh * p.c.ks_head + off, p.box, &bars.full[s]);
            bulk_load(sScale + s * 128 + 64 + b * p.box, p.c.vs + page * p.c.vs_page + kvh * p.c.vs_head + off, p.box, &bars.full[s]);
          }
        }
        if (++s == kDecStages) { s = 0; ph ^= 1; }
      }
      u = fu + t1;
    }
    pdl_trigger();
    return;
  }

  // ------------------------------------------------------------------ two pairs of warps take tiles in turn, 32 tokens a warp
  const int g = lane >> 2, t4 = lane & 3;
  int s = 0, turn = 0;
  uint32_t ph = 0;
  bool ok = true;
  for (int i = first, u = u0; u < u1; ++i) {
    const int fu = prefix[i], nt = prefix[i + 1] - fu, ta = u - fu, tb = min(prefix[i + 1], u1) - fu;
    if (tb <= ta) continue;
    u = fu + tb;
    const int seq = p.a.decode_seq[i];
    const int qs = p.a.q_start[seq], ql = p.a.q_len[seq], kl = p.a.kv_len[seq];
    const int rows = min(ql * G, 16);
    // queries: columns [16 t4, 16 t4 + 16) of each half of rows g and g + 8
    uint32_t qf[NH * 4][4];
    float qbig = 0.f;
    float qv[2][NH][16];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = g + 8 * h, row = qs + r / G;
      const bool valid = r < rows && row < p.a.T;
      const T* src = static_cast<const T*>(p.a.q) + static_cast<int64_t>(valid ? row : 0) * p.a.ldq + (kvh * G + r % G) * HD + t4 * 16;
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        load16(src + n * 64, qv[h][n], valid);
#pragma unroll
        for (int k = 0; k < 16; ++k) qbig = fmaxf(qbig, finite_abs(qv[h][n][k]));
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) qbig = fmaxf(qbig, __shfl_xor_sync(0xffffffffu, qbig, o));
    const int qe = f16_shift(qbig);
    const float qmul = pow2f(qe);
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        qf[n * 4 + k][0] = pack_f16(qv[0][n][4 * k] * qmul, qv[0][n][4 * k + 1] * qmul);
        qf[n * 4 + k][1] = pack_f16(qv[1][n][4 * k] * qmul, qv[1][n][4 * k + 1] * qmul);
        qf[n * 4 + k][2] = pack_f16(qv[0][n][4 * k + 2] * qmul, qv[0][n][4 * k + 3] * qmul);
        qf[n * 4 + k][3] = pack_f16(qv[1][n][4 * k + 2] * qmul, qv[1][n][4 * k + 3] * qmul);
      }
    const float sc = score_factor(p.a.scale * kLog2e, -qe);
    RowState<HD> st;
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) st.o[d][0] = st.o[d][1] = st.o[d][2] = st.o[d][3] = 0.f;
    st.m[0] = st.m[1] = kNoMax;
    st.l[0] = st.l[1] = 0.f;
    int limit[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) limit[h] = g + 8 * h < rows ? kl - ql + (g + 8 * h) / G : -1;

    for (int t = ta; t < tb; ++t) {
      const bool mine = turn == warp >> 1;
      turn ^= 1;
      if (mine && ok) {
        // (after a failed wait a warp skips the remaining tiles but meets the others at every barrier)
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.full[s], ph, abort_word, p.a.err, 742));
        if (ok) {
          const int row0 = (warp & 1) * 32, k0 = t * 64 + row0;     // first of this warp's tokens
          const uint32_t sK = smem_u32(smem + s * kStage), sV = sK + kCodes, sE = smem_u32(sScale + s * 128 + row0);
          // the last tokens of a sequence are masked row by row; before them every row sees all
          if (k0 + 32 <= kl - ql + 1) walk32<HD, false>(st, qf, sK, sV, sE, sc, row0, lane, k0, kl, limit);
          else if (k0 < kl) walk32<HD, true>(st, qf, sK, sV, sE, sc, row0, lane, k0, kl, limit);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.empty[s]);
        }
      }
      if (++s == kDecStages) { s = 0; ph ^= 1; }
    }

    // ---- the four warps' states become one, in the order of the warps
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      st.l[h] += __shfl_xor_sync(0xffffffffu, st.l[h], 1);
      st.l[h] += __shfl_xor_sync(0xffffffffu, st.l[h], 2);
      if (t4 == 0) { sML[warp * 32 + g + 8 * h] = st.m[h]; sML[warp * 32 + 16 + g + 8 * h] = st.l[h]; }
    }
    consumers_sync();
    float f[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = kNoMax;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, sML[w * 32 + g + 8 * h]);
      f[h] = exp2f(st.m[h] - top);
    }
    for (int w = 0; w < 4; ++w) {
      if (warp == w) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (g + 8 * h < rows) {
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
              float4* at = reinterpret_cast<float4*>(sO + (g + 8 * h) * (HD + 4) + c * 16 + t4 * 4);
              float4 v = w == 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *at;
              v.x = fmaf(st.o[2 * c][2 * h], f[h], v.x);
              v.y = fmaf(st.o[2 * c + 1][2 * h], f[h], v.y);
              v.z = fmaf(st.o[2 * c][2 * h + 1], f[h], v.z);
              v.w = fmaf(st.o[2 * c + 1][2 * h + 1], f[h], v.w);
              *at = v;
            }
          }
        }
      }
      consumers_sync();
    }
    const bool whole = ta == 0 && tb == nt;
    // a piece that begins its CTA's share goes to slot 0, one that ends it to slot 1
    float* slot = p.ws + (static_cast<int64_t>(kvh * p.GX + gx) * 2 + (ta > 0 ? 0 : 1)) * slot_floats<HD>(p.rows_alloc);
    for (int k = tid; k < rows * (HD / 4); k += 128) {
      const int r = k / (HD / 4), col = (k % (HD / 4)) * 4;
      float top = kNoMax, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, sML[w * 32 + r]);
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += sML[w * 32 + 16 + r] * exp2f(sML[w * 32 + r] - top);
      const float4 v = *reinterpret_cast<const float4*>(sO + r * (HD + 4) + col);
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int row = qs + r / G;
        if (row < p.a.T) store4(static_cast<T*>(p.a.out) + static_cast<int64_t>(row) * p.a.ldo + (kvh * G + r % G) * HD + col, v, inv);
      } else {
        *reinterpret_cast<float4*>(slot + r * HD + col) = v;
        if (col == 0) { slot[p.rows_alloc * HD + r] = top; slot[p.rows_alloc * HD + 16 + r] = sum; }
      }
    }
    consumers_sync();                               // sO and sML are free for the next sequence
  }
}

// Sequences that lie in several shares: a block per (sequence, head) finds them by the same sums and adds the pieces up.
template <int HD, typename T>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ DecParams p) {
  __shared__ int part[4], part_all[4];
  pdl_wait();
  const int i = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x, nd = p.a.n_decode, G = p.a.n_q / p.a.n_kv;
  int before = 0, all = 0;
  for (int k = tid; k < nd; k += 128) {
    const int n = tiles_of(p.a, k);
    all += n;
    if (k < i) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if ((tid & 31) == 0) { part[tid >> 5] = before; part_all[tid >> 5] = all; }
  __syncthreads();
  const int fu = part[0] + part[1] + part[2] + part[3], U = part_all[0] + part_all[1] + part_all[2] + part_all[3];
  const int nt = tiles_of(p.a, i);
  if (nt == 0) return;
  const int GE = shares_of(U, p.GX), g0 = share_holding(U, GE, fu), g1 = share_holding(U, GE, fu + nt - 1);
  if (g0 == g1) return;                              // finished by its CTA
  const int seq = p.a.decode_seq[i], qs = p.a.q_start[seq], rows = min(p.a.q_len[seq] * G, 16);
  const float* base = p.ws + static_cast<int64_t>(kvh) * p.GX * 2 * slot_floats<HD>(p.rows_alloc);
  auto slot_of = [&](int g) { return base + (static_cast<int64_t>(g) * 2 + (share_start(U, GE, g) > fu ? 0 : 1)) * slot_floats<HD>(p.rows_alloc); };
  for (int k = tid; k < rows * (HD / 4); k += 128) {
    const int r = k / (HD / 4), col = (k % (HD / 4)) * 4;
    float m = kNoMax, l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g = g0; g <= g1; ++g) {
      const float* slot = slot_of(g);
      const float mg = slot[p.rows_alloc * HD + r], lg = slot[p.rows_alloc * HD + 16 + r];
      const float4 x = *reinterpret_cast<const float4*>(slot + r * HD + col);
      const float mn = fmaxf(m, mg), a = exp2f(m - mn), b = exp2f(mg - mn);
      m = mn;
      l = l * a + lg * b;
      v.x = v.x * a + x.x * b; v.y = v.y * a + x.y * b; v.z = v.z * a + x.z * b; v.w = v.w * a + x.w * b;
    }
    const int row = qs + r / G;
    if (row < p.a.T) store4(static_cast<T*>(p.a.out) + static_cast<int64_t>(row) * p.a.ldo + (kvh * G + r % G) * HD + col, v, l == 0.f ? 0.f : 1.f / l);
  }
}

static int decode_ctas(int n_kv, int num_sms) { return max(1, kDecCtas * num_sms / n_kv); }

size_t decode_workspace(int n_decode, int n_q, int n_kv, int head_dim, int num_sms) {
  if (n_decode <= 0) return 0;
  return static_cast<size_t>(n_kv) * decode_ctas(n_kv, num_sms) * 2 * (16 * head_dim + 32) * sizeof(float);
}

template <int HD, typename T>
static int launch(const MbFp8Attention& a, const MbFp8Cache& c, int num_sms, cudaStream_t stream) {
  static PerDeviceOnce configured;
  auto kern = decode_kernel<HD, T>;
  const size_t fixed = kDecStages * (2 * 64 * HD + 128) + (16 * (HD + 4) + 128) * sizeof(float) + sizeof(DecBars);
  if (configured.needed()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(fixed + (kMaxDecode + 1) * sizeof(int))) != cudaSuccess)
      return MB_ERR_LAUNCH;
    configured.done();
  }
  DecParams p = {};
  p.c = c;
  p.box = c.page_size % 64 == 0 ? 64 : c.page_size % 32 == 0 ? 32 : 16;
  p.GX = decode_ctas(a.n_kv, num_sms);
  p.rows_alloc = 16;
  p.ws = static_cast<float*>(a.ws);
  CUtensorMap tk, tv;
  auto map = [&](CUtensorMap* m, const void* base, long long head, long long page) {
    const uint64_t h = a.n_kv > 1 ? head : static_cast<uint64_t>(c.page_size) * HD;
    return make_tmap_pages(m, base, HD, c.page_size, a.n_kv, c.pages, h, c.pages > 1 ? page : h * a.n_kv, p.box);
  };
  int rc = map(&tk, c.k, c.k_head, c.k_page);
  if (rc == MB_OK) rc = map(&tv, c.v, c.v_head, c.v_page);
  if (rc != MB_OK) return rc;
  for (int at = 0; at < a.n_decode; at += kMaxDecode) {
    p.a = a;
    p.a.decode_seq = a.decode_seq + at;
    p.a.n_decode = min(kMaxDecode, a.n_decode - at);
    const size_t smem = fixed + (p.a.n_decode + 1) * sizeof(int);
    if (launch_k(kern, dim3(p.GX, a.n_kv), dim3(kDecThreads), smem, stream, tk, tv, p) != cudaSuccess) return MB_ERR_LAUNCH;
    if (launch_k(join_kernel<HD, T>, dim3(p.a.n_decode, a.n_kv), dim3(128), 0, stream, p) != cudaSuccess) return MB_ERR_LAUNCH;
  }
  return MB_OK;
}

int decode_attention(const MbFp8Attention& a, const MbFp8Cache& c, int num_sms, cudaStream_t stream) {
  if (a.n_decode <= 0) return MB_OK;
  if (a.ws_bytes < decode_workspace(a.n_decode, a.n_q, a.n_kv, a.head_dim, num_sms)) return MB_ERR_TOO_LARGE;
  if (a.head_dim == 128) return a.dtype == 0 ? launch<128, __nv_bfloat16>(a, c, num_sms, stream) : launch<128, __half>(a, c, num_sms, stream);
  return a.dtype == 0 ? launch<64, __nv_bfloat16>(a, c, num_sms, stream) : launch<64, __half>(a, c, num_sms, stream);
}

}  // namespace a8
}  // namespace mb
