// The 8-bit paged key/value cache: rotation and store of a step's tokens, and rows read back in 16 or 32 bits.
//
// A row x in R^d (a token's key or value of one head) is held as d e4m3 codes and one exponent byte:
//
//   e = min { e >= -100 : max |x_i| <= 448 * 2^e },   code_i = e4m3(x_i * 2^-e) (nearest, ties to even),   byte = e + 127
//
// e4m3 is a floating format, so a code's relative error is 2^-4 at most whatever the scale, and a power of two costs nothing
// against max / 448: it only shifts the point (15 binades below the largest value) where small values lose bits. In
// exchange every product with it is exact: a row reads back as the same numbers in bf16, fp32 and inside attention. What is not
// finite is held as NaN and left out of the maximum. -100 keeps 2^e and 2^-e inside fp32 with room for sums.
//
// Both kernels are bound by memory: 8 values a thread, one row of a head by d / 8 lanes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/api.h"
#include "../common/launch.h"
#include "../common/ptx.cuh"

namespace mb {
namespace kv8 {

constexpr int kLeastExp = -100;

template <typename T>
struct Pack8 {
  T v[8];
};
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  __align__(16) Pack8<T> r;
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  } else {
    reinterpret_cast<uint4*>(&r)[0] = reinterpret_cast<const uint4*>(p)[0];
    reinterpret_cast<uint4*>(&r)[1] = reinterpret_cast<const uint4*>(p)[1];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(r.v[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  __align__(16) Pack8<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = static_cast<T>(x[i]);       // one rounding to nearest
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
  } else {
    reinterpret_cast<uint4*>(p)[0] = reinterpret_cast<const uint4*>(&r)[0];
    reinterpret_cast<uint4*>(p)[1] = reinterpret_cast<const uint4*>(&r)[1];
  }
}

// a * c + b * s such that every later rounding to 16 or 8 bits falls on the side of the exact value: the products' and the sum's
// rounding errors are kept (each is exact), and a result that lands on a short number moves one place towards the remainder, so that it
// is no tie (nor the border of an exponent) by rounding alone. A flipped e4m3 code would be a step of 2^-3.
// (Where the result itself is kept, in fp32, it stays the nearest: `to_short` false.)
__device__ __forceinline__ float turned(float a, float c, float b, float s, bool to_short) {
  const float p = a * c, q = b * s;
  const float sum = p + q, back = sum - p;
  const float rest = ((p - (sum - back)) + (q - back)) + (fmaf(a, c, -p) + fmaf(b, s, -q));
  const float r = sum + rest;
  if (!(fabsf(r) <= 3.0e38f)) return sum;           // not finite
  const float d = (sum - r) + rest;
  uint32_t u = __float_as_uint(r);
  if (to_short && d != 0.f && (u & 0x7fffu) == 0 && r != 0.f) u += ((d > 0.f) == (r > 0.f)) ? 1u : 0xffffffffu;
  return __uint_as_float(u);
}

struct StoreParams {
  const void* qkv;
  void* q_out;
  const int32_t* positions;
  const int64_t* slots;
  const float* cos_sin;
  MbFp8Cache c;
  int* err;
  int ld, ldq, T, n_q, n_kv, hd, rot, n_positions, interleaved;
};

// A row is held by LANES lanes of a warp (hd / 8 of them at work); rows of a token in turn: queries, keys, values.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) store_kernel(const StoreParams p) {
  pdl_wait();
  const int rows = p.n_q + 2 * p.n_kv;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LANES;
  const int col = (threadIdx.x % LANES) * 8;
  const bool there = row < static_cast<int64_t>(p.T) * rows;
  const int t = there ? static_cast<int>(row / rows) : 0, h = there ? static_cast<int>(row - static_cast<int64_t>(t) * rows) : 0;
  const bool on = there && col < p.hd;
  const T* src = static_cast<const T*>(p.qkv) + static_cast<int64_t>(t) * p.ld + static_cast<int64_t>(h) * p.hd;
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (on) load8(src + col, x);
  const bool turns = h < p.n_q + p.n_kv && p.rot > 0, to_short = sizeof(T) == 2 || h >= p.n_q;
  int pos = 0;
  if (there && turns) {
    pos = p.positions[t];
    if (pos < 0 || pos >= p.n_positions) {          // no such angles: nothing is read, the row goes on as it is
      if (p.err) atomicCAS(p.err, 0, 721);
      pos = -1;
    }
  }
  if (on && turns && pos >= 0 && col < p.rot) {
    const int half = p.rot >> 1;
    const float* cs = p.cos_sin + static_cast<int64_t>(pos) * p.rot;
    if (p.interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pr = (col >> 1) + i;
        if (pr < half) {
          const float c = cs[pr], s = cs[half + pr], u = x[2 * i], w = x[2 * i + 1];
          x[2 * i] = turned(u, c, w, -s, to_short);
          x[2 * i + 1] = turned(w, c, u, s, to_short);
        }
      }
    } else if (half % 8 == 0) {
      const bool upper = col >= half;
      float y[8];
      load8(src + (upper ? col - half : col + half), y);
      const float* at = cs + (upper ? col - half : col);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = turned(x[i], at[i], y[i], upper ? at[half + i] : -at[half + i], to_short);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = col + i;
        if (j >= p.rot) continue;
        const bool upper = j >= half;
        const int k = upper ? j - half : j;
        const float y = static_cast<float>(src[upper ? k : j + half]);
        x[i] = turned(x[i], cs[k], y, upper ? cs[half + k] : -cs[half + k], to_short);
      }
    }
  }
  __syncwarp();                                     // in place: every lane of the row has read what it needs
  if (h < p.n_q) {
    if (on) store8(static_cast<T*>(p.q_out) + static_cast<int64_t>(t) * p.ldq + static_cast<int64_t>(h) * p.hd + col, x);
  }
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(x[i]);
    big = fmaxf(big, a < INFINITY ? a : 0.f);       // (NaN compares false)
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  if (!on || h < p.n_q) return;
  const int64_t slot = p.slots[t];
  if (slot < 0) return;
  if (slot >= static_cast<int64_t>(p.c.pages) * p.c.page_size) {
    if (p.err) atomicCAS(p.err, 0, 722);
    return;
  }
  const uint32_t u = __float_as_uint(big);
  int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);        // 448 = 1.75 * 2^8
  e = e < kLeastExp ? kLeastExp : e;
  const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  uint32_t packed[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float2 f;
      f.x = x[4 * i + 2 * k]; f.y = x[4 * i + 2 * k + 1];
      f.x = fabsf(f.x) < INFINITY ? f.x * inv : NAN;
      f.y = fabsf(f.y) < INFINITY ? f.y * inv : NAN;
      w |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3)) << (16 * k);
    }
    packed[i] = w;
  }
  const bool is_v = h >= p.n_q + p.n_kv;
  const int kvh = h - p.n_q - (is_v ? p.n_kv : 0);
  const int64_t page = slot / p.c.page_size;
  const int off = static_cast<int>(slot - page * p.c.page_size);
  uint8_t* codes = static_cast<uint8_t*>(is_v ? p.c.v : p.c.k) + page * (is_v ? p.c.v_page : p.c.k_page) + kvh * (is_v ? p.c.v_head : p.c.k_head) +
                   static_cast<int64_t>(off) * p.hd;
  *reinterpret_cast<uint2*>(codes + col) = make_uint2(packed[0], packed[1]);
  if (col == 0) {
    uint8_t* bytes = is_v ? p.c.vs + page * p.c.vs_page + kvh * p.c.vs_head : p.c.ks + page * p.c.ks_page + kvh * p.c.ks_head;
    bytes[off] = static_cast<uint8_t>(e + 127);
  }
}

template <typename T>
static int launch_store(const StoreParams& p, cudaStream_t stream) {
  const int lanes = p.hd <= 64 ? 8 : p.hd <= 128 ? 16 : 32;
  const int64_t threads = static_cast<int64_t>(p.T) * (p.n_q + 2 * p.n_kv) * lanes, blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffff) return MB_ERR_TOO_LARGE;
  auto kern = lanes == 8 ? store_kernel<T, 8> : lanes == 16 ? store_kernel<T, 16> : store_kernel<T, 32>;
  return launch_k(kern, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, p) == cudaSuccess ? MB_OK : MB_ERR_LAUNCH;
}

// Rows [0, kv_len[s]) of every sequence at kv_start[s] of the outputs; 16 values a thread, keys and values as grid.y. Rows that belong to
// no sequence are zeros.
template <typename T>
__global__ void __launch_bounds__(256) load_kernel(const MbFp8Cache c, const int32_t* __restrict__ block_table, int bt_stride,
                                                   const int32_t* __restrict__ kv_start, const int32_t* __restrict__ kv_len, int B, int64_t rows,
                                                   int n_kv, int hd, T* __restrict__ k_out, T* __restrict__ v_out, int* err) {
  pdl_wait();
  const int per = n_kv * (hd / 16);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= rows * per) return;
  const int64_t row = i / per;
  const int at = static_cast<int>(i - row * per), h = at / (hd / 16), col = (at % (hd / 16)) * 16;
  int lo = 0, hi = B - 1;                            // the last sequence that starts at or before the row
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (kv_start[m] <= row) lo = m; else hi = m - 1;
  }
  const int64_t pos = row - kv_start[lo];
  T* dst = (blockIdx.y ? v_out : k_out) + (row * n_kv + h) * hd + col;
  float x[2][8];
#pragma unroll
  for (int k = 0; k < 16; ++k) x[k >> 3][k & 7] = 0.f;
  if (pos >= 0 && pos < kv_len[lo]) {
    const int64_t nth = pos / c.page_size;
    const int page = nth < bt_stride ? block_table[static_cast<int64_t>(lo) * bt_stride + nth] : -1, off = static_cast<int>(pos % c.page_size);
    if (page < 0 || page >= c.pages) {
      if (err) atomicCAS(err, 0, 723);
    } else {
      const uint8_t* codes = blockIdx.y ? static_cast<const uint8_t*>(c.v) + page * c.v_page + h * c.v_head
                                        : static_cast<const uint8_t*>(c.k) + page * c.k_page + h * c.k_head;
      const uint8_t byte = blockIdx.y ? c.vs[page * c.vs_page + h * c.vs_head + off] : c.ks[page * c.ks_page + h * c.ks_head + off];
      const uint4 w = *reinterpret_cast<const uint4*>(codes + static_cast<int64_t>(off) * hd + col);
      const float f = __uint_as_float(byte == 0 ? 0x400000u : static_cast<uint32_t>(byte) << 23);   // (2^-127 is no normal number)
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(words[k >> 1] >> (16 * (k & 1))), __NV_E4M3);
        const float2 v = __half22float2(__half2(r));
        x[k >> 2][2 * (k & 3)] = v.x * f;
        x[k >> 2][2 * (k & 3) + 1] = v.y * f;
      }
    }
  }
  store8(dst, x[0]);
  store8(dst + 8, x[1]);
}

}  // namespace kv8
}  // namespace mb

using namespace mb;

static int check_cache(const MbFp8Cache* c, int n_kv, int head_dim) {
  if (c->page_size < 16 || c->page_size % 16 || c->pages < 1 || n_kv < 1 || head_dim < 16 || head_dim > 256 || head_dim % 16) return MB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) | reinterpret_cast<uintptr_t>(c->ks) | reinterpret_cast<uintptr_t>(c->vs) |
       static_cast<uintptr_t>(c->k_page | c->k_head | c->v_page | c->v_head | c->ks_page | c->ks_head | c->vs_page | c->vs_head)) & 15)
    return MB_ERR_ALIGN;
  return MB_OK;
}

extern "C" int mb_rope_kv_store_fp8(const void* qkv, int ld, void* q_out, int ldq, int dtype, const int32_t* positions, const int64_t* slots,
                                    const float* cos_sin, int n_positions, const MbFp8Cache* cache, int T, int n_q, int n_kv, int head_dim,
                                    int rot_dims, int interleaved, int* err, cudaStream_t stream) {
  using namespace mb::kv8;
  if (T <= 0) return MB_OK;
  const int rc = check_cache(cache, n_kv, head_dim);
  if (rc != MB_OK) return rc;
  if (n_q < 0 || rot_dims < 0 || rot_dims % 2 || rot_dims > head_dim || (rot_dims && n_positions < 1)) return MB_ERR_SHAPE;
  if (((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & 15) || ld % 8 || ldq % 8) return MB_ERR_ALIGN;
  StoreParams p = {};
  p.qkv = qkv; p.q_out = q_out; p.positions = positions; p.slots = slots; p.cos_sin = cos_sin; p.c = *cache; p.err = err;
  p.ld = ld; p.ldq = ldq; p.T = T; p.n_q = n_q; p.n_kv = n_kv; p.hd = head_dim; p.rot = rot_dims; p.n_positions = n_positions;
  p.interleaved = interleaved;
  switch (dtype) {
    case 0: return launch_store<__nv_bfloat16>(p, stream);
    case 1: return launch_store<float>(p, stream);
    case 2: return launch_store<__half>(p, stream);
  }
  return MB_ERR_SHAPE;
}

extern "C" int mb_kv_load_fp8(const MbFp8Cache* cache, const int32_t* block_table, int bt_stride, const int32_t* kv_start, const int32_t* kv_len,
                              int B, long long rows, int n_kv, int head_dim, void* k_out, void* v_out, int dtype, int* err, cudaStream_t stream) {
  using namespace mb::kv8;
  if (rows <= 0) return MB_OK;
  const int rc = check_cache(cache, n_kv, head_dim);
  if (rc != MB_OK) return rc;
  if (B < 1) return MB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) return MB_ERR_ALIGN;
  const long long blocks = (rows * n_kv * (head_dim / 16) + 255) / 256;
  if (blocks > 0x7fffffff) return MB_ERR_TOO_LARGE;
  const dim3 grid(static_cast<unsigned>(blocks), 2);
  cudaError_t e;
  switch (dtype) {
    case 0: e = launch_k(load_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, *cache, block_table, bt_stride, kv_start, kv_len, B, rows, n_kv, head_dim, static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), err); break;
    case 1: e = launch_k(load_kernel<float>, grid, dim3(256), 0, stream, *cache, block_table, bt_stride, kv_start, kv_len, B, rows, n_kv, head_dim, static_cast<float*>(k_out), static_cast<float*>(v_out), err); break;
    case 2: e = launch_k(load_kernel<__half>, grid, dim3(256), 0, stream, *cache, block_table, bt_stride, kv_start, kv_len, B, rows, n_kv, head_dim, static_cast<__half*>(k_out), static_cast<__half*>(v_out), err); break;
    default: return MB_ERR_SHAPE;
  }
  return e == cudaSuccess ? MB_OK : MB_ERR_LAUNCH;
}
