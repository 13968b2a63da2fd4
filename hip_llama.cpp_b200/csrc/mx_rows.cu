// Rows into microscaled numbers and back, and the norm that ends in them (tha_mx_t).
//   mx_quant_kernel          a warp takes 512 consecutive values of a row at a time: two or four lanes a block, whose largest |value| is a maximum of bit patterns
//   mx_read_kernel           16 bytes of results a lane (mx_read_lanes_kernel: rows on no boundary)
//   mx_add_norm_kernel       a block of threads takes a row: x + left, the square sum in fp64, the norm, its codes
//   mx_add_norm_ring_kernel  the same for many wide rows, which come through a ring; mx_add_norm_wide_kernel: rows beyond what registers hold
// A value is read and written once: bound by memory, quantising at 5.4 TB/s (11008 x 4096 bf16 to 4 bits 21.2 us) to 6.1 (fp32 to 8 bits 37.0), reading back at 4.7 (4 bits to bf16 24.2) and
// 5.1 (8 bits to fp32 44.3); where values are 16 bits or less the instructions for each are as many as the SMs issue meanwhile.
#include <cuda_fp16.h>

#include "hybrid_ops.cuh"
#include "mx.cuh"
#include "tc_common.cuh"
#include "workspace.h"

namespace tha {

int mx_refuse(const char* who, const char* why) {
  char text[256];
  snprintf(text, sizeof text, "%s: %s", who, why);
  set_last_error(text, cudaErrorInvalidValue);
  return THA_STATUS_INVALID_ARG;
}
int mx_check(const tha_mx_t* m, const char* who) {
  if (!m) return mx_refuse(who, "a matrix is NULL");
  if (m->format != THA_MX_E2M1 && m->format != THA_MX_E4M3) return mx_refuse(who, "unknown format");
  if (m->rows < 0 || m->rows > MX_MOST || m->cols < 1 || m->cols > MX_MOST) return mx_refuse(who, "a matrix has at least one column, and 2^30 rows and columns at most");
  if (m->rows == 0) return THA_STATUS_SUCCESS;
  if (!m->codes || !m->scales) return mx_refuse(who, "codes or scales are NULL");
  if ((reinterpret_cast<uintptr_t>(m->codes) & 31u) || !aligned16(m->scales)) return mx_refuse(who, "codes on a 32-byte and scales on a 16-byte boundary are needed");
  return THA_STATUS_SUCCESS;
}

int gemm_tc_init(int** flag_out);
int mx_error_flag(int** flag) {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;   // allocated by a device's first call, which a capture allows in this mode
  THA_CUDA_OK(cudaThreadExchangeStreamCaptureMode(&mode));
  const int st = gemm_tc_init(flag);
  THA_CUDA_OK(cudaThreadExchangeStreamCaptureMode(&mode));
  return st;
}

namespace {

constexpr int MR_THREADS = 256;
constexpr int MR_WARPS = MR_THREADS / 32;
constexpr int MR_NORM_MOST = 512;                // threads of a row's block at most, twice that with few values each
constexpr int MR_N = 4;                           // values of a thread of the norm's at a time
constexpr int MR_V = 8;                           // values of a lane
constexpr int MR_SEG = 512;                       // values of a warp at a time

// four values as fp32, zeros (`none`) behind the first n; vec: p is on a boundary of four
__device__ __forceinline__ void mr_load(const float* p, int n, bool vec, float (&v)[MR_N], float none = 0.f) {
  if (vec && n >= MR_N) { hyb_load_vec(p, v); return; }
#pragma unroll
  for (int i = 0; i < MR_N; i++) v[i] = i < n ? p[i] : none;
}
__device__ __forceinline__ void mr_load(const __nv_bfloat16* p, int n, bool vec, float (&v)[MR_N]) {
  if (vec && n >= MR_N) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u); v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
    return;
  }
#pragma unroll
  for (int i = 0; i < MR_N; i++) v[i] = i < n ? __bfloat162float(p[i]) : 0.f;
}
__device__ __forceinline__ void mr_store(float* p, int n, bool vec, const float (&v)[MR_N]) {
  if (vec && n >= MR_N) { hyb_store_vec(p, v); return; }
#pragma unroll
  for (int i = 0; i < MR_N; i++) if (i < n) p[i] = v[i];
}
// sixteen bytes
__device__ __forceinline__ void mr_store(float* p, const float (&v)[4]) { hyb_store_vec(p, v); }
__device__ __forceinline__ void mr_store(__nv_bfloat16* p, const float (&v)[8]) {
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const unsigned*>(&t);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Four values of a lane at column `col` (a multiple of 4; zeros behind the row's end), eight lanes a block, into codes and, from every eighth lane, the block's scale.  All lanes of the warp.
template <int FMT>
__device__ __forceinline__ void mr_codes(const tha_mx_t& out, int row, int col, int padded, const float (&v)[MR_N]) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < MR_N; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(THA_FULL_MASK, top, o));
  const unsigned byte = mx_scale_byte<FMT>(top);
  const float inv = mx_inverse(byte);
  if (col >= padded) return;
  if (FMT == THA_MX_E2M1) {
    const unsigned w = mx_e2m1x2(v[0] * inv, v[1] * inv) | mx_e2m1x2(v[2] * inv, v[3] * inv) << 8;
    *reinterpret_cast<unsigned short*>(static_cast<char*>(out.codes) + (size_t)row * (padded / 2) + col / 2) = (unsigned short)(byte == 255u ? 0u : w);
  } else {
    const unsigned w = mx_e4m3x2(v[0] * inv, v[1] * inv) | mx_e4m3x2(v[2] * inv, v[3] * inv) << 16;
    *reinterpret_cast<unsigned*>(static_cast<char*>(out.codes) + (size_t)row * padded + col) = byte == 255u ? 0u : w;
  }
  if (!(threadIdx.x & 7)) out.scales[mx_scale_at(row, col / MX_TILE, padded / MX_TILE) + (col / MX_BLOCK & 3)] = (uint8_t)byte;
}
// Eight values of a lane at column `col` (a multiple of 8; zeros behind the row's end), four lanes a block, into codes and, from every fourth lane, the block's scale; top: the bits of
// the lane's largest |value|.  All lanes of the warp.
template <int FMT>
__device__ __forceinline__ void mr_codes(const tha_mx_t& out, int row, int col, int padded, unsigned top, const float (&v)[MR_V]) {
  top = max(top, __shfl_xor_sync(THA_FULL_MASK, top, 1));
  top = max(top, __shfl_xor_sync(THA_FULL_MASK, top, 2));
  const unsigned byte = mx_scale_byte<FMT>(top);
  const float inv = mx_inverse(byte);
  if (col >= padded) return;
  if (FMT == THA_MX_E2M1) {
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) w |= mx_e2m1x2(v[2 * i] * inv, v[2 * i + 1] * inv) << (8 * i);
    *reinterpret_cast<unsigned*>(static_cast<char*>(out.codes) + (size_t)row * (padded / 2) + col / 2) = byte == 255u ? 0u : w;
  } else {
    uint2 w;
    w.x = mx_e4m3x2(v[0] * inv, v[1] * inv) | mx_e4m3x2(v[2] * inv, v[3] * inv) << 16;
    w.y = mx_e4m3x2(v[4] * inv, v[5] * inv) | mx_e4m3x2(v[6] * inv, v[7] * inv) << 16;
    *reinterpret_cast<uint2*>(static_cast<char*>(out.codes) + (size_t)row * padded + col) = byte == 255u ? make_uint2(0u, 0u) : w;
  }
  if (!(threadIdx.x & 3)) out.scales[mx_scale_at(row, col / MX_TILE, padded / MX_TILE) + (col / MX_BLOCK & 3)] = (uint8_t)byte;
}
// Eight values as they lie in memory, zeros behind the first n; bf16 on a boundary: sixteen
__device__ __forceinline__ void mr_fetch(const float* p, int n, bool vec, uint4 (&q)[2]) {
  if (vec && n >= MR_V) { q[0] = *reinterpret_cast<const uint4*>(p); q[1] = *reinterpret_cast<const uint4*>(p + 4); return; }
  unsigned t[8];
#pragma unroll
  for (int i = 0; i < 8; i++) t[i] = i < n ? __float_as_uint(p[i]) : 0u;
  q[0] = make_uint4(t[0], t[1], t[2], t[3]); q[1] = make_uint4(t[4], t[5], t[6], t[7]);
}
__device__ __forceinline__ void mr_fetch(const __nv_bfloat16* p, int n, uint4 (&q)[1]) {
  const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
  unsigned t[4];
#pragma unroll
  for (int i = 0; i < 4; i++) t[i] = (2 * i < n ? h[2 * i] : 0u) | (2 * i + 1 < n ? h[2 * i + 1] : 0u) << 16;
  q[0] = make_uint4(t[0], t[1], t[2], t[3]);
}
__device__ __forceinline__ void mr_fetch(const __nv_bfloat16* p, int n, uint4 (&q)[2]) {
  uint4 h[1];
  if (n >= MR_V) q[0] = *reinterpret_cast<const uint4*>(p);
  else { mr_fetch(p, n, h); q[0] = h[0]; }
  if (n >= 2 * MR_V) q[1] = *reinterpret_cast<const uint4*>(p + MR_V);
  else { mr_fetch(p + MR_V, n - MR_V, h); q[1] = h[0]; }
}
__device__ __forceinline__ unsigned mr_values(const uint4 (&q)[2], float (&v)[MR_V]) {
  const unsigned w[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    v[i] = __uint_as_float(w[i]);
    top = max(top, w[i] & 0x7fffffffu);
  }
  return top;
}
__device__ __forceinline__ unsigned mr_values(const uint4 (&q)[1], float (&v)[MR_V]) {
  const unsigned w[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    top = __vmaxu2(top, w[i] & 0x7fff7fffu);
  }
  return max(top << 16, top & 0xffff0000u);
}
__device__ __forceinline__ unsigned mr_mul2(unsigned a, unsigned b) {   // two products of bf16
  const __nv_bfloat162 t = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const unsigned*>(&t);
}
// The same for sixteen values of bf16, two lanes a block: maxima and scaling two at a time (a power of two times a bf16 is one; what underflows has the code 0)
template <int FMT>
__device__ __forceinline__ void mr_codes(const tha_mx_t& out, int row, int col, int padded, const uint4 (&q)[2]) {
  const unsigned w[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
  top = __vmaxu2(top, __shfl_xor_sync(THA_FULL_MASK, top, 1));
  const unsigned byte = mx_scale_byte<FMT>(max(top << 16, top & 0xffff0000u));
  const unsigned inv = byte == 255u ? 0u : (254u - byte) * 0x00800080u;    // 1 / scale, twice
  if (col >= padded) return;
  unsigned c[FMT == THA_MX_E2M1 ? 2 : 4] = {};
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const unsigned y = mr_mul2(w[i], inv);
    const float a = __uint_as_float(y << 16), b = __uint_as_float(y & 0xffff0000u);
    if (FMT == THA_MX_E2M1) c[i >> 2] |= mx_e2m1x2(a, b) << (8 * (i & 3));
    else c[i >> 1] |= mx_e4m3x2(a, b) << (16 * (i & 1));
  }
#pragma unroll
  for (int i = 0; i < (FMT == THA_MX_E2M1 ? 2 : 4); i++) c[i] = byte == 255u ? 0u : c[i];
  if (FMT == THA_MX_E2M1) *reinterpret_cast<uint2*>(static_cast<char*>(out.codes) + (size_t)row * (padded / 2) + col / 2) = make_uint2(c[0], c[1]);
  else *reinterpret_cast<uint4*>(static_cast<char*>(out.codes) + (size_t)row * padded + col) = make_uint4(c[0], c[1], c[FMT == THA_MX_E2M1 ? 0 : 2], c[FMT == THA_MX_E2M1 ? 0 : 3]);
  if (!(threadIdx.x & 1)) out.scales[mx_scale_at(row, col / MX_TILE, padded / MX_TILE) + (col / MX_BLOCK & 3)] = (uint8_t)byte;
}

// A warp's way through the segments of all rows: the next one is `warps` segments further.  One division at its start (one a segment, in 64 bits, and a lane's eight values at a time: 11008 x
// 4096 values in 57 us).
struct MrWalk {
  int row, col, padded, drow, dcol;
  __device__ __forceinline__ MrWalk(int cols) {
    padded = (int)mx_padded(cols);
    const int segs = (padded + MR_SEG - 1) / MR_SEG, w = blockIdx.x * MR_WARPS + (threadIdx.x >> 5), warps = gridDim.x * MR_WARPS;
    row = w / segs; drow = warps / segs;
    col = (w - row * segs) * MR_SEG; dcol = (warps - drow * segs) * MR_SEG;
  }
  __device__ __forceinline__ void next() {
    row += drow; col += dcol;
    if (col >= padded) { col -= (padded + MR_SEG - 1) / MR_SEG * MR_SEG; row++; }
  }
};

// V values of a lane at a time.  bf16 on 16-byte boundaries: sixteen, two instructions for a pair (11008 x 4096 to 4 bits 21.2 us, eight 26.6); rows on no boundary, value by value: eight
// (4000 x 4097 16.4 us, sixteen 23.0)
template <int FMT, typename T, int V>
__global__ void __launch_bounds__(MR_THREADS) mx_quant_kernel(const T* x, long long ldx, const tha_mx_t out, bool vec) {
  hyb_pdl_enter();
  constexpr int U = MR_SEG / (32 * V), Q = V * sizeof(T) / 16;
  const int lane = (threadIdx.x & 31) * V;
  MrWalk at(out.cols);
  uint4 now[U][Q], next[U][Q];
  auto fetch = [&](uint4 (&q)[U][Q]) {
    const T* p = x + at.row * ldx + at.col + lane;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int n = out.cols - at.col - lane - u * 32 * V;
      if constexpr (sizeof(T) == 2) mr_fetch(p + u * 32 * V, n, q[u]);
      else mr_fetch(p + u * 32 * V, n, vec, q[u]);
    }
  };
  if (at.row < out.rows) fetch(now);
  while (at.row < out.rows) {
    const int row = at.row, col = at.col + lane;
    at.next();
    if (at.row < out.rows) fetch(next);           // on its way while this one is coded
#pragma unroll
    for (int u = 0; u < U; u++) {
      if constexpr (V == 16) {
        mr_codes<FMT>(out, row, col + u * 32 * V, at.padded, now[u]);
      } else {
        float v[MR_V];
        const unsigned top = mr_values(now[u], v);
        mr_codes<FMT>(out, row, col + u * 32 * V, at.padded, top, v);
      }
#pragma unroll
      for (int i = 0; i < Q; i++) now[u][i] = next[u][i];
    }
  }
}

// two codes as fp16, which holds every number of both formats
template <int FMT>
__device__ __forceinline__ float2 mr_pair(unsigned c) {
  unsigned h;
  if (FMT == THA_MX_E2M1) asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(c));
  else asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)c));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// G neighbouring values a lane (16 bytes of fp32 or bf16: a warp's stores lie side by side), MR_SEG of a row a warp
template <int FMT, typename T>
__global__ void __launch_bounds__(MR_THREADS) mx_read_kernel(const tha_mx_t m, T* x, long long ldx) {
  hyb_pdl_enter();
  constexpr int G = 16 / sizeof(T), U = MR_SEG / (32 * G);
  const int lane = (threadIdx.x & 31) * G;
  MrWalk at(m.cols);
  uint2 now[U] = {}, next[U] = {};
  unsigned scale[U] = {}, scale_next[U] = {};
  auto fetch = [&](uint2 (&c)[U], unsigned (&s)[U]) {
    const int col = at.col + lane, left = m.cols - col;
    const char* codes = static_cast<const char*>(m.codes) + (size_t)at.row * (FMT == THA_MX_E2M1 ? at.padded / 2 : at.padded) + (FMT == THA_MX_E2M1 ? col / 2 : col);
    const uint8_t* scales = m.scales + mx_scale_at(at.row, col / MX_TILE, at.padded / MX_TILE) + (col / MX_BLOCK & 3);
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (u * 32 * G >= left) continue;
      const char* p = codes + u * 32 * G / (FMT == THA_MX_E2M1 ? 2 : 1);
      if (FMT == THA_MX_E2M1 && G == 4) c[u].x = *reinterpret_cast<const unsigned short*>(p);
      else if (FMT == THA_MX_E2M1 || G == 4) c[u].x = *reinterpret_cast<const unsigned*>(p);
      else c[u] = *reinterpret_cast<const uint2*>(p);
      s[u] = scales[u * (32 * G / MX_TILE) * MX_TILE_BYTES];
    }
  };
  if (at.row < m.rows) fetch(now, scale);
  while (at.row < m.rows) {
    T* p = x + at.row * ldx + at.col + lane;
    const int left = m.cols - at.col - lane;
    at.next();
    if (at.row < m.rows) fetch(next, scale_next);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const float f = mx_scale(scale[u]);
      float v[G];
#pragma unroll
      for (int i = 0; i < G / 2; i++) {
        const float2 t = mr_pair<FMT>(FMT == THA_MX_E2M1 ? now[u].x >> (8 * i) & 0xffu : (i < 2 ? now[u].x : now[u].y) >> (16 * (i & 1)) & 0xffffu);
        v[2 * i] = t.x * f; v[2 * i + 1] = t.y * f;
      }
      const int n = left - u * 32 * G;
      if (n >= G) mr_store(p + u * 32 * G, v);
      else
#pragma unroll
        for (int i = 0; i < G; i++) if (i < n) hyb_store(p + u * 32 * G + i, v[i]);
      now[u] = next[u]; scale[u] = scale_next[u];
    }
  }
}
// rows on no boundary: one value of each block a lane, the scales of four blocks in a word
template <int FMT, typename T>
__global__ void __launch_bounds__(MR_THREADS) mx_read_lanes_kernel(const tha_mx_t m, T* x, long long ldx) {
  hyb_pdl_enter();
  constexpr int B = MR_SEG / MX_BLOCK, STEP = FMT == THA_MX_E2M1 ? MX_BLOCK / 2 : MX_BLOCK;      // blocks of a segment, bytes of a block
  const int lane = threadIdx.x & 31;
  for (MrWalk at(m.cols); at.row < m.rows; at.next()) {
    const uint8_t* codes = static_cast<const uint8_t*>(m.codes) + (size_t)at.row * (FMT == THA_MX_E2M1 ? at.padded / 2 : at.padded) + (at.col + lane) / (FMT == THA_MX_E2M1 ? 2 : 1);
    const int across = at.padded / MX_TILE, left = m.cols - at.col - lane, tiles = across - at.col / MX_TILE;
    const uint8_t* scales = m.scales + mx_scale_at(at.row, at.col / MX_TILE, across);
    unsigned c[B], s[B / 4];
#pragma unroll
    for (int u = 0; u < B; u++) c[u] = 32 * u < left ? codes[STEP * u] : 0u;
#pragma unroll
    for (int k = 0; k < B / 4; k++) s[k] = k < tiles ? *reinterpret_cast<const unsigned*>(scales + k * MX_TILE_BYTES) : 0u;
    T* p = x + at.row * ldx + at.col + lane;
#pragma unroll
    for (int u = 0; u < B; u++) {
      const float f = mx_scale(s[u >> 2] >> (8 * (u & 3)) & 0xffu);
      if (32 * u < left) hyb_store(p + 32 * u, mr_pair<FMT>(FMT == THA_MX_E2M1 ? c[u] >> (4 * (lane & 1)) & 15u : c[u]).x * f);
    }
  }
}

// A number in 64 bits as one of 32 that compares with every number of at most 23 bits as it does itself: cut off, with the last bit set where something was cut. So a code is one rounding.
__device__ __forceinline__ float mr_odd(double y) {
  if (fabs(y) >= 0x1p128) return (float)y;         // infinite in fp32
  const float f = __double2float_rz(y);
  return (double)f != y && y == y ? __uint_as_float(__float_as_uint(f) | 1u) : f;
}

// 1 / sqrt(m): two steps of Newton's from an fp32 root (1 / sqrt in fp64 holds a block up for longer than its loads)
__device__ __forceinline__ double mr_root(double m) {
  if (!(m > 0x1p-100 && m < 0x1p100)) return 1.0 / sqrt(m);
  double r = rsqrtf((float)m);
  r = r * fma(-0.5 * m * r, r, 1.5);
  return r * fma(-0.5 * m * r, r, 1.5);
}

// The norm of four values of a lane, (v r) (w_offset + w), into codes; behind the row's n values v is 0 and w -w_offset.  All lanes of the warp.
// In fp32 the norm is off by less than 2^-21 of itself (four roundings, a fifth with the scale); where scale and codes are the same for 1 - 2^-21 and 1 + 2^-21 of it, as for all but one value in
// some ten thousand, they are the norm's.  Else, or where fp32 ends, the warp takes its values in fp64.  (Every value in fp64, or in pairs of fp32 numbers: 2048 x 4096 29 and 27.5 us.)
// Where fp32 ends: r (w_offset + w) may be no number of it, or one of few bits, though the norm is an ordinary number.  Beyond its end y is infinite or NaN, and the block goes by fp64.  Below 2^-126,
// with r above 2^-60, w_offset + w is below 2^-66 and the norm, as |v| r is at most the root of 2^30 columns, below 2^-51: a code of 0 in a block whose largest value is above 2^-31.  Blocks below
// that go by fp64, but for those whose values are all 0.
template <int FMT>
__device__ __forceinline__ void mr_norm_codes(const tha_mx_t& out, int row, int col, int padded, int n, const float (&v)[MR_N], const float (&w)[MR_N], float w_offset, double r) {
  const float rf = (float)r;
  float y[MR_N];
  unsigned top = 0, some = 0;
#pragma unroll
  for (int i = 0; i < MR_N; i++) {
    y[i] = v[i] * (rf * (w_offset + w[i]));       // behind the row 0 times 0, whose code is 0 (that of 0 times less is not), or NaN: by fp64
    top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
    some |= __float_as_uint(v[i]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(THA_FULL_MASK, top, o));
  const unsigned byte = mx_scale_byte<FMT>(top);
  const float inv = mx_inverse(byte), lo = inv * (1.f - 0x1p-21f), hi = inv * (1.f + 0x1p-21f);
  unsigned c[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const float f = k ? hi : lo;
    c[k] = FMT == THA_MX_E2M1 ? mx_e2m1x2(y[0] * f, y[1] * f) | mx_e2m1x2(y[2] * f, y[3] * f) << 8 : mx_e4m3x2(y[0] * f, y[1] * f) | mx_e4m3x2(y[2] * f, y[3] * f) << 16;
  }
  // the scale changes behind a fraction of 1.5 or 1.75: sure where top is more than 8 units from that, above 2^-31 and more than 16 units from fp32's end
  const bool sure = (top | some << 1) == 0u || (c[0] == c[1] && (top - (FMT == THA_MX_E2M1 ? 0x400000u : 0x600000u) + 8u & 0x7fffffu) > 16u && top - 0x30000000u < 0x7f7ffff0u - 0x30000000u);
  if (!__all_sync(THA_FULL_MASK, sure && rf > 0x1p-60f && rf < 0x1p100f)) {
#pragma unroll
    for (int i = 0; i < MR_N; i++) y[i] = i < n ? mr_odd((double)v[i] * r * ((double)w_offset + (double)w[i])) : 0.f;
    mr_codes<FMT>(out, row, col, padded, y);
    return;
  }
  if (col >= padded) return;
  if (FMT == THA_MX_E2M1) *reinterpret_cast<unsigned short*>(static_cast<char*>(out.codes) + (size_t)row * (padded / 2) + col / 2) = (unsigned short)c[0];
  else *reinterpret_cast<unsigned*>(static_cast<char*>(out.codes) + (size_t)row * padded + col) = c[0];
  if (!(threadIdx.x & 7)) out.scales[mx_scale_at(row, col / MX_TILE, padded / MX_TILE) + (col / MX_BLOCK & 3)] = (uint8_t)byte;
}

// A block takes a row, P groups of four values a thread, kept in registers between the two passes.
template <int FMT, typename T, int P>
__global__ void __launch_bounds__(P <= 4 ? 2 * MR_NORM_MOST : MR_NORM_MOST) mx_add_norm_kernel(const float* x, const T* left, long long ldl, float* x_out, const float* w, float w_offset, float eps, double inv_cols,
                                                                   const tha_mx_t out, bool vec, bool vec_left) {
  hyb_pdl_enter();
  __shared__ double part[32];
  const int row = blockIdx.x, cols = out.cols, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int padded = (int)mx_padded(cols);
  float v[P][MR_N];
  double total = 0.0;
  auto there = [&](int i) { return min(MR_N, cols - (int)(threadIdx.x + i * blockDim.x) * MR_N); };    // values of group i, if above 0
#pragma unroll
  for (int i = 0; i < P; i++) mr_load(x + (size_t)row * cols + (threadIdx.x + i * blockDim.x) * MR_N, there(i), vec, v[i]);
  if (left) {
    float l[P][MR_N];
#pragma unroll
    for (int i = 0; i < P; i++) mr_load(left + row * ldl + (threadIdx.x + i * blockDim.x) * MR_N, there(i), vec_left, l[i]);
#pragma unroll
    for (int i = 0; i < P; i++)
#pragma unroll
      for (int j = 0; j < MR_N; j++) v[i][j] += l[i][j];
  }
#pragma unroll
  for (int i = 0; i < P; i++) {
    mr_store(x_out + (size_t)row * cols + (threadIdx.x + i * blockDim.x) * MR_N, there(i), vec, v[i]);
#pragma unroll
    for (int j = 0; j < MR_N; j++) total = fma((double)v[i][j], (double)v[i][j], total);          // values behind the row are 0
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(THA_FULL_MASK, total, o);
  if (lane == 0) part[threadIdx.x >> 5] = total;
  __syncthreads();
  total = lane < warps ? part[lane] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(THA_FULL_MASK, total, o);
  const double r = __shfl_sync(THA_FULL_MASK, mr_root(total * inv_cols + (double)eps), 0);
#pragma unroll
  for (int i = 0; i < P; i++) {
    const int col = (int)(threadIdx.x + i * blockDim.x) * MR_N, n = there(i);
    if (col - lane * MR_N >= padded) break;
    float g[MR_N];
    mr_load(w + col, n, vec, g, -w_offset);
    mr_norm_codes<FMT>(out, row, col, padded, n, v[i], g, w_offset, r);
  }
}

// Wide rows, many of them, whose pitches are multiples of 16 bytes: persistent blocks, rows of x and left on their way into a ring in shared memory by bulk copies while others are worked on.
// A thread has the same columns of every row, and the weights of these in registers.  2048 x 4096, left bf16: 25 us, 3.7 TB/s; bound by its instructions, some 45 a value, and their latencies.
constexpr int MR_RING_MOST = 6;                   // stages
template <int FMT, typename T, int P>
__global__ void __launch_bounds__(MR_NORM_MOST, P <= 2 ? 2 : 1)
mx_add_norm_ring_kernel(const float* x, const T* left, long long ldl, float* x_out, const float* w, float w_offset, float eps, double inv_cols, const tha_mx_t out, int stages, int* error_flag) {
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ double part[2][MR_NORM_MOST / 32];
  __shared__ uint64_t full[MR_RING_MOST];
  __shared__ int abort_flag;
  const int cols = out.cols, lane = threadIdx.x & 31, warps = blockDim.x >> 5, padded = (int)mx_padded(cols);
  const uint32_t x_bytes = (uint32_t)cols * 4u, l_bytes = left ? (uint32_t)(cols * sizeof(T)) : 0u;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; s++) tc_mbar_init(&full[s], 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  hyb_pdl_enter();
  int asked = 0;
  auto ask = [&](int s, long long row) {
    asked++;
    unsigned char* at = ring + (size_t)s * (x_bytes + l_bytes);
    tc_mbar_expect_tx(&full[s], x_bytes + l_bytes);
    tc_bulk(at, x + row * cols, x_bytes, &full[s]);
    if (l_bytes) tc_bulk(at + x_bytes, left + row * ldl, l_bytes, &full[s]);
  };
  if (threadIdx.x == 0)
    for (int s = 0; s < stages && blockIdx.x + (long long)s * gridDim.x < out.rows; s++) ask(s, blockIdx.x + (long long)s * gridDim.x);
  float g[P][MR_N];
  auto col_of = [&](int i) { return (int)(threadIdx.x + i * blockDim.x) * MR_N; };                 // cols is a multiple of 4
#pragma unroll
  for (int i = 0; i < P; i++) mr_load(w + col_of(i), cols - col_of(i), true, g[i], -w_offset);
  int n = 0;
  bool ok = true;                                 // a thread that has given up a wait waits and reads no more: its values are NaN from then on and, through the sums, its rows' codes
  for (long long row = blockIdx.x; row < out.rows; row += gridDim.x, n++) {
    const int s = n % stages;
    ok = ok && tc_mbar_wait(&full[s], (unsigned)(n / stages) & 1u, &abort_flag);
    const float none = ok ? 0.f : __uint_as_float(0x7fc00000u);
    const unsigned char* at = ring + (size_t)s * (x_bytes + l_bytes);
    float v[P][MR_N];
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < P; i++) {
      const int col = col_of(i);
      mr_load(reinterpret_cast<const float*>(at) + col, ok ? cols - col : 0, true, v[i], none);
      if (l_bytes) {
        float l[MR_N];
        mr_load(reinterpret_cast<const T*>(at + x_bytes) + col, ok ? cols - col : 0, true, l);
#pragma unroll
        for (int j = 0; j < MR_N; j++) v[i][j] += l[j];
      }
#pragma unroll
      for (int j = 0; j < MR_N; j++) total = fma((double)v[i][j], (double)v[i][j], total);        // values behind the row are 0
    }
    double* p = part[n & 1];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(THA_FULL_MASK, total, o);
    if (lane == 0) p[threadIdx.x >> 5] = total;
    __syncthreads();                              // and every thread has its values out of the ring
    total = lane < warps ? p[lane] : 0.0;
#pragma unroll
    for (int o = MR_NORM_MOST / 64; o > 0; o >>= 1) total += __shfl_xor_sync(THA_FULL_MASK, total, o);
    if (threadIdx.x == 0 && ok && row + (long long)stages * gridDim.x < out.rows) ask(s, row + (long long)stages * gridDim.x);
#pragma unroll
    for (int i = 0; i < P; i++) mr_store(x_out + (size_t)row * cols + col_of(i), cols - col_of(i), true, v[i]);
    const double r = __shfl_sync(THA_FULL_MASK, mr_root(total * inv_cols + (double)eps), 0);
#pragma unroll
    for (int i = 0; i < P; i++) {
      const int col = col_of(i);
      if (col - lane * MR_N >= padded) break;
      mr_norm_codes<FMT>(out, (int)row, col, padded, cols - col, v[i], g[i], w_offset, r);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && abort_flag) {
    tc_drain(full, stages, asked);
    *((volatile int*)error_flag) = 1;
  }
}

// rows of any width: read again where the norm is taken, in fp64
template <int FMT, typename T>
__global__ void __launch_bounds__(MR_THREADS) mx_add_norm_wide_kernel(const float* x, const T* left, long long ldl, float* x_out, const float* w, float w_offset, float eps, double inv_cols,
                                                                 const tha_mx_t out, bool vec, bool vec_left) {
  hyb_pdl_enter();
  __shared__ double part[MR_WARPS];
  const int row = blockIdx.x, cols = out.cols;
  const int padded = (int)mx_padded(cols);
  double sum = 0.0;
  for (int col = threadIdx.x * MR_N; col < cols; col += MR_THREADS * MR_N) {
    const int n = min(MR_N, cols - col);
    float v[MR_N], l[MR_N];
    mr_load(x + (size_t)row * cols + col, n, vec, v);
    if (left) {
      mr_load(left + row * ldl + col, n, vec_left, l);
#pragma unroll
      for (int i = 0; i < MR_N; i++) v[i] += l[i];
    }
    mr_store(x_out + (size_t)row * cols + col, n, vec, v);
#pragma unroll
    for (int i = 0; i < MR_N; i++) sum = fma((double)v[i], (double)v[i], sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(THA_FULL_MASK, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int i = 0; i < MR_WARPS; i++) sum += part[i];
  const double r = 1.0 / sqrt(sum * inv_cols + (double)eps);
  for (int col0 = (threadIdx.x >> 5) * 32 * MR_N; col0 < padded; col0 += MR_THREADS * MR_N) {
    const int col = col0 + (threadIdx.x & 31) * MR_N, n = max(0, min(MR_N, cols - col));
    float v[MR_N], g[MR_N];
    mr_load(x_out + (size_t)row * cols + col, n, vec, v);
    mr_load(w + col, n, vec, g);
#pragma unroll
    for (int i = 0; i < MR_N; i++) v[i] = i < n ? mr_odd((double)v[i] * r * ((double)w_offset + (double)g[i])) : 0.f;
    mr_codes<FMT>(out, row, col, padded, v);
  }
}

bool mr_aligned(const void* p, long long ld, size_t size) { return aligned16(p) && (ld * (long long)size) % 16 == 0; }

// blocks for `rows` rows of `padded` values, a warp a segment: at most eight an SM, whose warps go on to further segments
unsigned mr_blocks(long long rows, long long padded) {
  return (unsigned)min((long long)sm_budget() * 8, ((padded + MR_SEG - 1) / MR_SEG * rows + MR_WARPS - 1) / MR_WARPS);
}
template <int FMT, typename T>
int quant_form(cudaStream_t s, const T* x, long long ldx, const tha_mx_t* out) {
  const bool vec = mr_aligned(x, out->rows > 1 ? ldx : 0, sizeof(T));
  auto k = sizeof(T) == 2 && vec ? mx_quant_kernel<FMT, T, sizeof(T) == 2 ? 16 : 8> : mx_quant_kernel<FMT, T, 8>;
  THA_CUDA_OK(launch(k, dim3(mr_blocks(out->rows, mx_padded(out->cols))), dim3(MR_THREADS), 0, s, pdl_enabled() != 0, x, ldx, *out, vec));
  return THA_STATUS_SUCCESS;
}
template <int FMT, typename T>
int read_form(cudaStream_t s, const tha_mx_t* m, T* x, long long ldx) {
  const bool vec = mr_aligned(x, m->rows > 1 ? ldx : 0, sizeof(T));
  THA_CUDA_OK(launch(vec ? mx_read_kernel<FMT, T> : mx_read_lanes_kernel<FMT, T>, dim3(mr_blocks(m->rows, mx_padded(m->cols))), dim3(MR_THREADS), 0, s, pdl_enabled() != 0, *m, x, ldx));
  return THA_STATUS_SUCCESS;
}
template <int FMT, typename T, int P>
int ring_form(cudaStream_t s, const float* x, const T* left, long long ldl, float* x_out, const float* w, float w_offset, float eps, const tha_mx_t* out, int threads, int stages, size_t stage) {
  int* flag = nullptr;
  THA_TRY_RC(mx_error_flag(&flag));
  auto k = mx_add_norm_ring_kernel<FMT, T, P>;
  static std::atomic<unsigned long long> asked{0};
  THA_TRY_RC(mx_room(k, 212 * 1024, &asked));
  const int blocks = sm_budget() * (P <= 2 && 2 * (stages * stage + 2048) <= 224 * 1024 ? 2 : 1);
  THA_CUDA_OK(launch(k, dim3(min(blocks, out->rows)), dim3(threads), stages * stage, s, pdl_enabled() != 0, x, left, ldl, x_out, w, w_offset, eps, 1.0 / out->cols, *out, stages, flag));
  return THA_STATUS_SUCCESS;
}
// The ring for wide rows that are many and fit it twice; else a block a row.  us, a block a row / ring: 2048 x 4096 with bf16 28.7 / 25.1, fp32 23.9 / 25.0; 1000 x 8192 bf16 42 / 26;
// 1000 x 11008 bf16 58 / 35; 300 x 11008 fp32 18.9 / 16.9; 8000 x 2048 bf16 42 / 53; 4000 x 1024 fp32 13.0 / 19.7.
// Threads of a row's block: few rows are done the sooner the more there are (1 x 4096 with 128, 256, 512, 1024: 6.6, 4.1, 2.9, 2.6; 64 x 11008 with 256, 512, 1024: 15.6, 9.1, 6.7), many fill the
// SMs with 256 (2000 x 2048 fp32 13.6, 12.3, 13.5 with 128, 256, 512).
template <int FMT, typename T>
int add_norm_form(cudaStream_t s, const float* x, const T* left, long long ldl, float* x_out, const float* w, float w_offset, float eps, const tha_mx_t* out) {
  const bool vec = mr_aligned(x, out->rows > 1 ? out->cols : 0, 4) && aligned16(x_out) && aligned16(w), vec_left = mr_aligned(left, out->rows > 1 ? ldl : 0, sizeof(T));
  const int need = ceil_div(out->cols, MR_N * 32) * 32;                                                       // a thread for four values
  const size_t stage = (size_t)out->cols * (4 + (left ? sizeof(T) : 0));
  if (vec && vec_left && (out->cols * sizeof(T)) % 16 == 0 && out->rows >= 2 * sm_budget() && need >= 1024 && need <= 6 * MR_NORM_MOST && 2 * stage <= 208 * 1024) {
    const int threads = MR_NORM_MOST, p = ceil_div(need, threads);
    const int stages = (int)min((size_t)MR_RING_MOST, (p <= 2 && 2 * stage <= 104 * 1024 ? 104 * 1024 : 208 * 1024) / stage);
    if (p <= 2) return ring_form<FMT, T, 2>(s, x, left, ldl, x_out, w, w_offset, eps, out, threads, stages, stage);
    if (p <= 4) return ring_form<FMT, T, 4>(s, x, left, ldl, x_out, w, w_offset, eps, out, threads, stages, stage);
    return ring_form<FMT, T, 6>(s, x, left, ldl, x_out, w, w_offset, eps, out, threads, stages, stage);
  }
  const int threads = min(need, out->rows > 4 * sm_budget() && need <= 1024 ? 256 : need <= 8 * MR_NORM_MOST ? 2 * MR_NORM_MOST : MR_NORM_MOST), p = ceil_div(need, threads);
  auto k = p <= 1 ? mx_add_norm_kernel<FMT, T, 1> : p <= 2 ? mx_add_norm_kernel<FMT, T, 2> : p <= 4 ? mx_add_norm_kernel<FMT, T, 4>
           : p <= 16 ? mx_add_norm_kernel<FMT, T, 16> : mx_add_norm_wide_kernel<FMT, T>;
  THA_CUDA_OK(launch(k, dim3(out->rows), dim3(p <= 16 ? threads : MR_THREADS), 0, s, pdl_enabled() != 0, x, left, ldl, x_out, w, w_offset, eps, 1.0 / out->cols, *out, vec, vec_left));
  return THA_STATUS_SUCCESS;
}

}  // namespace
}  // namespace tha

using namespace tha;

extern "C" size_t tha_hyb_mx_codes_bytes(int format, int rows, int cols) {
  if ((format != THA_MX_E2M1 && format != THA_MX_E4M3) || rows < 1 || rows > MX_MOST || cols < 1 || cols > MX_MOST) return 0;
  return (size_t)rows * mx_pitch(format, cols);
}
extern "C" size_t tha_hyb_mx_scales_bytes(int rows, int cols) {
  if (rows < 1 || rows > MX_MOST || cols < 1 || cols > MX_MOST) return 0;
  return (((size_t)rows + MX_TILE - 1) / MX_TILE) * (mx_padded(cols) / MX_TILE) * MX_TILE_BYTES;
}

extern "C" int tha_hyb_mx_quant(void* stream, int dtype, const void* x, long long ldx, const tha_mx_t* out) {
  const char* who = "tha_hyb_mx_quant";
  THA_TRY_RC(mx_check(out, who));
  if (dtype != THA_DT_F32 && dtype != THA_DT_BF16) return mx_refuse(who, "unknown dtype");
  if (out->rows == 0) return THA_STATUS_SUCCESS;
  if (!x) return mx_refuse(who, "x is NULL");
  if (ldx < out->cols && out->rows > 1) return mx_refuse(who, "a row pitch below the row");
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == THA_DT_F32) return out->format == THA_MX_E2M1 ? quant_form<THA_MX_E2M1>(s, (const float*)x, ldx, out) : quant_form<THA_MX_E4M3>(s, (const float*)x, ldx, out);
  return out->format == THA_MX_E2M1 ? quant_form<THA_MX_E2M1>(s, (const __nv_bfloat16*)x, ldx, out) : quant_form<THA_MX_E4M3>(s, (const __nv_bfloat16*)x, ldx, out);
}

extern "C" int tha_hyb_mx_read(void* stream, int dtype, const tha_mx_t* m, void* x, long long ldx) {
  const char* who = "tha_hyb_mx_read";
  THA_TRY_RC(mx_check(m, who));
  if (dtype != THA_DT_F32 && dtype != THA_DT_BF16) return mx_refuse(who, "unknown dtype");
  if (m->rows == 0) return THA_STATUS_SUCCESS;
  if (!x) return mx_refuse(who, "x is NULL");
  if (ldx < m->cols && m->rows > 1) return mx_refuse(who, "a row pitch below the row");
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == THA_DT_F32) return m->format == THA_MX_E2M1 ? read_form<THA_MX_E2M1>(s, m, (float*)x, ldx) : read_form<THA_MX_E4M3>(s, m, (float*)x, ldx);
  return m->format == THA_MX_E2M1 ? read_form<THA_MX_E2M1>(s, m, (__nv_bfloat16*)x, ldx) : read_form<THA_MX_E4M3>(s, m, (__nv_bfloat16*)x, ldx);
}

extern "C" int tha_hyb_mx_add_norm(void* stream, int dtype, const float* x, const void* left, long long ldl, float* x_out, const float* w, float w_offset, float eps, const tha_mx_t* out) {
  const char* who = "tha_hyb_mx_add_norm";
  THA_TRY_RC(mx_check(out, who));
  if (dtype != THA_DT_F32 && dtype != THA_DT_BF16) return mx_refuse(who, "unknown dtype");
  if (out->rows == 0) return THA_STATUS_SUCCESS;
  if (!x || !x_out || !w) return mx_refuse(who, "x, x_out or w is NULL");
  if (left && ldl < out->cols && out->rows > 1) return mx_refuse(who, "a row pitch below the row");
  if (!(eps >= 0.f)) return mx_refuse(who, "eps is below 0");       // a root above 1 / rms, which the norm's way through fp32 counts on not to meet
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == THA_DT_F32)
    return out->format == THA_MX_E2M1 ? add_norm_form<THA_MX_E2M1>(s, x, (const float*)left, ldl, x_out, w, w_offset, eps, out)
                                      : add_norm_form<THA_MX_E4M3>(s, x, (const float*)left, ldl, x_out, w, w_offset, eps, out);
  return out->format == THA_MX_E2M1 ? add_norm_form<THA_MX_E2M1>(s, x, (const __nv_bfloat16*)left, ldl, x_out, w, w_offset, eps, out)
                                    : add_norm_form<THA_MX_E4M3>(s, x, (const __nv_bfloat16*)left, ldl, x_out, w, w_offset, eps, out);
}
