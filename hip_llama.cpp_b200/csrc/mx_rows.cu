// Rows into microscaled numbers and back, and the norm that ends in them (tha_mx_t).
//   mx_quant_kernel     a warp takes 256 consecutive values of a row: a lane eight of them, four lanes a block, whose largest |value| is a maximum of bit patterns
//   mx_read_kernel      eight values a thread
//   mx_add_norm_kernel  a block of threads takes a row: x + left, the square sum, the norm, its codes
// All three are bound by memory: a value is read and written once.
#include <string.h>

#include "mx.cuh"

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
  if (m->rows < 0 || m->cols < 1 || m->cols > 0x7fffff00) return mx_refuse(who, "a matrix has at least one column");
  if (m->rows == 0) return THA_STATUS_SUCCESS;
  if (!m->codes || !m->scales) return mx_refuse(who, "codes or scales are NULL");
  if ((reinterpret_cast<uintptr_t>(m->codes) & 31u) || !aligned16(m->scales)) return mx_refuse(who, "codes on a 32-byte and scales on a 16-byte boundary are needed");
  return THA_STATUS_SUCCESS;
}

namespace {

constexpr int MR_THREADS = 256;
constexpr int MR_WARPS = MR_THREADS / 32;
constexpr int MR_V = 8;                           // values of a lane
constexpr int MR_SEG = 32 * MR_V;                 // values of a warp

// `n` values at p as fp32, zeros behind them; vec: p is 16-byte aligned
__device__ __forceinline__ void mr_load(const float* p, int n, bool vec, float (&v)[MR_V]) {
  if (vec && n >= MR_V) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < MR_V; i++) v[i] = i < n ? p[i] : 0.f;
}
__device__ __forceinline__ void mr_load(const __nv_bfloat16* p, int n, bool vec, float (&v)[MR_V]) {
  if (vec && n >= MR_V) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    return;
  }
#pragma unroll
  for (int i = 0; i < MR_V; i++) v[i] = i < n ? __bfloat162float(p[i]) : 0.f;
}
__device__ __forceinline__ void mr_store(float* p, int n, bool vec, const float (&v)[MR_V]) {
  if (vec && n >= MR_V) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
#pragma unroll
  for (int i = 0; i < MR_V; i++) if (i < n) p[i] = v[i];
}
__device__ __forceinline__ void mr_store(__nv_bfloat16* p, int n, bool vec, const float (&v)[MR_V]) {
  if (vec && n >= MR_V) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const unsigned*>(&t);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < MR_V; i++) if (i < n) p[i] = __float2bfloat16_rn(v[i]);
}

// The whole warp's 256 values from column `col0` of a row on, a lane's eight in v (zeros behind the row's end), into codes and scales.
template <int FMT>
__device__ __forceinline__ void mr_codes(const tha_mx_t& out, int row, long long col0, long long padded, const float (&v)[MR_V]) {
  const int lane = threadIdx.x & 31;
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < MR_V; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(THA_FULL_MASK, top, 1));
  top = max(top, __shfl_xor_sync(THA_FULL_MASK, top, 2));
  const unsigned byte = mx_scale_byte<FMT>(top);
  const float inv = mx_inverse(byte);
  float y[MR_V];
#pragma unroll
  for (int i = 0; i < MR_V; i++) y[i] = byte == 255u ? 0.f : v[i] * inv;
  const long long col = col0 + lane * MR_V;
  if (col < padded) {
    if (FMT == THA_MX_E2M1) {
      unsigned w = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) w |= mx_e2m1x2(y[2 * i], y[2 * i + 1]) << (8 * i);
      *reinterpret_cast<unsigned*>(static_cast<char*>(out.codes) + (size_t)row * (padded / 2) + col / 2) = w;
    } else {
      uint2 w;
      w.x = mx_e4m3x2(y[0], y[1]) | mx_e4m3x2(y[2], y[3]) << 16;
      w.y = mx_e4m3x2(y[4], y[5]) | mx_e4m3x2(y[6], y[7]) << 16;
      *reinterpret_cast<uint2*>(static_cast<char*>(out.codes) + (size_t)row * padded + col) = w;
    }
  }
  unsigned four = 0;                              // lanes 0 and 1: the scales of four blocks each
#pragma unroll
  for (int q = 0; q < 4; q++) four |= __shfl_sync(THA_FULL_MASK, byte, (16 * lane + 4 * q) & 31) << (8 * q);
  const int across = (int)(padded / MX_TILE), t = (int)(col0 / MX_TILE) + lane;
  if (lane < 2 && t < across) *reinterpret_cast<unsigned*>(out.scales + mx_scale_at(row, t, across)) = four;
}

template <int FMT, typename T>
__global__ void __launch_bounds__(MR_THREADS) mx_quant_kernel(const T* x, long long ldx, const tha_mx_t out, bool vec) {
  const long long padded = mx_padded(out.cols), segs = (padded + MR_SEG - 1) / MR_SEG;
  const long long w = (long long)blockIdx.x * MR_WARPS + (threadIdx.x >> 5);
  if (w >= segs * out.rows) return;
  const int row = (int)(w / segs);
  const long long col0 = (w - row * segs) * MR_SEG, col = col0 + (threadIdx.x & 31) * MR_V;
  float v[MR_V];
  mr_load(x + row * ldx + col, (int)min((long long)MR_V, max(0ll, out.cols - col)), vec, v);
  mr_codes<FMT>(out, row, col0, padded, v);
}

template <int FMT, typename T>
__global__ void __launch_bounds__(MR_THREADS) mx_read_kernel(const tha_mx_t m, T* x, long long ldx, bool vec) {
  const long long padded = mx_padded(m.cols), each = (m.cols + MR_V - 1) / MR_V;
  const long long w = (long long)blockIdx.x * MR_THREADS + threadIdx.x;
  if (w >= each * m.rows) return;
  const int row = (int)(w / each);
  const long long col = (w - row * each) * MR_V;
  const int across = (int)(padded / MX_TILE);
  const float scale = mx_scale(m.scales[mx_scale_at(row, (int)(col / MX_TILE), across) + (col / MX_BLOCK & 3)]);
  float v[MR_V];
  if (FMT == THA_MX_E2M1) {
    const unsigned c = *reinterpret_cast<const unsigned*>(static_cast<const char*>(m.codes) + (size_t)row * (padded / 2) + col / 2);
#pragma unroll
    for (int i = 0; i < MR_V; i++) {
      // 1 bit of mantissa, exponents from 2^0 on, below them steps of a half
      const unsigned k = c >> (4 * i) & 7u;
      const float a = k < 2u ? 0.5f * k : __uint_as_float((k >> 1) + 126u << 23 | (k & 1u) << 22);
      v[i] = (c >> (4 * i) & 8u ? -a : a) * scale;
    }
  } else {
    const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const char*>(m.codes) + (size_t)row * padded + col);
#pragma unroll
    for (int i = 0; i < MR_V; i++) {
      // 3 bits of mantissa, exponents from 2^-6 on, below them steps of 2^-9; all exponent and mantissa bits set: NaN
      const unsigned b = (i < 4 ? c.x : c.y) >> (8 * (i & 3)), k = b & 0x7fu;
      const float a = k < 8u ? k * 0.001953125f : k == 0x7fu ? __uint_as_float(0x7fc00000u) : __uint_as_float((k >> 3) + 120u << 23 | (k & 7u) << 20);
      v[i] = (b & 0x80u ? -a : a) * scale;
    }
  }
  mr_store(x + row * ldx + col, (int)min((long long)MR_V, m.cols - col), vec, v);
}

// A number in 64 bits as one of 32 that compares with every number of at most 23 bits as it does itself: cut off, with the last bit set where something was cut. So a code is one rounding.
__device__ __forceinline__ float mr_odd(double y) {
  const float f = __double2float_rz(y);
  return (double)f != y && y == y ? __uint_as_float(__float_as_uint(f) | 1u) : f;
}

template <int FMT, typename T>
__global__ void __launch_bounds__(MR_THREADS) mx_add_norm_kernel(const float* x, const T* left, long long ldl, float* x_out, const float* w, float w_offset, float eps, const tha_mx_t out,
                                                                 bool vec, bool vec_left) {
  __shared__ double part[MR_WARPS];
  const int row = blockIdx.x, cols = out.cols;
  const long long padded = mx_padded(cols);
  double sum = 0.0;
  for (long long col = threadIdx.x * MR_V; col < cols; col += MR_THREADS * MR_V) {
    const int n = (int)min((long long)MR_V, cols - col);
    float v[MR_V], l[MR_V];
    mr_load(x + (size_t)row * cols + col, n, vec, v);
    if (left) {
      mr_load(left + row * ldl + col, n, vec_left, l);
#pragma unroll
      for (int i = 0; i < MR_V; i++) v[i] += l[i];
    }
    mr_store(x_out + (size_t)row * cols + col, n, vec, v);
#pragma unroll
    for (int i = 0; i < MR_V; i++) sum = fma((double)v[i], (double)v[i], sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(THA_FULL_MASK, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int i = 0; i < MR_WARPS; i++) sum += part[i];
  const double r = 1.0 / sqrt(sum / cols + (double)eps);
  for (long long col0 = (threadIdx.x >> 5) * MR_SEG; col0 < padded; col0 += MR_THREADS * MR_V) {
    const long long col = col0 + (threadIdx.x & 31) * MR_V;
    const int n = (int)min((long long)MR_V, max(0ll, cols - col));
    float v[MR_V], g[MR_V];
    mr_load(x_out + (size_t)row * cols + col, n, vec, v);
    mr_load(w + col, n, vec, g);
#pragma unroll
    for (int i = 0; i < MR_V; i++) v[i] = i < n ? mr_odd((double)v[i] * r * ((double)w_offset + (double)g[i])) : 0.f;
    mr_codes<FMT>(out, row, col0, padded, v);
  }
}

bool mr_aligned(const void* p, long long ld, size_t size) { return aligned16(p) && (ld * (long long)size) % 16 == 0; }

template <int FMT, typename T>
int quant_form(cudaStream_t s, const T* x, long long ldx, const tha_mx_t* out) {
  const long long warps = (mx_padded(out->cols) + MR_SEG - 1) / MR_SEG * out->rows, blocks = (warps + MR_WARPS - 1) / MR_WARPS;
  if (blocks > 0x7fffffff) return mx_refuse("tha_hyb_mx_quant", "too many values for one call");
  THA_CUDA_OK(launch(mx_quant_kernel<FMT, T>, dim3((unsigned)blocks), dim3(MR_THREADS), 0, s, false, x, ldx, *out, mr_aligned(x, ldx, sizeof(T))));
  return THA_STATUS_SUCCESS;
}
template <int FMT, typename T>
int read_form(cudaStream_t s, const tha_mx_t* m, T* x, long long ldx) {
  const long long threads = ((long long)m->cols + MR_V - 1) / MR_V * m->rows, blocks = (threads + MR_THREADS - 1) / MR_THREADS;
  if (blocks > 0x7fffffff) return mx_refuse("tha_hyb_mx_read", "too many values for one call");
  THA_CUDA_OK(launch(mx_read_kernel<FMT, T>, dim3((unsigned)blocks), dim3(MR_THREADS), 0, s, false, *m, x, ldx, mr_aligned(x, ldx, sizeof(T))));
  return THA_STATUS_SUCCESS;
}
template <int FMT, typename T>
int add_norm_form(cudaStream_t s, const float* x, const T* left, long long ldl, float* x_out, const float* w, float w_offset, float eps, const tha_mx_t* out) {
  const bool vec = mr_aligned(x, out->cols, 4) && aligned16(x_out) && aligned16(w);
  THA_CUDA_OK(launch(mx_add_norm_kernel<FMT, T>, dim3(out->rows), dim3(MR_THREADS), 0, s, false, x, left, ldl, x_out, w, w_offset, eps, *out, vec,
                     mr_aligned(left, ldl, sizeof(T))));
  return THA_STATUS_SUCCESS;
}

}  // namespace
}  // namespace tha

using namespace tha;

extern "C" size_t tha_hyb_mx_codes_bytes(int format, int rows, int cols) {
  if ((format != THA_MX_E2M1 && format != THA_MX_E4M3) || rows < 1 || cols < 1 || cols > 0x7fffff00) return 0;
  return (size_t)rows * mx_pitch(format, cols);
}
extern "C" size_t tha_hyb_mx_scales_bytes(int rows, int cols) {
  if (rows < 1 || cols < 1 || cols > 0x7fffff00) return 0;
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
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == THA_DT_F32)
    return out->format == THA_MX_E2M1 ? add_norm_form<THA_MX_E2M1>(s, x, (const float*)left, ldl, x_out, w, w_offset, eps, out)
                                      : add_norm_form<THA_MX_E4M3>(s, x, (const float*)left, ldl, x_out, w, w_offset, eps, out);
  return out->format == THA_MX_E2M1 ? add_norm_form<THA_MX_E2M1>(s, x, (const __nv_bfloat16*)left, ldl, x_out, w, w_offset, eps, out)
                                    : add_norm_form<THA_MX_E4M3>(s, x, (const __nv_bfloat16*)left, ldl, x_out, w, w_offset, eps, out);
}
