// Rows into the cache in 8 bits and back (include/tha_hybrid.h, tha_kv8_t).
//
// A code is the format's number nearest to the real quotient x / scale.  The usual way is y = x * (1 / scale), off by 2^-22 of itself at most, and rounding
// y; only where y is that near to a border between two numbers the quotient itself is asked for, rounded towards zero with its last bit set where it is not exact ("round to
// odd"), from which a second rounding to fewer bits gives what one rounding of the real quotient gives.
#include <stdio.h>

#include "kv8.cuh"

namespace tha {

int kv8_refuse(const char* who, const char* why) {
  char text[256];
  snprintf(text, sizeof text, "%s: %s", who, why);
  set_last_error(text, cudaErrorInvalidValue);
  return THA_STATUS_INVALID_ARG;
}
int kv8_check(const tha_rows_t* rows, const tha_kv8_t* kv, int cache_layer, const char* who) {
  if (!rows->pos || !rows->row_seq || !rows->seq_first || !rows->seq_slot || rows->n_seqs < 1) return kv8_refuse(who, "rows without their arrays");
  if (rows->max_seq_rows < 1 || rows->max_seq_rows > rows->n_rows || rows->n_seqs > rows->n_rows) return kv8_refuse(who, "a sequence of the step has at least one row");
  if (!kv->k_pool || !kv->v_pool || !kv->k_scale || !kv->v_scale || !kv->table) return kv8_refuse(who, "a pool, its scales or the table is NULL");
  if (kv->format != THA_KV8_INT8 && kv->format != THA_KV8_E4M3) return kv8_refuse(who, "unknown format");
  if (kv->block_size < 16 || kv->block_size > 128 || (kv->block_size & (kv->block_size - 1))) return kv8_refuse(who, "blocks of 16, 32, 64 or 128 positions");
  if (kv->dim < 16 || kv->dim > 128 || kv->dim % 16 || kv->vdim < 16 || kv->vdim > 128 || kv->vdim % 16) return kv8_refuse(who, "heads of 16, 32, .. 128 channels");
  if (kv->kv_heads < 1 || kv->kv_heads > 65535 || kv->n_cache_layers < 1 || kv->n_blocks < 1 || kv->table_stride < 1) return kv8_refuse(who, "an extent of the cache is below 1");
  if (cache_layer < 0 || cache_layer >= kv->n_cache_layers) return kv8_refuse(who, "no such cache layer");
  if (rows->max_pos >= (long long)kv->table_stride * kv->block_size) return kv8_refuse(who, "a position behind the last block of the table");
  if (!aligned16(kv->k_pool) || !aligned16(kv->v_pool)) return kv8_refuse(who, "pools on 16-byte boundaries");
  return THA_STATUS_SUCCESS;
}

// x / s, s > 0 and |x| finite: towards zero, the last bit set where the quotient is not exact
__device__ __forceinline__ float quotient_to_odd(float x, float s) {
  if (s < 1e-18f) { x *= 18446744073709551616.0f; s *= 18446744073709551616.0f; }   // 2^64: the remainder below stays a normal number
  const float y = __fdiv_rz(x, s);
  return fmaf(-y, s, x) != 0.f ? __uint_as_float(__float_as_uint(y) | 1u) : y;
}
template <int FMT>
__device__ __forceinline__ uint32_t kv8_encode4(float4 x, float s, float inv) {
  constexpr float MOST = FMT == THA_KV8_INT8 ? 127.f : 448.f;
  float v[4] = {x.x, x.y, x.z, x.w}, y[4];
  bool close = false;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    y[i] = v[i] * inv;
    y[i] = y[i] == y[i] ? fminf(fmaxf(y[i], -MOST), MOST) : 0.f;      // infinities, and NaN
    if (FMT == THA_KV8_INT8) {
      close |= fabsf(fabsf(y[i] - rintf(y[i])) - 0.5f) < 1e-4f;        // 127 * 2^-22 = 3e-5
    } else {
      // a border is where bit 19 begins what is cut off, from 2^-6 upwards; below, steps are 2^-9 all the way, and few values are there
      const uint32_t b = __float_as_uint(y[i]);
      close |= (fabsf(y[i]) < 0.015625f && y[i] != 0.f) || ((b & 0xFFFFFu) - 0x80000u + 16u) < 33u;
    }
  }
  if (close) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (fabsf(v[i]) < INFINITY && s > 0.f) y[i] = fminf(fmaxf(quotient_to_odd(v[i], s), -MOST), MOST);
  }
  if (FMT == THA_KV8_INT8) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) w |= ((uint32_t)__float2int_rn(y[i]) & 0xFFu) << (8 * i);
    return w;
  }
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

template <bool VEC>
__device__ __forceinline__ float4 kv8_row4(const float* p) { return VEC ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]); }
template <bool VEC>
__device__ __forceinline__ float4 kv8_row4(const __nv_bfloat16* p) {
  if (!VEC) return make_float4(__bfloat162float(p[0]), __bfloat162float(p[1]), __bfloat162float(p[2]), __bfloat162float(p[3]));
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u));
}

// Blocks that sequence s touches, but the last of several: the thread block of its first block also makes the last one, because it reads the slot's open rows and the last one
// replaces them.
__device__ __forceinline__ int kv8_units(const tha_rows_t& rows, int s, int block_size) {
  const int first = rows.seq_first[s], n = rows.seq_first[s + 1] - first;
  if (n < 1) return 0;
  const int p0 = rows.pos[first];
  if (p0 < 0) return 0;
  const int blocks = (p0 + n - 1) / block_size - p0 / block_size + 1;
  return blocks > 1 ? blocks - 1 : 1;
}

// One thread block: a block of the cache, one head, K or V; its rows in registers (N float4 a thread) between the maximum and the codes, so that they are read once.
// grid (units, kv_heads, 2)
template <typename T, int FMT, int N, bool VEC>
__global__ void __launch_bounds__(256) kv8_write_kernel(tha_rows_t rows, tha_kv8_t kv, int layer, const T* k, long long ldk, const T* v, long long ldv) {
  hyb_pdl_enter();
  constexpr float MOST = FMT == THA_KV8_INT8 ? 127.f : 448.f;
  __shared__ float red[33];
  const int B = kv.block_size, h = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const int W = is_v ? kv.vdim : kv.dim, w4 = W / 4;
  int seq = blockIdx.x, unit = 0;
  if (rows.max_seq_rows > 1) {
    const Kv8Piece pc = kv8_find(rows.n_seqs, (int)blockIdx.x, [&](int s) { return kv8_units(rows, s, B); });
    seq = pc.seq; unit = pc.at;
  }
  if (seq < 0) return;
  const int r0 = rows.seq_first[seq], n = rows.seq_first[seq + 1] - r0, slot = rows.seq_slot[seq];
  const int p0 = n > 0 ? rows.pos[r0] : -1;
  if (p0 < 0) return;
  const int p_end = p0 + n, first = p0 / B, last = (p_end - 1) / B;
  const size_t open_at = kv8_tile(kv, slot, layer, h) * (size_t)B * W;
  float* open = (is_v ? kv.v_open : kv.k_open) + open_at;
  const T* src = is_v ? v + (long long)r0 * ldv + (long long)h * W : k + (long long)r0 * ldk + (long long)h * W;
  const long long ld = is_v ? ldv : ldk;
  uint8_t* pool = static_cast<uint8_t*>(is_v ? kv.v_pool : kv.k_pool);
  float* scales = is_v ? kv.v_scale : kv.k_scale;

  auto make = [&](int b) {
    const int id = kv8_block(kv, slot, b * B);
    float4 x[N];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int e = threadIdx.x + i * blockDim.x, row = e / w4, c = 4 * (e - row * w4), t = b * B + row;
      x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < B && t < p_end) {
        if (t < p0) x[i] = *reinterpret_cast<const float4*>(open + (size_t)row * W + c);
        else x[i] = kv8_row4<VEC>(src + (long long)(t - p0) * ld + c);
      }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float m[4] = {fabsf(x[i].x), fabsf(x[i].y), fabsf(x[i].z), fabsf(x[i].w)};
#pragma unroll
      for (int j = 0; j < 4; j++) top = fmaxf(top, m[j] < INFINITY ? m[j] : 0.f);      // false for NaN too
    }
    top = block_max(top, red);
    const float s = top > 0.f ? fmaxf(__fdiv_rn(top, MOST), 1.17549435e-38f) : 0.f, inv = s > 0.f ? __fdividef(1.0f, s) : 0.f;
    const bool open_block = (b + 1) * B > p_end;
    const size_t tile = id >= 0 ? kv8_tile(kv, id, layer, h) : 0;
    if (id >= 0 && threadIdx.x == 0) scales[tile] = s;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int e = threadIdx.x + i * blockDim.x, row = e / w4, c = 4 * (e - row * w4), t = b * B + row;
      if (row >= B) continue;
      if (id >= 0) *reinterpret_cast<uint32_t*>(pool + tile * (size_t)B * W + (size_t)row * W + c) = kv8_encode4<FMT>(x[i], s, inv);
      if (open_block && t >= p0 && t < p_end) *reinterpret_cast<float4*>(open + (size_t)row * W + c) = x[i];
    }
  };
  make(first + unit);
  if (unit == 0 && last > first) {
    __syncthreads();                                       // the open rows of the first block have been read
    make(last);
  }
}

// V codes a thread: 16 bytes of result
template <typename T> struct Kv8Out;
template <> struct Kv8Out<float> {
  static constexpr int V = 4;
  template <int FMT>
  static __device__ __forceinline__ void put(float* dst, const uint8_t* src, float s) {
    const float4 x = kv8_decode4<FMT>(*reinterpret_cast<const uint32_t*>(src));
    *reinterpret_cast<float4*>(dst) = make_float4(x.x * s, x.y * s, x.z * s, x.w * s);
  }
};
template <> struct Kv8Out<__nv_bfloat16> {
  static constexpr int V = 8;
  template <int FMT>
  static __device__ __forceinline__ void put(__nv_bfloat16* dst, const uint8_t* src, float s) {
    const uint2 w = *reinterpret_cast<const uint2*>(src);
    const float4 a = kv8_decode4<FMT>(w.x), b = kv8_decode4<FMT>(w.y);
    const __nv_bfloat162 p[4] = {__floats2bfloat162_rn(a.x * s, a.y * s), __floats2bfloat162_rn(a.z * s, a.w * s), __floats2bfloat162_rn(b.x * s, b.y * s),
                                 __floats2bfloat162_rn(b.z * s, b.w * s)};
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(p);
  }
};

// grid (rows, 2): a row's heads, K or V
template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(256) kv8_read_kernel(tha_rows_t rows, tha_kv8_t kv, int layer, T* k, long long ldk, T* v, long long ldv) {
  hyb_pdl_enter();
  constexpr int V = Kv8Out<T>::V;
  const bool is_v = blockIdx.y != 0;
  T* out = is_v ? v : k;
  if (!out) return;
  const int r = blockIdx.x, W = is_v ? kv.vdim : kv.dim, wv = W / V, B = kv.block_size;
  out += (long long)r * (is_v ? ldv : ldk);
  const int t = rows.pos[r], slot = rows.seq_slot[rows.row_seq[r]];
  const int id = t >= 0 ? kv8_block(kv, slot, t) : -1;
  const size_t tile = id >= 0 ? kv8_tile(kv, id, layer, 0) : 0;
  const uint8_t* pool = static_cast<const uint8_t*>(is_v ? kv.v_pool : kv.k_pool) + (tile * B + (id >= 0 ? t % B : 0)) * W;
  const float* scales = (is_v ? kv.v_scale : kv.k_scale) + tile;
#pragma unroll 4
  for (int e = threadIdx.x; e < kv.kv_heads * wv; e += blockDim.x) {
    const int h = e / wv, c = V * (e - h * wv);
    alignas(16) T x[V] = {};
    if (id >= 0) Kv8Out<T>::template put<FMT>(x, pool + (size_t)h * B * W + c, scales[h]);
    T* dst = out + (size_t)h * W + c;
    if (VEC) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(x);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) dst[i] = x[i];
    }
  }
}

template <typename T, int FMT, bool VEC>
static int write_launch(cudaStream_t s, const tha_rows_t* rows, const tha_kv8_t* kv, int layer, const T* k, long long ldk, const T* v, long long ldv) {
  const int most = kv->block_size * (kv->dim > kv->vdim ? kv->dim : kv->vdim) / 4;       // float4 of a block and head: 64 .. 4096
  const int threads = most > 1024 ? 256 : 128, per = ceil_div(most, threads);
  const int units = rows->max_seq_rows == 1 ? rows->n_seqs : rows->n_rows / kv->block_size + rows->n_seqs;
  const dim3 grid(units, kv->kv_heads, 2);
  auto go = [&](auto kernel) -> int {
    THA_CUDA_OK(launch(kernel, grid, dim3(threads), 0, s, pdl_enabled() != 0, *rows, *kv, layer, k, ldk, v, ldv));
    return THA_STATUS_SUCCESS;
  };
  if (per <= 2) return go(kv8_write_kernel<T, FMT, 2, VEC>);
  if (per <= 4) return go(kv8_write_kernel<T, FMT, 4, VEC>);
  if (per <= 8) return go(kv8_write_kernel<T, FMT, 8, VEC>);
  return go(kv8_write_kernel<T, FMT, 16, VEC>);
}
template <typename T>
static int write_form(cudaStream_t s, const tha_rows_t* rows, const tha_kv8_t* kv, int layer, const T* k, long long ldk, const T* v, long long ldv) {
  const bool vec = ldk % 4 == 0 && ldv % 4 == 0 && ((uintptr_t)k | (uintptr_t)v) % (4 * sizeof(T)) == 0;
  if (kv->format == THA_KV8_INT8)
    return vec ? write_launch<T, THA_KV8_INT8, true>(s, rows, kv, layer, k, ldk, v, ldv) : write_launch<T, THA_KV8_INT8, false>(s, rows, kv, layer, k, ldk, v, ldv);
  return vec ? write_launch<T, THA_KV8_E4M3, true>(s, rows, kv, layer, k, ldk, v, ldv) : write_launch<T, THA_KV8_E4M3, false>(s, rows, kv, layer, k, ldk, v, ldv);
}
template <typename T>
static int read_form(cudaStream_t s, const tha_rows_t* rows, const tha_kv8_t* kv, int layer, T* k, long long ldk, T* v, long long ldv) {
  const bool vec = ((k ? ldk : 0) | (v ? ldv : 0)) % Kv8Out<T>::V == 0 && aligned16(k) && aligned16(v);
  const int most = kv->kv_heads * (kv->dim > kv->vdim ? kv->dim : kv->vdim) / Kv8Out<T>::V;
  const dim3 grid(rows->n_rows, 2), block(most > 128 ? 256 : most > 64 ? 128 : 64);
  auto go = [&](auto kernel) -> int {
    THA_CUDA_OK(launch(kernel, grid, block, 0, s, pdl_enabled() != 0, *rows, *kv, layer, k, ldk, v, ldv));
    return THA_STATUS_SUCCESS;
  };
  if (kv->format == THA_KV8_INT8) return vec ? go(kv8_read_kernel<T, THA_KV8_INT8, true>) : go(kv8_read_kernel<T, THA_KV8_INT8, false>);
  return vec ? go(kv8_read_kernel<T, THA_KV8_E4M3, true>) : go(kv8_read_kernel<T, THA_KV8_E4M3, false>);
}

}  // namespace tha

using namespace tha;

extern "C" int tha_hyb_kv8_write(void* stream, int dtype, const tha_rows_t* rows, const tha_kv8_t* kv, int cache_layer, const void* k, long long ldk, const void* v,
                                 long long ldv) {
  if (rows->n_rows < 1) return THA_STATUS_SUCCESS;
  THA_TRY_RC(kv8_check(rows, kv, cache_layer, "tha_hyb_kv8_write"));
  if (!k || !v) return kv8_refuse("tha_hyb_kv8_write", "k or v is NULL");
  if (!kv->k_open || !kv->v_open || !aligned16(kv->k_open) || !aligned16(kv->v_open)) return kv8_refuse("tha_hyb_kv8_write", "open rows on 16-byte boundaries are needed");
  if (ldk < (long long)kv->kv_heads * kv->dim || ldv < (long long)kv->kv_heads * kv->vdim) return kv8_refuse("tha_hyb_kv8_write", "a row pitch below the row");
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == THA_DT_BF16) return write_form(s, rows, kv, cache_layer, (const __nv_bfloat16*)k, ldk, (const __nv_bfloat16*)v, ldv);
  if (dtype == THA_DT_F32) return write_form(s, rows, kv, cache_layer, (const float*)k, ldk, (const float*)v, ldv);
  return kv8_refuse("tha_hyb_kv8_write", "unknown dtype");
}

extern "C" int tha_hyb_kv8_read(void* stream, int dtype, const tha_rows_t* rows, const tha_kv8_t* kv, int cache_layer, void* k_out, long long ldk, void* v_out,
                                long long ldv) {
  if (rows->n_rows < 1 || (!k_out && !v_out)) return THA_STATUS_SUCCESS;
  THA_TRY_RC(kv8_check(rows, kv, cache_layer, "tha_hyb_kv8_read"));
  if ((k_out && ldk < (long long)kv->kv_heads * kv->dim) || (v_out && ldv < (long long)kv->kv_heads * kv->vdim))
    return kv8_refuse("tha_hyb_kv8_read", "a row pitch below the row");
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == THA_DT_BF16) return read_form(s, rows, kv, cache_layer, (__nv_bfloat16*)k_out, ldk, (__nv_bfloat16*)v_out, ldv);
  if (dtype == THA_DT_F32) return read_form(s, rows, kv, cache_layer, (float*)k_out, ldk, (float*)v_out, ldv);
  return kv8_refuse("tha_hyb_kv8_read", "unknown dtype");
}
