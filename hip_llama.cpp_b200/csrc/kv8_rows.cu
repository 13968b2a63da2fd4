// Rows into the cache in 8 bits and back (include/tha_hybrid.h, tha_kv8_t).
//
// A code is the format's number nearest to the real quotient x / scale.  The usual way is y = x * (1 / scale), off by 2^-22 of itself at most, and rounding
// y; only where y is that near to a border between two numbers the quotient itself is asked for, rounded towards zero with its last bit set where it is not exact ("round to
// odd"), from which a second rounding to fewer bits gives what one rounding of the real quotient gives.
//
// Both directions are bound by memory, and are a chain of three or four loads (rows, block ids, values) ahead of it: a block of threads finds its rows once for several heads or rows, and
// then has all its values on their way at once.
#include <stdio.h>

#include "kv8.cuh"
#include "workspace.h"

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
// odd: a value of the tile is an infinity or NaN
template <int FMT>
__device__ __forceinline__ uint32_t kv8_encode4(float4 x, float s, float inv, bool odd) {
  constexpr float MOST = FMT == THA_KV8_INT8 ? 127.f : 448.f;
  const float v[4] = {x.x, x.y, x.z, x.w};
  float y[4];
  bool close = odd;
  if (FMT == THA_KV8_INT8) {
    constexpr float MAGIC = 12582912.f;                     // 1.5 * 2^23: what is added to it is rounded to an integer, which the sum's low bits hold
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float r = fmaf(v[i], inv, MAGIC);
      close |= fabsf(fmaf(v[i], inv, MAGIC - r)) > 0.4999f; // 127 * 2^-22 = 3e-5
      w[i] = __float_as_uint(r);
    }
    if (!close) return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      y[i] = v[i] * inv;
      // a border is where bit 19 begins what is cut off, from 2^-6 upwards; below, steps are 2^-9 all the way, and few values are there
      const uint32_t b = __float_as_uint(y[i]);
      close |= (fabsf(y[i]) < 0.015625f && y[i] != 0.f) || ((b & 0xFFFFFu) - 0x80000u + 16u) < 33u;
    }
  }
  if (close) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      y[i] = fabsf(v[i]) < INFINITY ? (s > 0.f ? quotient_to_odd(v[i], s) : 0.f) : v[i] == v[i] ? (s > 0.f ? copysignf(MOST, v[i]) : 0.f) : 0.f;
      y[i] = fminf(fmaxf(y[i], -MOST), MOST);
    }
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
  const int sh = kv8_shift(block_size), blocks = ((p0 + n - 1) >> sh) - (p0 >> sh) + 1;
  return blocks > 1 ? blocks - 1 : 1;
}

constexpr int KW_WARPS = 16, KW_ROWS = 8;
// `words` words of codes under the scale *s (NULL: there is no block) into open rows, as the values that they stand for: a warp, every lane those that it has in kv8_write_kernel.
template <int FMT>
__device__ __forceinline__ void kv8_back_from_codes(const uint8_t* codes, const float* scale, int words, float* open) {
  const float s = scale ? *scale : 0.f;
#pragma unroll 1
  for (int i = threadIdx.x & 31; i < words; i += 32) {
    const float4 x = kv8_decode4<FMT>(scale ? reinterpret_cast<const uint32_t*>(codes)[i] : 0u);
    reinterpret_cast<float4*>(open)[i] = make_float4(x.x * s, x.y * s, x.z * s, x.w * s);
  }
}

// A warp: 8 rows of a block of the cache, one head, K or V; their values in registers (up to 8 float4 a lane) between the maximum and the codes, so that they are read once.  The
// block_size / 8 warps of a tile are neighbours and tell each other their maxima.  A thread block takes `each` units in turn, so that what it looks up for the first serves the others.
// Prompts of 37, 1042 and 2048 rows, 32 heads of 128, fp32: a thread block a tile, with the quotients and positions made value by value, 68 us, like this 47 (behind cold caches;
// 128 MB are 20).
// grid (units / each, groups of 16 / (block_size / 8) heads, 2)
// FULL: heads of 128 channels, a row a warp's float4.  ENDS: what the open rows hold is known (tha_kv8_t.open_end) and kept: a load more ahead of the
// first block's rows, three prompts 49 us for 47, single rows 0.6 us more; 4 us more where a long prompt's first rows come back from codes.
template <typename T, int FMT, bool VEC, bool FULL, bool ENDS>
__global__ void __launch_bounds__(32 * KW_WARPS, 2) kv8_write_kernel(tha_rows_t rows, tha_kv8_t kv, int layer, int each, const T* k, long long ldk, const T* v, long long ldv) {
  hyb_pdl_enter();
  constexpr float MOST = FMT == THA_KV8_INT8 ? 127.f : 448.f;
  constexpr int N = KW_ROWS;                                 // float4 a lane
  __shared__ float s_top[2][KW_WARPS];                       // two tiles in turn: one barrier a tile
  __shared__ int s_odd[2][KW_WARPS];
  const int B = kv.block_size, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sh = kv8_shift(B), per = B / KW_ROWS, part = warp & (per - 1);
  const int h = (blockIdx.y * KW_WARPS + warp) >> (sh - 3);
  const bool is_v = blockIdx.z != 0, live = h < kv.kv_heads;
  static_assert(KW_ROWS == 8, "block_size / 8 warps");
  const int W = FULL ? 128 : is_v ? kv.vdim : kv.dim, w4 = W >> 2;
  const long long ld = is_v ? ldv : ldk;
  uint8_t* pool = static_cast<uint8_t*>(is_v ? kv.v_pool : kv.k_pool);
  float* scales = is_v ? kv.v_scale : kv.k_scale;
  // float4 lane + 32 i of the warp's rows: its row and column, one after the other
  const int in0 = lane / w4, c0 = lane - in0 * w4, rows_on = 32 / w4, c_on = 32 - rows_on * w4;
  auto next = [&](int& in, int& c) {
    if (FULL) { in++; return; }
    in += rows_on; c += c_on;
    if (c >= w4) { c -= w4; in++; }
  };
  int turn = 0;
  // of the present sequence
  int p0 = 0, p_end = 0, slot = 0;
  float* open = nullptr;
  const T* src = nullptr;
  auto make = [&](int b) {                                   // the whole thread block: one sequence, one block of positions
    const int id = kv8_block(kv, slot, b << sh), t0 = (b << sh) + KW_ROWS * part;   // the warp's first position
    float4 x[N];
    float top = 0.f;
    int in = in0, c = c0;
    const T* from = src + (long long)(t0 - p0) * ld;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int t = t0 + in;
      x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (live && (FULL || in < KW_ROWS) && t < p_end) {
        if (t < p0) x[i] = *reinterpret_cast<const float4*>(open + (KW_ROWS * part + in) * W + 4 * c);
        else x[i] = kv8_row4<VEC>(from + in * ld + 4 * c);
      }
      next(in, c);
    }
    float2 none = make_float2(0.f, 0.f);                     // 0 times what is finite
#pragma unroll
    for (int i = 0; i < N; i++) {
      top = k8_max3(top, k8_max3(fabsf(x[i].x), fabsf(x[i].y), fabsf(x[i].z)), fabsf(x[i].w));
      none = f32x2_fma(make_float2(x[i].x, x[i].y), make_float2(0.f, 0.f), none);
      none = f32x2_fma(make_float2(x[i].z, x[i].w), make_float2(0.f, 0.f), none);
    }
    const bool odd_here = none.x != 0.f || none.y != 0.f;    // true for NaN
    if (odd_here) {
      top = 0.f;
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float m[4] = {fabsf(x[i].x), fabsf(x[i].y), fabsf(x[i].z), fabsf(x[i].w)};
#pragma unroll
        for (int j = 0; j < 4; j++) top = fmaxf(top, m[j] < INFINITY ? m[j] : 0.f);   // false for NaN too
      }
    }
    top = warp_max(top);
    bool odd = __any_sync(THA_FULL_MASK, odd_here);
    if (lane == 0) { s_top[turn][warp] = top; s_odd[turn][warp] = odd; }
    __syncthreads();                                         // and the open rows of this block have been read
    for (int i = 0; i < per; i++) { top = fmaxf(top, s_top[turn][warp - part + i]); odd |= s_odd[turn][warp - part + i] != 0; }
    turn ^= 1;
    const float s = top > 0.f ? fmaxf(__fdiv_rn(top, MOST), 1.17549435e-38f) : 0.f, inv = s > 0.f ? __fdividef(1.0f, s) : 0.f;
    const bool open_block = ((b + 1) << sh) > p_end;
    const size_t tile = id >= 0 && live ? kv8_tile(kv, id, layer, h) : 0;
    if (id >= 0 && live && part == 0 && lane == 0) scales[tile] = s;
    uint8_t* codes = pool + (tile * B + KW_ROWS * part) * W;
    in = in0; c = c0;
    asm volatile("" : "+r"(in), "+r"(c));                    // counted anew: rows and columns kept from above are registers that the values need
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int t = t0 + in;
      if (live && (FULL || in < KW_ROWS)) {
        if (id >= 0) *reinterpret_cast<uint32_t*>(codes + in * W + 4 * c) = kv8_encode4<FMT>(x[i], s, inv, odd);
        if (open_block && t >= p0 && t < p_end) *reinterpret_cast<float4*>(open + (KW_ROWS * part + in) * W + 4 * c) = x[i];
      }
      next(in, c);
    }
  };
  int seq = -1, unit = 0, units = 0;
  for (int u = 0; u < each; u++) {
    const int i = blockIdx.x * each + u;
    if (seq >= 0 && unit + 1 < units) {
      unit++;
    } else {
      if (rows.max_seq_rows > 1) {
        const Kv8Piece pc = kv8_find(rows.n_seqs, i, [&](int s) { return kv8_units(rows, s, B); });
        seq = pc.seq; unit = pc.at;
      } else {                                               // every sequence is a row: a unit
        seq = i < rows.n_seqs ? i : -1; unit = 0;
      }
      if (seq < 0) return;
      const int r0 = rows.max_seq_rows > 1 ? rows.seq_first[seq] : seq, n = rows.max_seq_rows > 1 ? rows.seq_first[seq + 1] - r0 : 1;
      slot = rows.seq_slot[seq];
      p0 = rows.pos[r0];
      p_end = p0 + n;
      units = p0 >= 0 ? ((p_end - 1) >> sh) - (p0 >> sh) : 0;
      open = (is_v ? kv.v_open : kv.k_open) + (live ? kv8_tile(kv, slot, layer, h) * (size_t)B * W : 0);
      src = (is_v ? v : k) + (long long)r0 * ld + (live ? (long long)h * W : 0);
      if (ENDS && p0 >= 0 && unit == 0 && live && (p0 & (B - 1))) {
        // rows of the block ahead of p0 that the open rows do not hold (they are a later block's): from the codes
        const int lead = p0 & (B - 1), e = kv.open_end[2 * kv8_tile(kv, slot, layer, h) + is_v];
        if (e >= 0 && (e < p0 || e > p0 - lead + B)) {
          const int id = kv8_block(kv, slot, p0);
          const size_t tile = id >= 0 ? kv8_tile(kv, id, layer, h) : 0;
          kv8_back_from_codes<FMT>(pool + (tile * B + KW_ROWS * part) * W, id >= 0 ? scales + tile : nullptr, min(max(lead - KW_ROWS * part, 0), KW_ROWS) * w4, open + KW_ROWS * part * W);
        }
      }
    }
    if (p0 < 0) continue;
    make((p0 >> sh) + unit);
    // The thread block of a sequence's first block also makes its last one, because it reads the slot's open rows (behind make's barrier they have been read) and the last one
    // replaces them.
    if (unit == 0 && units > 0) make((p_end - 1) >> sh);
    // what the open rows hold now: the last block's, or, where that is full, the first's ahead of p0 as before.  All warps of the tile have read the number ahead of make's barrier.
    if (ENDS && unit == 0 && live && part == 0 && lane == 0)
      kv.open_end[2 * kv8_tile(kv, slot, layer, h) + is_v] = p_end & (B - 1) ? p_end : p0 & (B - 1) ? p0 : 0;
  }
}

// V codes a thread: 16 bytes of result
template <typename T> struct Kv8Out;
template <> struct Kv8Out<float> {
  using Word = uint32_t;
  template <int FMT>
  static __device__ __forceinline__ uint4 make(uint32_t w, float s) {
    const float4 x = kv8_decode4<FMT>(w);
    return make_uint4(__float_as_uint(x.x * s), __float_as_uint(x.y * s), __float_as_uint(x.z * s), __float_as_uint(x.w * s));
  }
};
template <> struct Kv8Out<__nv_bfloat16> {
  using Word = uint2;
  template <int FMT>
  static __device__ __forceinline__ uint4 make(uint2 w, float s) {
    const float4 a = kv8_decode4<FMT>(w.x), b = kv8_decode4<FMT>(w.y);
    const __nv_bfloat162 p[4] = {__floats2bfloat162_rn(a.x * s, a.y * s), __floats2bfloat162_rn(a.z * s, a.w * s), __floats2bfloat162_rn(b.x * s, b.y * s),
                                 __floats2bfloat162_rn(b.z * s, b.w * s)};
    return *reinterpret_cast<const uint4*>(p);
  }
};

// grid (groups of R rows, 2): the rows' heads, K or V.  Eight words of codes of a thread are on their way at once.  8 contexts of 301 .. 2048 rows, 32 heads of 128, bf16: a thread
// block a row 63 us, 8 rows 42.
constexpr int KR_ROWS = 8;
template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(256) kv8_read_kernel(tha_rows_t rows, tha_kv8_t kv, int layer, int R, T* k, long long ldk, T* v, long long ldv) {
  hyb_pdl_enter();
  using Word = typename Kv8Out<T>::Word;
  constexpr int V = 16 / (int)sizeof(T), DEEP = 8;
  const bool is_v = blockIdx.y != 0;
  T* out = is_v ? v : k;
  if (!out) return;
  __shared__ long long s_at[KR_ROWS];                        // of the row's tile of head 0, -1: it has none
  __shared__ int s_in[KR_ROWS];
  const int W = is_v ? kv.vdim : kv.dim, wv = W / V, B = kv.block_size, r0 = blockIdx.x * R, here = min(R, rows.n_rows - r0), words = kv.kv_heads * wv;
  const long long ld = is_v ? ldv : ldk;
  if (threadIdx.x < here) {
    const int r = r0 + threadIdx.x, t = rows.pos[r], id = t >= 0 ? kv8_block(kv, rows.seq_slot[rows.row_seq[r]], t) : -1;
    s_at[threadIdx.x] = id >= 0 ? (long long)kv8_tile(kv, id, layer, 0) : -1;
    s_in[threadIdx.x] = t >= 0 ? t & (B - 1) : 0;
  }
  __syncthreads();
  const uint8_t* pool = static_cast<const uint8_t*>(is_v ? kv.v_pool : kv.k_pool);
  const float* scales = is_v ? kv.v_scale : kv.k_scale;
  // x / wv for x < 2^22: words of a row are below 65536 * 32
  const unsigned inverse = (unsigned)((0x100000000ull + wv - 1) / (unsigned)wv);
  int row = threadIdx.x / words, x = threadIdx.x - row * words;   // of the word that is asked for next
  auto next = [&](int& row, int& x) {
    for (x += blockDim.x; x >= words; x -= words) row++;
  };
  while (row < here) {
    Word w[DEEP];
    float s[DEEP];
    int put_row = row, put_x = x;
#pragma unroll
    for (int i = 0; i < DEEP; i++) {
      const int h = (int)__umulhi((unsigned)x, inverse), c = V * (x - h * wv);
      const long long at = row < here ? s_at[row] : -1;
      w[i] = {};
      s[i] = 0.f;
      if (at >= 0) {
        w[i] = __ldg(reinterpret_cast<const Word*>(pool + (((size_t)at + h) * B + s_in[row]) * W + c));
        s[i] = __ldg(scales + at + h);
      }
      next(row, x);
    }
#pragma unroll
    for (int i = 0; i < DEEP; i++) {
      if (put_row >= here) break;
      const uint4 y = Kv8Out<T>::template make<FMT>(w[i], s[i]);
      T* dst = out + (long long)(r0 + put_row) * ld + V * put_x;   // heads follow one another
      if (VEC) {
        *reinterpret_cast<uint4*>(dst) = y;
      } else {
#pragma unroll
        for (int j = 0; j < V; j++) dst[j] = reinterpret_cast<const T*>(&y)[j];
      }
      next(put_row, put_x);
    }
  }
}

template <typename T, int FMT, bool VEC>
static int write_launch(cudaStream_t s, const tha_rows_t* rows, const tha_kv8_t* kv, int layer, const T* k, long long ldk, const T* v, long long ldv) {
  const int units = rows->max_seq_rows == 1 ? rows->n_seqs : rows->n_rows / kv->block_size + rows->n_seqs;
  const int groups = ceil_div(kv->kv_heads, KW_WARPS * KW_ROWS / kv->block_size);
  const int sms = sm_budget(), each = units * groups >= 8 * sms ? 4 : units * groups >= 4 * sms ? 2 : 1;   // two rounds of two blocks on every SM, K and V
  auto go = [&](auto kernel) -> int {
    THA_CUDA_OK(launch(kernel, dim3(ceil_div(units, each), groups, 2), dim3(32 * KW_WARPS), 0, s, pdl_enabled() != 0, *rows, *kv, layer, each, k, ldk, v, ldv));
    return THA_STATUS_SUCCESS;
  };
  const bool full = kv->dim == 128 && kv->vdim == 128;
  if (kv->open_end) return full ? go(kv8_write_kernel<T, FMT, VEC, true, true>) : go(kv8_write_kernel<T, FMT, VEC, false, true>);
  return full ? go(kv8_write_kernel<T, FMT, VEC, true, false>) : go(kv8_write_kernel<T, FMT, VEC, false, false>);
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
  constexpr int V = 16 / (int)sizeof(T);
  const bool vec = ((k ? ldk : 0) | (v ? ldv : 0)) % V == 0 && aligned16(k) && aligned16(v);
  const int R = rows->n_rows > 2 * sm_budget() * KR_ROWS ? KR_ROWS : 1;   // blocks for every SM first: 700 rows of 4 heads 8.1 us one by one, 9.5 in pairs
  const int words = R * kv->kv_heads * (kv->dim > kv->vdim ? kv->dim : kv->vdim) / V;
  const dim3 grid(ceil_div(rows->n_rows, R), 2), block(words > 128 ? 256 : words > 64 ? 128 : 64);
  auto go = [&](auto kernel) -> int {
    THA_CUDA_OK(launch(kernel, grid, block, 0, s, pdl_enabled() != 0, *rows, *kv, layer, R, k, ldk, v, ldv));
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
