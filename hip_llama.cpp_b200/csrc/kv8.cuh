// The cache in 8 bits: what its kernels share.  A block of positions and a head is [position][channel] bytes without gaps, so that 16 positions are one
// contiguous run of 16 * dim bytes; all offsets are multiples of 16 bytes because channels are multiples of 16.
#pragma once
#include <cuda_fp8.h>

#include "hybrid_ops.cuh"
#include "split_f16.cuh"

namespace tha {

// index of (block, layer, head): of its scale, and in units of block_size * width of its codes and open rows
__device__ __forceinline__ size_t kv8_tile(const tha_kv8_t& kv, int block, int layer, int head) {
  return ((size_t)block * kv.n_cache_layers + layer) * kv.kv_heads + head;
}
// log2 of a block size
__device__ __forceinline__ int kv8_shift(int block_size) { return 31 - __clz(block_size); }
// block id of a slot's position, -1 where the table holds none that exists
__device__ __forceinline__ int kv8_block(const tha_kv8_t& kv, int slot, int t) {
  const int b = t >> kv8_shift(kv.block_size);
  if (t < 0 || b >= kv.table_stride) return -1;
  const int id = kv.table[(size_t)slot * kv.table_stride + b];
  return (unsigned)id < (unsigned)kv.n_blocks ? id : -1;
}
// Piece `i` of the pieces that `of(seq)` counts for every sequence, in order; seq -1 behind the last.  A whole warp asks.
struct Kv8Piece { int seq, at; };
template <typename F>
__device__ __forceinline__ Kv8Piece kv8_find(int n_seqs, int i, F of) {
  const int lane = threadIdx.x & 31;
  for (int s0 = 0; s0 < n_seqs; s0 += 32) {
    const int mine = s0 + lane < n_seqs ? of(s0 + lane) : 0;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(THA_FULL_MASK, upto, o); if (lane >= o) upto += v; }
    const unsigned past = __ballot_sync(THA_FULL_MASK, upto > i);
    if (past) {
      const int l = __ffs(past) - 1;
      return {s0 + l, i - __shfl_sync(THA_FULL_MASK, upto - mine, l)};
    }
    i -= __shfl_sync(THA_FULL_MASK, upto, 31);
  }
  return {-1, 0};
}

// hyb_attn_sees for the 32 keys from kt on, as bits: a query at `pos` whose chunk begins at `first`
__device__ __forceinline__ uint32_t kv8_sees32(const tha_attn_t& a, int kt, int pos, int first) {
  auto below = [&](int t) { const int n = t - kt; return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; };   // keys kt .. t - 1
  uint32_t seen = ~below(first);
  if (a.window > 0) seen &= ~below(pos - a.window + 1) | below(a.keep_first);
  return seen & below(pos + 1);
}

// four codes to fp32
template <int FMT>
__device__ __forceinline__ float4 kv8_decode4(uint32_t w) {
  if (FMT == THA_KV8_INT8)
    return make_float4((float)(int8_t)(w & 0xFFu), (float)(int8_t)(w >> 8 & 0xFFu), (float)(int8_t)(w >> 16 & 0xFFu), (float)(int8_t)(w >> 24));
  const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3);
  const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
  const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
  return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ float k8_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 k8_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// Bytes 0 and 2 of w as fp16.  int8: a byte with its sign flipped is code + 128; in the low half of 0x6400 = 1024.0 that is 1024 + 128 + code exactly.
__device__ __forceinline__ uint32_t k8_bytes02(uint32_t w) {
  const uint32_t u = (w & 0x00FF00FFu) ^ 0x64806480u;
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t k8_e4m3x2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return (uint32_t)h.x | (uint32_t)h.y << 16;
}

// x log2(e), finite where x is: numbers from 2^127 on, as the type's lowest that stands for "not this key", would become infinities.  They are brought closer together there, in their
// order, and stay further apart than any weight reaches.
__device__ __forceinline__ float k8_log2_units(float x) {
  return fabsf(x) > 0x1p127f && fabsf(x) < INFINITY ? fmaf(0.5f, x, copysignf(1.88539f * 0x1p126f, x)) : x * 1.4426950408889634f;   // 2^127 log2(e) = 2^126 + 1.88539 2^126
}
// The factor of a (query, head)'s accumulator with m the maximum (times log2(e)) and l the sum: 1 / (l + exp(sink - m)) times the head's gate; 0 where nothing was seen.
__device__ __forceinline__ float k8_final(const tha_attn_t& a, int h, float m, float l, const float* gate_row) {
  if (!(m > -INFINITY)) return m != m ? m : 0.f;            // a NaN stays one
  float f;
  if (a.sink) {
    const float sk = k8_log2_units(a.sink[h]), M = fmaxf(m, sk), e = exp2f(m - M);
    f = e / (l * e + exp2f(sk - M));
  } else {
    f = 1.0f / l;
  }
  if (gate_row) f *= hyb_sigmoid(gate_row[h]);
  return f;
}
__device__ __forceinline__ void k8_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void k8_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Partial results of `splits` parts of `all` (row, head)s: maxima and sums [part][all][2], rounded up to 16 bytes, then weighted means [part][all][E]
__host__ __device__ __forceinline__ size_t k8_sums_floats(int splits, size_t all) { return (2 * all * splits + 3) & ~(size_t)3; }
__host__ __device__ __forceinline__ size_t k8_partial_floats(int splits, size_t all, int E) { return k8_sums_floats(splits, all) + all * splits * E; }

// host side: kv8_rows.cu
int kv8_check(const tha_rows_t* rows, const tha_kv8_t* kv, int cache_layer, const char* who);
int kv8_refuse(const char* who, const char* why);
// whether every operand of the products is two fp16: portions with bf16 results take one, unless the caller asks for fp32 scores
inline bool kv8_exact(const tha_attn_t* a, int dtype) { return dtype == THA_DT_F32 || a->fp32_scores; }
// kv8_attn_tc.cu: sequences of at least min_rows rows; THA_STATUS_NOT_SUPPORTED (nothing launched): the caller takes another form
int kv8_attn_tc_splits(const tha_attn_t* a, const tha_rows_t* rows, int dtype, int most_tiles);
size_t kv8_attn_tc_stage_bytes(const tha_attn_t* a, const tha_rows_t* rows, int most_tiles, int min_rows);
int kv8_attn_tc_room_for(const tha_attn_t* a, int most_tiles);   // sequences whose visible keys may be staged at once
int kv8_attn_tc_launch(cudaStream_t s, int dtype, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, void* out, int min_rows, int most_tiles,
                       int splits, void* staged, float* partial, const float* gate, long long ldg);

}  // namespace tha
