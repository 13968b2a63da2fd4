// Microscaled numbers (tha_mx_t): where a block's scale lies, which scale a block gets, and its values as codes.
#pragma once
#include <cuda_bf16.h>

#include <atomic>

#include "common.cuh"
#include "tha_hybrid.h"

namespace tha {

constexpr int MX_BLOCK = 32;      // values under one scale
constexpr int MX_TILE = 128;      // rows, and values of a row, of a tile of scales
constexpr int MX_TILE_BYTES = 512;
constexpr int MX_MOST = 1 << 30;  // rows, columns

__host__ __device__ __forceinline__ long long mx_padded(int cols) { return ((long long)cols + MX_TILE - 1) / MX_TILE * MX_TILE; }
__host__ __device__ __forceinline__ long long mx_pitch(int format, int cols) { return format == THA_MX_E2M1 ? mx_padded(cols) / 2 : mx_padded(cols); }
// the first of the four scale bytes of row r and column tile t (values 128 t ..), `across` column tiles in all
__host__ __device__ __forceinline__ size_t mx_scale_at(int r, int t, int across) {
  return ((size_t)(r / MX_TILE) * across + t) * MX_TILE_BYTES + (size_t)((r & 31) * 16 + (r >> 5 & 3) * 4);
}
int mx_refuse(const char* who, const char* why);
int mx_check(const tha_mx_t* m, const char* who);   // the matrix by itself
int mx_error_flag(int** flag);                      // where a kernel that gives up on a barrier says so (tha_gemm_check_error)
// More shared memory than 48 KB for a kernel's blocks, asked for once a device (0.3 us a call); devices beyond the bits ask every time.
template <typename K>
int mx_room(K kernel, int bytes, std::atomic<unsigned long long>* asked) {
  int dev = 0;
  THA_CUDA_OK(cudaGetDevice(&dev));
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (asked->load(std::memory_order_acquire) & bit) return THA_STATUS_SUCCESS;
  THA_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  asked->fetch_or(bit, std::memory_order_release);
  return THA_STATUS_SUCCESS;
}

#ifdef __CUDACC__
// The scale byte of a block whose largest |value| has the bits `top` (of an fp32 not below 0): with 2^e <= top < 2^(e + 1), the largest number of the format 1.5 * 2^2
// (1.75 * 2^8) is reached at 2^(e - 2) (2^(e - 8)) where the fraction of top is at most 1.5 (1.75), at the next power above it.  Infinities and NaN: 255.
template <int FMT>
__device__ __forceinline__ unsigned mx_scale_byte(unsigned top) {
  if (top >= 0x7f800000u) return 255u;
  constexpr unsigned most = FMT == THA_MX_E2M1 ? 0x400000u : 0x600000u;
  const int c = (int)(top >> 23) - (FMT == THA_MX_E2M1 ? 2 : 8) + ((top & 0x7fffffu) > most);
  return (unsigned)max(c, 0);
}
// 1 / scale: a power of two, so that a value times it is exact as far as codes can tell (what underflows is far below the smallest code's half)
__device__ __forceinline__ float mx_inverse(unsigned byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }
// scale itself: byte 0 is 2^-127, below fp32's normal numbers
__device__ __forceinline__ float mx_scale(unsigned byte) { return byte == 255u ? __uint_as_float(0x7fc00000u) : byte ? __uint_as_float(byte << 23) : __uint_as_float(0x400000u); }
// the codes of two values already divided by their scale, a in the low part: 4 bits each
__device__ __forceinline__ unsigned mx_e2m1x2(float a, float b) {
  unsigned r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(a), "f"(b));
  return r;
}
// 8 bits each
__device__ __forceinline__ unsigned mx_e4m3x2(float a, float b) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(a), "f"(b));
  return r;
}
#endif

}  // namespace tha
