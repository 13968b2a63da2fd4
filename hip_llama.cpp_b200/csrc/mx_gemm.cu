// Products over microscaled numbers (tha_mx_t) on the tensor cores' block-scaled kinds:
//
//   C[n, m] = sum_k A[n, k] W[m, k],   A [N, K] rows in 8 or 4 bits, W [M, K] in 4 bits, scales powers of two for each 32 values of a row
//
// tcgen05.mma multiplies codes, which are exact, and the two scales of a block of k, which are powers of two, and sums in fp32 in TMEM.  Which kind goes by A's format:
//   E4M3 x E2M1   kind::mxf8f6f4, 32 values of k an instruction; 4-bit codes lie in shared memory as 8 bytes of codes and 8 of nothing for each 16, which TMA makes of the packed rows
//   E2M1 x E2M1   kind::mxf4, 64 values of k an instruction, codes packed
// Weight rows are the instruction's M (128 TMEM lanes), activation rows its N.  Scales lie in TMEM too: a tile of 128 rows and 4 blocks (512 bytes, as tha_mx_t keeps them) becomes
// 4 columns by one tcgen05.cp, lane l and column j holding the four bytes of row 32 j + l.
//
// A block of threads takes a tile of 128 weight rows (of each of two matrices for a gated activation) and NT activation rows: warp 0 asks for codes (TMA) and scales (bulk copies)
// into a ring of stages, warp 1 issues copies of scales and MMAs, warps 4-7 read the accumulators out: a thread a weight row, a warp 32 neighbouring results of one activation row.
// A feed-forward's activation and the quantising of its result happen there: the 32 values of a block are the 32 lanes of a warp.
#include "hybrid_ops.cuh"
#include "mx.cuh"
#include "tc_common.cuh"

namespace tha {

int gemm_tc_init(int** flag_out);

namespace {

constexpr int MG_THREADS = 256;
enum { MG_F8 = 0, MG_F4 = 1 };                     // kind::mxf8f6f4, kind::mxf4
enum { MG_PLAIN = 0, MG_UNGATED = 1, MG_GATED = 2 };

struct MgP {
  int M, N, K;                                     // weight rows, activation rows, values of a row
  int ny;                                          // tiles of activation rows
  int across;                                      // tiles of 128 values along k
  const uint8_t *sw0, *sw1, *sx;                   // scales of the matrices
  uint32_t idesc;                                  // formats, sizes; without the places of the scales
  int w_bytes, x_bytes;                            // what a whole stage's TMA copies of codes bring
  void* out; long long ldo; int bf16;              // MG_PLAIN
  tha_mx_t y; int act; float limit, alpha;         // MG_UNGATED, MG_GATED
  int* error_flag;
};

template <int KIND, int NT, int READ>
struct MgSmem {
  static constexpr int WT = READ == MG_GATED ? 2 : 1;                 // weight matrices
  static constexpr int XT = (NT + 127) / 128;                         // scale tiles of the activation rows
  static constexpr int CH = KIND == MG_F4 ? 2 : 1;                    // scale tiles along k in a stage (128 bytes of a row of codes)
  static constexpr int W_BYTES = WT * TC_BM * 128, X_BYTES = NT * 128;
  static constexpr int SW_BYTES = CH * MX_TILE_BYTES, SX_BYTES = CH * MX_TILE_BYTES;   // of one matrix, of one row tile
  static constexpr int STAGE = (W_BYTES + X_BYTES + WT * SW_BYTES + XT * SX_BYTES + 1023) / 1024 * 1024;
  static constexpr int ROOM = STAGE <= 24 * 1024 ? 110 * 1024 : 220 * 1024;             // two blocks an SM, or one
  static constexpr int NST = ROOM / STAGE > 8 ? 8 : ROOM / STAGE;
  static constexpr int ACC_COLS = WT * NT;
  static constexpr int SET = CH * 4 * (WT + XT);                      // TMEM columns of a stage's scales
  static constexpr int COLS = ACC_COLS + NST * SET;
  static constexpr int TMEM_COLS = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static constexpr int TOTAL = NST * STAGE + 1024 + (2 * NST + 1) * 8 + 64;
  static_assert(COLS <= 512 && TOTAL <= TC_SMEM_LIMIT && NST >= 3, "a stage is too large");
};

__device__ __forceinline__ void mg_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(tc_smem_u32(dst)), "l"(src), "r"(bytes), "r"(tc_smem_u32(bar)) : "memory");
}
// 512 bytes of scales, 32 rows of 16 bytes in a row, into 4 TMEM columns, for each of the four lane quarters
__device__ __forceinline__ void mg_copy_scales(uint32_t taddr, uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;   // groups of 8 rows are 128 bytes apart, no swizzle
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}
template <int KIND>
__device__ __forceinline__ void mg_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  if (KIND == MG_F8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}
// Block-scaled instruction descriptor: formats of A and B, N / 8, scales as powers of two, M / 16.  Which of a scale word's four bytes an instruction takes is in bits 4-5 (B), 29-30 (A).
uint32_t mg_idesc(int kind, int fa, int fb, int nt) {
  const uint32_t a = kind == MG_F4 ? 1u : fa == THA_MX_E2M1 ? 5u : 0u, b = kind == MG_F4 ? 1u : fb == THA_MX_E2M1 ? 5u : 0u;
  return a << 7 | b << 10 | (uint32_t)(nt >> 3) << 17 | 1u << 23 | (uint32_t)(TC_BM >> 4) << 24;
}

// One result a lane, the warp's 32 a block: into codes and the block's scale.  col: the lane's column, a multiple of 32 in lane 0.  All lanes of the warp.
template <int FMT>
__device__ __forceinline__ void mg_store_block(const tha_mx_t& y, int row, int col, long long padded, float v) {
  const int lane = threadIdx.x & 31;
  const unsigned top = __reduce_max_sync(THA_FULL_MASK, __float_as_uint(v) & 0x7fffffffu), byte = mx_scale_byte<FMT>(top);
  v = byte == 255u ? 0.f : v * mx_inverse(byte);
  if (FMT == THA_MX_E2M1) {
    const float next = __shfl_down_sync(THA_FULL_MASK, v, 1);
    if (!(lane & 1)) static_cast<uint8_t*>(y.codes)[(size_t)row * (padded / 2) + col / 2] = (uint8_t)mx_e2m1x2(v, next);
  } else {
    static_cast<uint8_t*>(y.codes)[(size_t)row * padded + col] = (uint8_t)mx_e4m3x2(v, 0.f);
  }
  if (lane == 0) y.scales[mx_scale_at(row, col / MX_TILE, (int)(padded / MX_TILE)) + (col / MX_BLOCK & 3)] = (uint8_t)byte;
}

template <int KIND, int NT, int READ>
__global__ void __launch_bounds__(MG_THREADS)
mx_gemm_kernel(const __grid_constant__ CUtensorMap mw0, const __grid_constant__ CUtensorMap mw1, const __grid_constant__ CUtensorMap mx, const MgP p) {
  using S = MgSmem<KIND, NT, READ>;
  constexpr int WT = S::WT, CH = S::CH, KB = CH * MX_TILE;             // KB: values of k in a stage
  extern __shared__ unsigned char tc_smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tc_smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::NST * S::STAGE);   // stage landed
  uint64_t* empty = full + S::NST;                                          // the MMAs that read the stage have completed
  uint64_t* accum = empty + S::NST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = (int)blockIdx.x / p.ny, row0 = tile * TC_BM, n0 = ((int)blockIdx.x - tile * p.ny) * NT;
  const int nkb = (p.across + CH - 1) / CH;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::NST; s++) { tc_mbar_init(&full[s], 1); tc_mbar_init(&empty[s], 1); }
    tc_mbar_init(accum, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(tmem_slot)), "r"(S::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_sf = tmem + S::ACC_COLS;

  if (warp == 0) {
    if (tc_elect()) {
      for (int i = 0; i < nkb; i++) {
        const int s = i % S::NST;
        if (i >= S::NST && !tc_mbar_wait(&empty[s], ((i / S::NST) & 1u) ^ 1u, abort_flag)) { tc_drain(full, S::NST, i); break; }
        const int t0 = i * CH, chunks = min(CH, p.across - t0);              // scale tiles of this stage: one in an odd matrix's last stage
        unsigned char* st = smem + s * S::STAGE;
        unsigned char* sw = st + S::W_BYTES + S::X_BYTES;
        unsigned char* sx = sw + WT * S::SW_BYTES;
        const uint32_t some = (uint32_t)(chunks * MX_TILE_BYTES);
        tc_mbar_expect_tx(&full[s], p.w_bytes + p.x_bytes + (WT + S::XT) * some);
        tc_tma_2d(st, &mw0, i * (KIND == MG_F4 ? KB / 2 : KB), row0, &full[s]);
        if (WT == 2) tc_tma_2d(st + TC_BM * 128, &mw1, i * (KIND == MG_F4 ? KB / 2 : KB), row0, &full[s]);
        tc_tma_2d(st + S::W_BYTES, &mx, i * (KIND == MG_F4 ? KB / 2 : KB), n0, &full[s]);
        mg_bulk(sw, p.sw0 + mx_scale_at(row0, t0, p.across), some, &full[s]);
        if (WT == 2) mg_bulk(sw + S::SW_BYTES, p.sw1 + mx_scale_at(row0, t0, p.across), some, &full[s]);
#pragma unroll
        for (int x = 0; x < S::XT; x++) mg_bulk(sx + x * S::SX_BYTES, p.sx + mx_scale_at(n0 + 128 * x, t0, p.across), some, &full[s]);
      }
    }
  } else if (warp == 1) {
    if (tc_elect()) {
      bool ok = true;
      for (int i = 0; i < nkb; i++) {
        const int s = i % S::NST;
        if (!tc_mbar_wait(&full[s], (i / S::NST) & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const int chunks = min(CH, p.across - i * CH);
        const uint32_t st = tc_smem_u32(smem + s * S::STAGE), sw = st + S::W_BYTES + S::X_BYTES, sx = sw + WT * S::SW_BYTES;
        // a stage has TMEM columns of its own for its scales: the MMAs that read their last contents have completed when the stage was filled again
        const uint32_t sf = tmem_sf + (uint32_t)(s * S::SET);
        for (int c = 0; c < chunks; c++) {
#pragma unroll
          for (int w = 0; w < WT; w++) mg_copy_scales(sf + (uint32_t)(4 * (c * (WT + S::XT) + w)), sw + (uint32_t)(w * S::SW_BYTES + c * MX_TILE_BYTES));
#pragma unroll
          for (int x = 0; x < S::XT; x++) mg_copy_scales(sf + (uint32_t)(4 * (c * (WT + S::XT) + WT + x)), sx + (uint32_t)(x * S::SX_BYTES + c * MX_TILE_BYTES));
        }
        const uint64_t adesc = tc_smem_desc(st), bdesc = tc_smem_desc(st + S::W_BYTES);
#pragma unroll
        for (int k = 0; k < 4; k++) {                // 32 bytes of codes each: 2 descriptor units
          const int c = KIND == MG_F4 ? k >> 1 : 0, id = KIND == MG_F4 ? 2 * (k & 1) : k;
          if (c < chunks) {
            const uint32_t at = sf + (uint32_t)(4 * c * (WT + S::XT));
#pragma unroll
            for (int w = 0; w < WT; w++)
              mg_mma<KIND>(tmem + (uint32_t)(w * NT), adesc + (uint64_t)(1024 * w + 2 * k), bdesc + (uint64_t)(2 * k), p.idesc | (uint32_t)id << 4 | (uint32_t)id << 29, at + 4 * w,
                           at + 4 * WT, (uint32_t)((i | k) != 0));
          }
        }
        tc_commit(&empty[s]);
      }
      if (ok) tc_commit(accum);
    }
  } else if (warp >= 4) {
    const int q = warp & 3, row = row0 + q * 32 + lane;                      // the weight row, a column of the result
    const bool ok = tc_mbar_wait_warp(accum, 0u, abort_flag);
    tc_fence_after();
    const uint32_t ta = tmem + ((uint32_t)(q * 32) << 16);
    const int cols = min(NT, p.N - n0);
    const long long padded = READ == MG_PLAIN ? 0 : mx_padded(p.M);
#pragma unroll 1
    for (int c = 0; c < cols; c += 16) {
      uint32_t v[16], g[16];
      if (ok) {
        tc_tmem_ld16(ta + (uint32_t)c, READ == MG_GATED ? g : v);
        if (READ == MG_GATED) tc_tmem_ld16(ta + (uint32_t)(NT + c), v);
        tc_wait_ld();
      }
#pragma unroll
      for (int j = 0; j < 16; j++) {
        if (c + j < cols) {
          float x = ok ? __uint_as_float(v[j]) : __uint_as_float(0x7fc00000u);
          if (READ == MG_PLAIN) {
            if (row < p.M) {
              const size_t at = (size_t)(n0 + c + j) * p.ldo + row;
              if (p.bf16) hyb_store(static_cast<__nv_bfloat16*>(p.out) + at, x);
              else static_cast<float*>(p.out)[at] = x;
            }
          } else {
            x = row < p.M ? hyb_act_value(p.act, READ == MG_GATED && ok ? __uint_as_float(g[j]) : x, x, p.limit, p.alpha) : 0.f;   // padding holds zeros
            if (p.y.format == THA_MX_E2M1) mg_store_block<THA_MX_E2M1>(p.y, n0 + c + j, row, padded, x);
            else mg_store_block<THA_MX_E4M3>(p.y, n0 + c + j, row, padded, x);
          }
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLS));
  }
  if (threadIdx.x == 0 && *abort_flag && p.error_flag) *((volatile int*)p.error_flag) = 1;
}

// ------------------------------------------------------------------ host side ----
// The codes of a matrix as TMA takes them: packed bytes for kind::mxf4; for kind::mxf8f6f4 bytes, or 4-bit values that are spread over 16 bytes for each 16.  `bytes`: what a box brings.
int mg_map(int kind, const tha_mx_t* m, int box_rows, CUtensorMap* out, int* bytes) {
  const long long padded = mx_padded(m->cols), pitch = mx_pitch(m->format, m->cols);
  const bool spread = kind == MG_F8 && m->format == THA_MX_E2M1;
  *bytes = box_rows * (spread ? 64 : 128);         // a barrier counts the bytes that are read
  if (spread) return tc_map_of(out, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, m->codes, m->rows, padded, pitch, box_rows, 128);
  return tc_map_of(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, m->codes, m->rows, pitch, pitch, box_rows, 128);
}

struct MgArgs { const tha_mx_t *A, *W0, *W1; MgP p; };

template <int KIND, int NT, int READ>
int mg_launch(cudaStream_t s, const MgArgs& a) {
  using S = MgSmem<KIND, NT, READ>;
  MgP p = a.p;
  CUtensorMap mw0, mw1, mx;
  int wb = 0;
  THA_TRY_RC(mg_map(KIND, a.W0, TC_BM, &mw0, &wb));
  mw1 = mw0;
  if (S::WT == 2) THA_TRY_RC(mg_map(KIND, a.W1, TC_BM, &mw1, &wb));
  THA_TRY_RC(mg_map(KIND, a.A, NT, &mx, &p.x_bytes));
  p.w_bytes = S::WT * wb;
  p.idesc = mg_idesc(KIND, a.W0->format, a.A->format, NT);
  p.ny = ceil_div(p.N, NT);
  const long long items = (long long)ceil_div(p.M, TC_BM) * p.ny;
  if (items > 0x7fffffff) return mx_refuse("tha_hyb_mx_linear", "too many results for one call");
  auto k = mx_gemm_kernel<KIND, NT, READ>;
  THA_CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL));
  THA_CUDA_OK(launch(k, dim3((unsigned)items), dim3(MG_THREADS), (size_t)S::TOTAL, s, false, mw0, mw1, mx, p));
  return THA_STATUS_SUCCESS;
}
template <int KIND, int READ>
int mg_width(cudaStream_t s, const MgArgs& a) {
  if (a.p.N <= 16) return mg_launch<KIND, 16, READ>(s, a);
  if (a.p.N <= 64) return mg_launch<KIND, 64, READ>(s, a);
  return mg_launch<KIND, 128, READ>(s, a);
}
template <int READ>
int mg_run(cudaStream_t s, const MgArgs& a) {
  return a.A->format == THA_MX_E2M1 ? mg_width<MG_F4, READ>(s, a) : mg_width<MG_F8, READ>(s, a);
}

int mg_check(const tha_mx_t* A, const tha_mx_t* W, const char* who) {
  THA_TRY_RC(mx_check(A, who));
  THA_TRY_RC(mx_check(W, who));
  if (W->format != THA_MX_E2M1) return mx_refuse(who, "the matrix is E2M1");
  if (A->cols != W->cols) return mx_refuse(who, "rows and matrix have different columns");
  return THA_STATUS_SUCCESS;
}
int mg_fill(MgArgs* a, const tha_mx_t* A, const tha_mx_t* W0, const tha_mx_t* W1) {
  a->A = A; a->W0 = W0; a->W1 = W1;
  a->p.M = W0->rows; a->p.N = A->rows; a->p.K = A->cols;
  a->p.across = (int)(mx_padded(A->cols) / MX_TILE);
  a->p.sw0 = W0->scales; a->p.sw1 = W1 ? W1->scales : nullptr; a->p.sx = A->scales;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;   // allocated by a device's first call, which a capture allows in this mode
  THA_CUDA_OK(cudaThreadExchangeStreamCaptureMode(&mode));
  const int st = gemm_tc_init(&a->p.error_flag);
  THA_CUDA_OK(cudaThreadExchangeStreamCaptureMode(&mode));
  return st;
}

}  // namespace
}  // namespace tha

using namespace tha;

extern "C" int tha_hyb_mx_linear(void* stream, int dtype, void* C, long long ldc, const tha_mx_t* A, const tha_mx_t* W) {
  const char* who = "tha_hyb_mx_linear";
  THA_TRY_RC(mg_check(A, W, who));
  if (dtype != THA_DT_F32 && dtype != THA_DT_BF16) return mx_refuse(who, "unknown dtype");
  if (A->rows == 0 || W->rows == 0) return THA_STATUS_SUCCESS;
  if (!C) return mx_refuse(who, "C is NULL");
  if (ldc < W->rows && A->rows > 1) return mx_refuse(who, "a row pitch below the row");
  MgArgs a = {};
  THA_TRY_RC(mg_fill(&a, A, W, nullptr));
  a.p.out = C; a.p.ldo = ldc; a.p.bf16 = dtype == THA_DT_BF16;
  return mg_run<MG_PLAIN>((cudaStream_t)stream, a);
}

extern "C" int tha_hyb_mx_linear_act(void* stream, int act, const tha_mx_t* A, const tha_mx_t* W_gate, const tha_mx_t* W_up, float limit, float alpha, const tha_mx_t* out) {
  const char* who = "tha_hyb_mx_linear_act";
  THA_TRY_RC(mg_check(A, W_up, who));
  THA_TRY_RC(mx_check(out, who));
  if (act < THA_ACT_GLU_CLAMPED || act > THA_ACT_SILU_GLU) return mx_refuse(who, "unknown activation");
  const bool gated = hyb_act_gated(act);
  if (gated != (W_gate != nullptr)) return mx_refuse(who, gated ? "a gated activation without its gate" : "a gate for an ungated activation");
  if (gated) {
    THA_TRY_RC(mg_check(A, W_gate, who));
    if (W_gate->rows != W_up->rows) return mx_refuse(who, "gate and up have different rows");
  }
  if (out->rows != A->rows || out->cols != W_up->rows) return mx_refuse(who, "the result is as many rows as A and as many columns as W_up has rows");
  if (A->rows == 0) return THA_STATUS_SUCCESS;
  if (act == THA_ACT_XIELU) {   // the two stored numbers p, q -> the factors the kernel multiplies with
    const float p = limit, q = alpha;
    limit = fmaxf(p, 0.f) + log1pf(expf(-fabsf(p)));
    alpha = 0.5f + fmaxf(q, 0.f) + log1pf(expf(-fabsf(q)));
  }
  MgArgs a = {};
  THA_TRY_RC(mg_fill(&a, A, gated ? W_gate : W_up, gated ? W_up : nullptr));
  a.p.y = *out; a.p.act = act; a.p.limit = limit; a.p.alpha = alpha;
  return gated ? mg_run<MG_GATED>((cudaStream_t)stream, a) : mg_run<MG_UNGATED>((cudaStream_t)stream, a);
}
