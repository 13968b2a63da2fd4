// Products over microscaled numbers (tha_mx_t) on the tensor cores' block-scaled kinds:
//
//   C[n, m] = sum_k A[n, k] W[m, k],   A [N, K] rows in 8 or 4 bits, W [M, K] in 4 bits, scales powers of two for each 32 values of a row
//
// tcgen05.mma multiplies codes, which are exact, and the two scales of a block of k, which are powers of two, and sums in fp32 in TMEM.  Sums that 24 bits hold are exact; others are cut off
// at each instruction, so that rows of one sign come out low: of sum |a| |w|, 8-bit rows of 1024 / 4096 / 11008 / 32768 columns are off by 4e-8 / 1.9e-7 / 8.3e-7 / 6.8e-6 (a product in plain
// fp32 by 3e-8 / 7e-8 / 1.4e-7 / 4.7e-7), less where a cluster's blocks share the columns (32768: 1.8e-7); with signs at random 2e-9 at most.  Which kind goes by A's format:
//   E4M3 x E2M1   kind::mxf8f6f4, 32 values of k an instruction; 4-bit codes lie in shared memory as 8 bytes of codes and 8 of nothing for each 16, which TMA makes of the packed rows
//   E2M1 x E2M1   kind::mxf4, 64 values of k an instruction, codes packed
// Weight rows are the instruction's M (128 TMEM lanes), activation rows its N.  Scales lie in TMEM too: a tile of 128 rows and 4 blocks (512 bytes, as tha_mx_t keeps them) becomes
// 4 columns by one tcgen05.cp, lane l and column j holding the four bytes of row 32 j + l.
//
// A block of threads takes a tile of 128 weight rows (of each of two matrices for a gated activation) and NT activation rows: warp 0 asks for codes (TMA) and scales (bulk copies)
// into a ring of stages, warp 1 issues copies of scales and MMAs, then all warps (of 16 rows 4-7) read the accumulators out: a thread a weight row, a warp 32 neighbouring results of one
// activation row.  A feed-forward's activation and the quantising of its result happen there: the 32 values of a block are the 32 lanes of a warp.
// Few rows are bound by the way of a block's stages through its ring and by the meeting of a cluster: 1 row x [4096, 4096] 5.8 us on cold weights (1.4 at the copy rate), 16 rows x
// [2 x 11008, 4096] with silu 14.1 (7.4).  Prompts go to pairs of blocks (below).
#include "hybrid_ops.cuh"
#include "mx.cuh"
#include "tc_common.cuh"
#include "workspace.h"

namespace tha {

namespace {

constexpr int MG_THREADS = 256;
enum { MG_F8 = 0, MG_F4 = 1 };                     // kind::mxf8f6f4, kind::mxf4
enum { MG_PLAIN = 0, MG_UNGATED = 1, MG_GATED = 2 };

struct MgP {
  int M, N;                                        // weight rows, activation rows
  int ny, n_items;                                 // tiles of activation rows, items in all (pairs of blocks)
  int across;                                      // tiles of 128 values along k
  int ranks, share;                                // blocks of a cluster that share a tile, stages of each
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
  static constexpr int CH = KIND == MG_F4 ? 2 : 1;                    // scale tiles along k in a stage (128 bytes of a row of codes)
  static constexpr int W_BYTES = WT * TC_BM * 128, X_BYTES = NT * 128;
  static constexpr int SC_BYTES = CH * MX_TILE_BYTES;                 // scales of one matrix; of the activation rows, which lie in one tile
  static constexpr int STAGE = (W_BYTES + X_BYTES + (WT + 1) * SC_BYTES + 1023) / 1024 * 1024;
  static constexpr int ROOM = STAGE <= 37 * 1024 ? 111 * 1024 : 220 * 1024;             // two blocks an SM, or one
  static constexpr int NST = ROOM / STAGE > 8 ? 8 : ROOM / STAGE;
  static constexpr int ACC_COLS = WT * NT;
  static constexpr int SET = CH * 4 * (WT + 1);                       // TMEM columns of a stage's scales
  static constexpr int COLS = ACC_COLS + NST * SET;
  static constexpr int TMEM_COLS = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static constexpr int TOTAL = NST * STAGE + 1024 + (2 * NST + 2) * 8 + 64;
  static_assert(NST * STAGE >= ACC_COLS * TC_BM * 4, "the partial tile lies over the ring");
  static_assert(ROOM > 111 * 1024 || 2 * (TOTAL + 1024) <= 228 * 1024, "two blocks an SM");
  static_assert(COLS <= (ROOM <= 111 * 1024 ? 256 : 512) && TOTAL <= TC_SMEM_LIMIT && NST >= 3, "a stage is too large");
};

__device__ __forceinline__ void mg_prefetch(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
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
uint32_t mg_idesc(int kind, int rows, int nt) {
  const uint32_t a = kind == MG_F4 ? 1u : 5u, b = kind == MG_F4 ? 1u : 0u;       // E2M1 x E2M1; E2M1 x E4M3
  return a << 7 | b << 10 | (uint32_t)(nt >> 3) << 17 | 1u << 23 | (uint32_t)(rows >> 4) << 24;
}

// C results of a lane, the warp's 32 of each a block: into codes and scales.  Rows n .. of the result, `count` of them there; col: the lane's column, a multiple of 32 in lane 0.  All lanes
// of the warp.  Sixteen at a time: the maxima and codes of different rows wait for nothing of one another (one at a time 100 rows x [2 x 4608, 1024] 43.6 us).
template <int FMT, int C>
__device__ __forceinline__ void mg_store_blocks(const tha_mx_t& y, int n, int count, int col, long long padded, float (&v)[C]) {
  const int lane = threadIdx.x & 31;
  unsigned byte[C], mine = 0;
#pragma unroll
  for (int j = 0; j < C; j++) {
    byte[j] = mx_scale_byte<FMT>(__reduce_max_sync(THA_FULL_MASK, __float_as_uint(v[j]) & 0x7fffffffu));
    v[j] = byte[j] == 255u ? 0.f : v[j] * mx_inverse(byte[j]);
    if (lane == j) mine = byte[j];
  }
  if (FMT == THA_MX_E2M1) {
    uint8_t* at = static_cast<uint8_t*>(y.codes) + (size_t)n * (padded / 2) + col / 2;
#pragma unroll
    for (int j = 0; j < C; j++) {
      const float next = __shfl_down_sync(THA_FULL_MASK, v[j], 1);
      if (!(lane & 1) && j < count) at[j * (padded / 2)] = (uint8_t)mx_e2m1x2(v[j], next);
    }
  } else {
    uint8_t* at = static_cast<uint8_t*>(y.codes) + (size_t)n * padded + col;
#pragma unroll
    for (int j = 0; j < C; j++)
      if (j < count) at[j * padded] = (uint8_t)mx_e4m3x2(v[j], 0.f);
  }
  if (lane < min(C, count)) y.scales[mx_scale_at(n + lane, col / MX_TILE, (int)(padded / MX_TILE)) + (col / MX_BLOCK & 3)] = (uint8_t)mine;
}
// 1 / (1 + e^-z) without a branch: divisions and expf in full precision leave the straight line for their rare cases, which keeps sixteen of them from running side by side (100 rows x
// [2 x 4608, 1024] 24.9 us).  -z log2 e in two parts, so that the power is good to 2^-22 at any z; the reciprocal to 1 unit.  Beyond +-200 it is 1 or 0, whatever gelu's cube has become.
__device__ __forceinline__ float mg_sigmoid(float z) {
  z = fminf(fmaxf(z, -200.f), 200.f);
  const float hi = -1.44269504f * z, lo = fmaf(-1.44269504f, z, -hi) - 1.92596303e-8f * z;
  const float e = hyb_ex2(hi), more = e < INFINITY ? fmaf(e, 0.693147181f * lo, e) : e;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + more));
  return r;
}
// x, at most and at least a limit, as fminf and fmaxf have them but for what is no number: that stays none
__device__ __forceinline__ float mg_most(float x, float limit) { return x > limit ? limit : x; }
__device__ __forceinline__ float mg_least(float x, float limit) { return x < limit ? limit : x; }
// hyb_act_value, its gated ones by the sigmoid above: 0.5 (1 + tanh t) is the sigmoid of 2 t.  Every one of them keeps NaN: of a block that is none, of a sum that a kernel gave up.
template <int ACT>
__device__ __forceinline__ float mg_act_value(float g, float u, float limit, float alpha) {
  if (ACT == THA_ACT_SILU_GLU) return g * mg_sigmoid(g) * u;
  if (ACT == THA_ACT_GELU_TANH_GLU) return g * mg_sigmoid(1.5957691216057308f * (g + 0.044715f * g * g * g)) * u;
  if (ACT == THA_ACT_GLU_CLAMPED) {
    const float gc = mg_most(g, limit);
    return gc * mg_sigmoid(alpha * gc) * (mg_most(mg_least(u, -limit), limit) + 1.0f);
  }
  if (ACT == THA_ACT_RELU2) {
    const float t = mg_least(u, 0.f);
    return t * t;
  }
  return hyb_act_value(ACT, g, u, limit, alpha);
}
template <int ACT, int G, int C>
__device__ __forceinline__ void mg_act(const float (&g)[G], float (&x)[C], bool there, float limit, float alpha) {
#pragma unroll
  for (int j = 0; j < C; j++) x[j] = there ? mg_act_value<ACT>(g[j], x[j], limit, alpha) : 0.f;   // what pads the result holds zeros
}
// C sums (g: of the gate) of a weight row that is there or not, through the activation
template <int READ, int G, int C>
__device__ __forceinline__ void mg_activate(const MgP& p, const float (&g)[G], float (&x)[C], bool there) {
  if (READ == MG_UNGATED) {
    if (p.act == THA_ACT_RELU2) mg_act<THA_ACT_RELU2>(x, x, there, p.limit, p.alpha);
    else mg_act<THA_ACT_XIELU>(x, x, there, p.limit, p.alpha);
  } else if (READ == MG_GATED) {
    if (p.act == THA_ACT_SILU_GLU) mg_act<THA_ACT_SILU_GLU>(g, x, there, p.limit, p.alpha);
    else if (p.act == THA_ACT_GELU_TANH_GLU) mg_act<THA_ACT_GELU_TANH_GLU>(g, x, there, p.limit, p.alpha);
    else mg_act<THA_ACT_GLU_CLAMPED>(g, x, there, p.limit, p.alpha);
  }
}
// C results of activation rows n .. (`count` of them there) and weight row `row`, a warp's rows neighbours from a multiple of 32 on.  All lanes of the warp, which may leave one
// by one: what follows for the whole of it (tcgen05.ld, the cluster's barrier) has a __syncwarp ahead.
template <int READ, int C>
__device__ __forceinline__ void mg_store(const MgP& p, long long padded, int n, int count, int row, float (&x)[C]) {
  if (READ == MG_PLAIN) {
    if (row >= p.M) return;
    if (p.bf16) {
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + (size_t)n * p.ldo + row;
#pragma unroll
      for (int j = 0; j < C; j++, o += p.ldo)
        if (j < count) hyb_store(o, x[j]);
    } else {
      float* o = static_cast<float*>(p.out) + (size_t)n * p.ldo + row;
#pragma unroll
      for (int j = 0; j < C; j++, o += p.ldo)
        if (j < count) *o = x[j];
    }
  } else if (p.y.format == THA_MX_E2M1) {
    mg_store_blocks<THA_MX_E2M1>(p.y, n, count, row, padded, x);
  } else {
    mg_store_blocks<THA_MX_E4M3>(p.y, n, count, row, padded, x);
  }
}

// ranks > 1: the blocks of a cluster take a share of the tile's stages each, leave their partial tiles in shared memory and sum each other's, ranks in ascending order.
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
  uint64_t* mmadone = accum + 1;                                            // all MMAs complete, where a wait was given up
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mmadone + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)blockIdx.x % p.ranks, item = (int)blockIdx.x / p.ranks;
  const int tile = item / p.ny, row0 = tile * TC_BM, n0 = (item - tile * p.ny) * NT;
  const int kb0 = rank * p.share, nkb = max(0, min((p.across + CH - 1) / CH - kb0, p.share));

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::NST; s++) { tc_mbar_init(&full[s], 1); tc_mbar_init(&empty[s], 1); }
    tc_mbar_init(accum, 1);
    tc_mbar_init(mmadone, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 0 && lane < 3) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &mw0 : lane == 1 ? &mx : &mw1) : "memory");
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(tmem_slot)), "r"(S::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_sf = tmem + S::ACC_COLS;
  pdl_trigger();
  if (warp == 0 && tc_elect()) {
    // the first weights into L2 while the kernel ahead ends: nothing is read of them, so that it may still be writing them
    for (int i = 0; i < min(nkb, S::NST); i++) {
      mg_prefetch(&mw0, (kb0 + i) * (KIND == MG_F4 ? KB / 2 : KB), row0);
      if (WT == 2) mg_prefetch(&mw1, (kb0 + i) * (KIND == MG_F4 ? KB / 2 : KB), row0);
    }
  }
  pdl_wait();

  if (warp == 0) {
    if (tc_elect()) {
      for (int i = 0; i < nkb; i++) {
        const int s = i % S::NST;
        if (i >= S::NST && !tc_mbar_wait(&empty[s], ((i / S::NST) & 1u) ^ 1u, abort_flag)) { tc_drain(full, S::NST, i); break; }
        const int t0 = (kb0 + i) * CH, chunks = min(CH, p.across - t0);              // scale tiles of this stage: one in an odd matrix's last stage
        unsigned char* st = smem + s * S::STAGE;
        unsigned char* sw = st + S::W_BYTES + S::X_BYTES;
        const uint32_t some = (uint32_t)(chunks * MX_TILE_BYTES);
        tc_mbar_expect_tx(&full[s], p.w_bytes + p.x_bytes + (WT + 1) * some);
        tc_tma_2d(st, &mw0, (kb0 + i) * (KIND == MG_F4 ? KB / 2 : KB), row0, &full[s]);
        if (WT == 2) tc_tma_2d(st + TC_BM * 128, &mw1, (kb0 + i) * (KIND == MG_F4 ? KB / 2 : KB), row0, &full[s]);
        tc_tma_2d(st + S::W_BYTES, &mx, (kb0 + i) * (KIND == MG_F4 ? KB / 2 : KB), n0, &full[s]);
        tc_bulk(sw, p.sw0 + mx_scale_at(row0, t0, p.across), some, &full[s]);
        if (WT == 2) tc_bulk(sw + S::SC_BYTES, p.sw1 + mx_scale_at(row0, t0, p.across), some, &full[s]);
        tc_bulk(sw + WT * S::SC_BYTES, p.sx + mx_scale_at(n0 & ~127, t0, p.across), some, &full[s]);
      }
    }
  } else if (warp == 1) {
    if (tc_elect()) {
      bool ok = true;
      const uint32_t shift = NT == 64 ? (uint32_t)(n0 & 64) / 32 : 0u;        // a tile of 64 may be the second half of a tile of scales (narrower tiles are alone)
      for (int i = 0; i < nkb; i++) {
        const int s = i % S::NST;
        if (!tc_mbar_wait(&full[s], (i / S::NST) & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const int chunks = min(CH, p.across - (kb0 + i) * CH);
        const uint32_t st = tc_smem_u32(smem + s * S::STAGE), sc = st + S::W_BYTES + S::X_BYTES;
        // a stage has TMEM columns of its own for its scales: the MMAs that read their last contents have completed when the stage was filled again
        const uint32_t sf = tmem_sf + (uint32_t)(s * S::SET);
        for (int c = 0; c < chunks; c++) {
#pragma unroll
          for (int t = 0; t <= WT; t++) mg_copy_scales(sf + (uint32_t)(4 * (c * (WT + 1) + t)), sc + (uint32_t)(t * S::SC_BYTES + c * MX_TILE_BYTES));   // the matrices', the activation rows'
        }
        const uint64_t adesc = tc_smem_desc(st), bdesc = tc_smem_desc(st + S::W_BYTES);
#pragma unroll
        for (int k = 0; k < 4; k++) {                // 32 bytes of codes each: 2 descriptor units
          const int c = KIND == MG_F4 ? k >> 1 : 0, id = KIND == MG_F4 ? 2 * (k & 1) : k;
          if (c < chunks) {
            const uint32_t at = sf + (uint32_t)(4 * c * (WT + 1));
#pragma unroll
            for (int w = 0; w < WT; w++)
              mg_mma<KIND>(tmem + (uint32_t)(w * NT), adesc + (uint64_t)(1024 * w + 2 * k), bdesc + (uint64_t)(2 * k), p.idesc | (uint32_t)id << 4 | (uint32_t)id << 29, at + 4 * w,
                           at + 4 * WT + shift, (uint32_t)((i | k) != 0));
          }
        }
        tc_commit(&empty[s]);
      }
      if (ok && nkb > 0) tc_commit(accum);
      if (!ok) {                         // MMAs that have been issued end ahead of the block
        tc_commit(mmadone);
        tc_drain(mmadone, 1, 1);
      }
    }
  }
  __syncwarp();
  const int cols = min(NT, p.N - n0);
  const long long padded = READ == MG_PLAIN ? 0 : mx_padded(p.M);
  float* part = reinterpret_cast<float*>(smem);      // [WT][NT][128], over the ring once its last MMA has read it
  if (NT > 16 || warp >= 4) {                        // sixteen columns at a time, dealt to two warps of a lane quarter: warps 4-7 and, done with theirs, 0-3
    const int q = warp & 3, r = q * 32 + lane;                               // the thread's weight row of the tile
    const bool ok = nkb > 0 && tc_mbar_wait_warp(accum, 0u, abort_flag);
    tc_fence_after();
    const uint32_t ta = tmem + ((uint32_t)(q * 32) << 16);
    const float none = nkb > 0 ? __uint_as_float(0x7fc00000u) : 0.f;         // given up: no number; no share of the stages: nothing to add
#pragma unroll 1
    for (int c = warp >= 4 ? 0 : 16; c < cols; c += NT > 16 ? 32 : 16) {
      uint32_t v[16], g[16];
      if (ok) {
        tc_tmem_ld16(ta + (uint32_t)c, READ == MG_GATED ? g : v);
        if (READ == MG_GATED) tc_tmem_ld16(ta + (uint32_t)(NT + c), v);
        tc_wait_ld();
      }
      float x[16], gate[16];
#pragma unroll
      for (int j = 0; j < 16; j++) {
        x[j] = ok ? __uint_as_float(v[j]) : none;
        gate[j] = READ == MG_GATED && ok ? __uint_as_float(g[j]) : none;
      }
      if (p.ranks == 1) {
        mg_activate<READ>(p, gate, x, row0 + r < p.M);
        mg_store<READ>(p, padded, n0 + c, cols - c, row0 + r, x);
        __syncwarp();
      } else {
#pragma unroll
        for (int j = 0; j < 16; j++) {
          part[(c + j) * TC_BM + r] = READ == MG_GATED ? gate[j] : x[j];
          if (READ == MG_GATED) part[(NT + c + j) * TC_BM + r] = x[j];
        }
      }
    }
    tc_fence_before();
  }
  if (p.ranks > 1) {
    __syncthreads();
    if (*((volatile int*)abort_flag)) {              // copies that were under way have landed by now, over the partial tile maybe
      for (int i = threadIdx.x; i < WT * NT * TC_BM; i += MG_THREADS) part[i] = __uint_as_float(0x7fc00000u);
      __syncthreads();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    // this rank's columns of the tile, C neighbours at a time; half of the threads take one such group at a time, a thread a weight row
    constexpr int C = NT == 16 ? 2 : 4;
    const int r = threadIdx.x & (TC_BM - 1);
    const uint32_t base = tc_smem_u32(part) + (uint32_t)r * 4u;
    for (int c = C * (rank + p.ranks * (int)(threadIdx.x >> 7)); c < cols; c += 2 * C * p.ranks) {
      float sum[WT][C];
#pragma unroll
      for (int j = 0; j < C; j++) sum[0][j] = sum[WT - 1][j] = 0.f;
      for (int z = 0; z < p.ranks; z++) {
        uint32_t a;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(base + (uint32_t)(c * TC_BM * 4)), "r"(z));
        float v[WT][C];
#pragma unroll
        for (int w = 0; w < WT; w++)
#pragma unroll
          for (int j = 0; j < C; j++) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[w][j]) : "r"(a + (uint32_t)((w * NT + j) * TC_BM * 4)) : "memory");
#pragma unroll
        for (int w = 0; w < WT; w++)
#pragma unroll
          for (int j = 0; j < C; j++) sum[w][j] += v[w][j];
      }
      mg_activate<READ>(p, sum[0], sum[WT - 1], row0 + r < p.M);
      mg_store<READ>(p, padded, n0 + c, cols - c, row0 + r, sum[WT - 1]);
      __syncwarp();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // a block's shared memory stays until every rank has read it
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLS));
  }
  if (threadIdx.x == 0 && *abort_flag && p.error_flag) *((volatile int*)p.error_flag) = 1;
}

// ---- prompts: pairs of blocks ------------------------------------------------------------------------------------------------
// A pair (cta_group::2) takes 256 weight rows (of each of two matrices for a gated activation) x NT activation rows: each block has 128 of the weight rows and half of the activation rows
// in its shared memory, an MMA reads both halves, and each block's TMEM gets 128 lanes of results.  Persistent: 74 pairs walk the items with running counters.  The accumulators take
// 256 of TMEM's 512 columns and scales the others, so there is one set of them: eight warps fetch an item's sums into registers, 128 a thread, and hand the columns back before they do
// anything with them; activation, quantising and stores run behind the next item's MMAs.  2048 rows x [12288, 4096] e4m3 80 us with random codes of one sign (2.6 PFLOP/s), 97 with those
// of normal numbers, 3333 rows x [11008, 4096] e2m1 68 and 75, 2048 rows x [2 x 11008, 4096] with silu 132 and 165: bound by power (960 to 1000 W at 1475 MHz), the tensor pipe at 54 to 65 % of
// the cycles, some 43 bytes a cycle and SM from L2.
// Scales: a block's TMEM holds those of its own weight rows and of all NT activation rows.  NT is a multiple of 128, so that an item's scales start with a tile of them: an MMA's scale
// address has to be even (in columns of 32 rows), and a tile of 96 activation rows would start at an odd one every other time.
template <int KIND, int READ>
struct MgpSmem {
  static constexpr int WT = READ == MG_GATED ? 2 : 1, NT = 256 / WT, XT = NT / 128, CH = KIND == MG_F4 ? 2 : 1;
  static constexpr int W_BYTES = WT * TC_BM * 128, X_BYTES = NT / 2 * 128, SC_BYTES = CH * MX_TILE_BYTES;
  static constexpr int STAGE = (W_BYTES + X_BYTES + (WT + XT) * SC_BYTES + 1023) / 1024 * 1024;
  static constexpr int SET = CH * 4 * (WT + XT);
  static constexpr int NST = (TC_SMEM_LIMIT - 2048) / STAGE;           // a stage has TMEM columns of its own for its scales
  static constexpr int TOTAL = NST * STAGE + 1024 + (3 * NST + 3) * 8 + 64;
  static_assert(NST >= 3 && TOTAL <= TC_SMEM_LIMIT && 256 + NST * SET <= 512, "a stage is too large");
};
constexpr int MGP_THREADS = 384;
// Activation rows of an item: NT, or what is left rounded up; each block has half of them
template <int NT>
__device__ __forceinline__ int mgp_width(int left) { return min(NT, (left + 31) & ~31); }

__device__ __forceinline__ void mgp_copy_scales(uint32_t taddr, uint32_t saddr) {   // in both blocks, each from its own shared memory
  uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}
template <int KIND>
__device__ __forceinline__ void mgp_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  if (KIND == MG_F8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}

template <int KIND, int READ>
__global__ void __launch_bounds__(MGP_THREADS, 1)
mx_gemm_pair_kernel(const __grid_constant__ CUtensorMap mw0, const __grid_constant__ CUtensorMap mw1, const __grid_constant__ CUtensorMap mx, const __grid_constant__ MgP p) {
  using S = MgpSmem<KIND, READ>;
  constexpr int WT = S::WT, NT = S::NT, XT = S::XT, CH = S::CH, KC = 128;          // KC: a stage's extent along k in the tensor maps' elements (bytes or values)
  extern __shared__ unsigned char tc_smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tc_smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::NST * S::STAGE);   // stage landed
  uint64_t* peer = full + S::NST;        // rank 0: ... in rank 1
  uint64_t* empty = peer + S::NST;       // the MMAs that read it have completed
  uint64_t* accum = empty + S::NST;      // sums of an item complete
  uint64_t* accfree = accum + 1;         // rank 0: ... and fetched in both blocks
  uint64_t* mmadone = accfree + 1;       // all MMAs complete, where a wait was given up
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mmadone + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int nkb = (p.across + CH - 1) / CH;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::NST; s++) { tc_mbar_init(&full[s], 1); tc_mbar_init(&peer[s], 1); tc_mbar_init(&empty[s], 1); }
    tc_mbar_init(accum, 1);
    tc_mbar_init(accfree, 16);
    tc_mbar_init(mmadone, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 0 && lane < 3) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &mw0 : lane == 1 ? &mx : &mw1) : "memory");
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // both blocks' barriers are there
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_sf = tmem + 256;
  hyb_pdl_enter();

  int gb = 0;                            // stages so far
  bool ok = true;
  if (warp == 0) {
    if (tc_elect()) {
      int sent = -1;                     // stages that have been asked for, where the producer has given up
      for (int it = pair; it < p.n_items && ok; it += n_pairs) {
        const int tile = it / p.ny, row0 = tile * 256 + rank * TC_BM, n0 = (it - tile * p.ny) * NT;
        const int half = rank * (mgp_width<NT>(p.N - n0) / 2);
        const int srow = min(row0, (p.M - 1) / MX_TILE * MX_TILE);          // a tile that lies wholly behind the matrix takes the last one's scales: its results go nowhere
        const int xt = (min(NT, p.N - n0) + 127) / 128;                     // tiles of scales that the item's activation rows touch
        for (int i = 0; i < nkb; i++) {
          const int g = gb + i, s = g % S::NST;
          if (g >= S::NST && !tc_mbar_wait(&empty[s], ((g / S::NST) & 1u) ^ 1u, abort_flag)) { ok = false; sent = g; break; }
          const int t0 = i * CH, chunks = min(CH, p.across - t0);
          unsigned char* st = smem + s * S::STAGE;
          unsigned char* sw = st + S::W_BYTES + S::X_BYTES;
          unsigned char* sx = sw + WT * S::SC_BYTES;
          const uint32_t some = (uint32_t)(chunks * MX_TILE_BYTES);
          tc_mbar_expect_tx(&full[s], p.w_bytes + p.x_bytes + (WT + xt) * some);
          tc_tma_2d(st, &mw0, i * KC, row0, &full[s]);
          if (WT == 2) tc_tma_2d(st + TC_BM * 128, &mw1, i * KC, row0, &full[s]);
          tc_tma_2d(st + S::W_BYTES, &mx, i * KC, n0 + half, &full[s]);
          tc_bulk(sw, p.sw0 + mx_scale_at(srow, t0, p.across), some, &full[s]);
          if (WT == 2) tc_bulk(sw + S::SC_BYTES, p.sw1 + mx_scale_at(srow, t0, p.across), some, &full[s]);
          for (int x = 0; x < xt; x++) tc_bulk(sx + x * S::SC_BYTES, p.sx + mx_scale_at(n0 + 128 * x, t0, p.across), some, &full[s]);
        }
        gb += nkb;
      }
      if (!ok) tc_drain(full, S::NST, sent);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (tc_elect()) {
      int n_it = 0;
      for (int it = pair; it < p.n_items && ok; it += n_pairs, n_it++) {
        if (rank) {                      // what has landed here is told to rank 0, whose MMAs read it
          for (int i = 0; i < nkb; i++) {
            const int g = gb + i, s = g % S::NST;
            if (!tc_mbar_wait(&full[s], (g / S::NST) & 1u, abort_flag)) { ok = false; break; }
            tc_pair_arrive(&peer[s]);
          }
          gb += nkb;
          continue;
        }
        const uint32_t idesc = p.idesc | (uint32_t)(mgp_width<NT>(p.N - it % p.ny * NT) >> 3) << 17;
        if (n_it >= 1 && !tc_mbar_wait(accfree, (unsigned)(n_it - 1) & 1u, abort_flag)) { ok = false; break; }
        for (int i = 0; i < nkb; i++) {
          const int g = gb + i, s = g % S::NST;
          if (!tc_mbar_wait(&full[s], (g / S::NST) & 1u, abort_flag) || !tc_mbar_wait(&peer[s], (g / S::NST) & 1u, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const int chunks = min(CH, p.across - i * CH);
          const uint32_t st = tc_smem_u32(smem + s * S::STAGE), sw = st + S::W_BYTES + S::X_BYTES, sx = sw + WT * S::SC_BYTES;
          const uint32_t sf = tmem_sf + (uint32_t)(s * S::SET);
          for (int c = 0; c < chunks; c++) {
#pragma unroll
            for (int w = 0; w < WT; w++) mgp_copy_scales(sf + (uint32_t)(4 * (c * (WT + XT) + w)), sw + (uint32_t)(w * S::SC_BYTES + c * MX_TILE_BYTES));
#pragma unroll
            for (int x = 0; x < XT; x++) mgp_copy_scales(sf + (uint32_t)(4 * (c * (WT + XT) + WT + x)), sx + (uint32_t)(x * S::SC_BYTES + c * MX_TILE_BYTES));
          }
          const uint64_t adesc = tc_smem_desc(st), bdesc = tc_smem_desc(st + S::W_BYTES);
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const int c = KIND == MG_F4 ? k >> 1 : 0, id = KIND == MG_F4 ? 2 * (k & 1) : k;
            if (c < chunks) {
              const uint32_t at = sf + (uint32_t)(4 * c * (WT + XT));
#pragma unroll
              for (int w = 0; w < WT; w++)
                mgp_mma<KIND>(tmem + (uint32_t)(w * NT), adesc + (uint64_t)(1024 * w + 2 * k), bdesc + (uint64_t)(2 * k), idesc | (uint32_t)id << 4 | (uint32_t)id << 29, at + 4 * w,
                              at + 4 * WT, (uint32_t)((i | k) != 0));
            }
          }
          tc_pair_commit(&empty[s]);
        }
        if (ok) tc_pair_commit(accum);
        gb += nkb;
      }
      if (!ok && rank == 0) {            // MMAs that have been issued end ahead of the blocks
        tc_pair_commit(mmadone);
        tc_drain(mmadone, 1, 1);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    constexpr int HC = NT / 2;                                         // columns of a warp
    const int q = warp & 3, half = (warp - 4) >> 2;
    const long long padded = READ == MG_PLAIN ? 0 : mx_padded(p.M);
    int n_it = 0;
    for (int it = pair; it < p.n_items; it += n_pairs, n_it++) {
      const int tile = it / p.ny, row0 = tile * 256 + rank * TC_BM, n0 = (it - tile * p.ny) * NT + half * HC;
      const int cols = row0 < p.M ? p.N - n0 : 0;
      if (ok) ok = tc_mbar_wait_warp(accum, (unsigned)n_it & 1u, abort_flag);
      tc_fence_after();
      const uint32_t ta = tmem + (uint32_t)(half * HC) + ((uint32_t)(q * 32) << 16);
      float x[HC], gate[WT == 2 ? HC : 16];
      if (ok) {
#pragma unroll
        for (int c = 0; c < HC; c += 32) {
          tc_tmem_ld32(ta + (uint32_t)((WT - 1) * NT + c), *reinterpret_cast<uint32_t(*)[32]>(x + c));
          if (WT == 2) tc_tmem_ld32(ta + (uint32_t)c, *reinterpret_cast<uint32_t(*)[32]>(gate + c));
        }
        tc_wait_ld();
      } else {
#pragma unroll
        for (int c = 0; c < HC; c++) {
          x[c] = __uint_as_float(0x7fc00000u);
          if (WT == 2) gate[c] = x[c];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) tc_pair_arrive(accfree);
      if (cols <= 0) continue;
      mg_activate<READ>(p, gate, x, row0 + q * 32 + lane < p.M);
#pragma unroll
      for (int c = 0; c < HC; c += 16)
        if (c < cols) mg_store<READ>(p, padded, n0 + c, cols - c, row0 + q * 32 + lane, *reinterpret_cast<float(*)[16]>(x + c));
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // a block's barriers and shared memory stay until both are done
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
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

// Which form a product takes, by its tiles of 128 weight rows, activation rows and stages along K (us on cold weights, a call behind the other).
// Tiles of 16, 32 or 64 activation rows as long as all of them run at once, on two blocks an SM (one for a gated activation, whose stages hold two matrices); pairs beyond:
//   192 rows x [12288, 4096] e4m3: 288 tiles of 64 14.4, pairs 16.5; 256 rows, 384 tiles 24.6, pairs 17.4      e2m1 10.6 / 11.9, 17.1 / 12.5
//   gated [2 x 4096, 4096]: 256 rows, 128 tiles 19.2, pairs 21.9; [2 x 12288, 4096]: 64 rows, 96 tiles 20.6, pairs 24.9; 128 rows, 192 tiles 38.2, pairs 26.0
// Tiles of 128 rows were between the two or behind both everywhere (256 rows x [4096, 4096]: 64 11.1, 128 12.1, pairs 15.0), 32 rows take 5 % less time than 64 with so few.
// The blocks of a cluster share a tile's stages: 8, 4, 3 or 2 of them while the SMs hold them, where there are stages enough to share:
//   1 row x [4096, 11008], 86 stages, at 1 / 2 / 4 / 8 blocks 22.1 / 14.0 / 9.6 / 8.5;  [4096, 4096], 32 stages 9.7 / 7.4 / 5.8 / 5.8;  [2048, 2048], 16 stages 5.9 / 5.2 / 4.4 / 4.2;
//   16 rows x [1024, 1024], 8 stages 3.6 / 4.3 / 3.9 / 3.8;  128 rows x [4096, 4096] 11.9 / 10.5 / 9.3;  16 rows x [12288, 4096] 10.7 / 9.9 / 13.9
//   16 rows x [2 x 11008, 4096] 20.2 / 15.6 / (3) 14.0;
//   a gated one's blocks share the activation, too: 16 rows x [2 x 1024, 1024] - / 5.5 / 4.7 / 4.8
// Clusters have to fit the SMs of a GPC together: seven eighths of the places are counted (96 tiles x 3 blocks on 296 places: 15.7 where 2 take 9.9).
struct MgForm { int nt, ranks; };                  // nt 0: pairs
MgForm mg_form(int read, int tiles, int rows, int stages) {
  const int sms = sm_budget(), nt = rows <= 16 ? 16 : rows <= 32 && read != MG_GATED ? 32 : 64;
  const int places = read == MG_GATED && nt == 64 ? sms : 2 * sms;
  const long long items = (long long)tiles * ceil_div(rows, nt);
  if (items > places) return {rows > 64 ? 0 : nt, 1};
  for (int ranks = stages >= 64 || (read == MG_GATED && nt == 16 && stages >= 16) ? 8 : 4; ranks > 1; ranks = ranks == 8 ? 4 : ranks - 1)
    if (stages >= (read == MG_GATED ? 8 : 16) && items * ranks * 8 <= (long long)places * 7) return {nt, ranks};
  return {nt, 1};
}

struct MgArgs { const tha_mx_t *A, *W0, *W1; MgP p; };

template <int KIND, int NT, int READ>
int mg_launch(cudaStream_t s, const MgArgs& a, int ranks) {
  using S = MgSmem<KIND, NT, READ>;
  MgP p = a.p;
  CUtensorMap mw0, mw1, mx;
  int wb = 0;
  THA_TRY_RC(mg_map(KIND, a.W0, TC_BM, &mw0, &wb));
  mw1 = mw0;
  if (S::WT == 2) THA_TRY_RC(mg_map(KIND, a.W1, TC_BM, &mw1, &wb));
  THA_TRY_RC(mg_map(KIND, a.A, NT, &mx, &p.x_bytes));
  p.w_bytes = S::WT * wb;
  p.idesc = mg_idesc(KIND, TC_BM, NT);
  p.ny = ceil_div(p.N, NT);
  const long long items = (long long)ceil_div(p.M, TC_BM) * p.ny;      // 2^23 at most: mg_form sends no more here than the SMs have places for, or 64 activation rows
  const int stages = ceil_div(p.across, S::CH);
  p.ranks = ranks;
  p.share = ceil_div(stages, p.ranks);
  auto k = mx_gemm_kernel<KIND, NT, READ>;
  static std::atomic<unsigned long long> asked{0};
  THA_TRY_RC(mx_room(k, S::TOTAL, &asked));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3((unsigned)(items * p.ranks)); cfg.blockDim = dim3(MG_THREADS); cfg.dynamicSmemBytes = S::TOTAL; cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = pdl_enabled() ? 2 : 1;
  count_launch();
  THA_CUDA_OK(cudaLaunchKernelEx(&cfg, k, mw0, mw1, mx, p));
  trace_launch(reinterpret_cast<const void*>(k), s);
  return THA_STATUS_SUCCESS;
}
template <int KIND, int READ>
int mgp_launch(cudaStream_t s, const MgArgs& a) {
  using S = MgpSmem<KIND, READ>;
  MgP p = a.p;
  CUtensorMap mw0, mw1, mx;
  int wb = 0;
  THA_TRY_RC(mg_map(KIND, a.W0, TC_BM, &mw0, &wb));
  mw1 = mw0;
  if (S::WT == 2) THA_TRY_RC(mg_map(KIND, a.W1, TC_BM, &mw1, &wb));
  THA_TRY_RC(mg_map(KIND, a.A, S::NT / 2, &mx, &p.x_bytes));
  p.w_bytes = S::WT * wb;
  p.idesc = mg_idesc(KIND, 2 * TC_BM, 0);
  p.ny = ceil_div(p.N, S::NT);
  p.n_items = ceil_div(p.M, 2 * TC_BM) * p.ny;
  const int pairs = max(1, sm_budget() / 2);
  auto k = mx_gemm_pair_kernel<KIND, READ>;
  static std::atomic<unsigned long long> asked{0};
  THA_TRY_RC(mx_room(k, S::TOTAL, &asked));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(2u * (unsigned)min(pairs, p.n_items)); cfg.blockDim = dim3(MGP_THREADS); cfg.dynamicSmemBytes = S::TOTAL; cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = pdl_enabled() ? 2 : 1;
  count_launch();
  THA_CUDA_OK(cudaLaunchKernelEx(&cfg, k, mw0, mw1, mx, p));
  trace_launch(reinterpret_cast<const void*>(k), s);
  return THA_STATUS_SUCCESS;
}
template <int KIND, int READ>
int mg_width(cudaStream_t s, const MgArgs& a) {
  const MgForm f = mg_form(READ, ceil_div(a.p.M, TC_BM), a.p.N, ceil_div(a.p.across, KIND == MG_F4 ? 2 : 1));
  if (f.nt == 0) return mgp_launch<KIND, READ>(s, a);
  if (f.nt == 16) return mg_launch<KIND, 16, READ>(s, a, f.ranks);
  if constexpr (READ != MG_GATED) if (f.nt == 32) return mg_launch<KIND, 32, READ>(s, a, f.ranks);
  return mg_launch<KIND, 64, READ>(s, a, f.ranks);
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
int mg_fill(MgArgs* a, const tha_mx_t* A, const tha_mx_t* W0, const tha_mx_t* W1, const char* who) {
  if ((long long)ceil_div(W0->rows, 2 * TC_BM) * ceil_div(A->rows, W1 ? 128 : 256) > 0x3fffffff) return mx_refuse(who, "too many results for one call");   // items of pairs are counted in 31 bits
  a->A = A; a->W0 = W0; a->W1 = W1;
  a->p.M = W0->rows; a->p.N = A->rows;
  a->p.across = (int)(mx_padded(A->cols) / MX_TILE);
  a->p.sw0 = W0->scales; a->p.sw1 = W1 ? W1->scales : nullptr; a->p.sx = A->scales;
  return mx_error_flag(&a->p.error_flag);
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
  THA_TRY_RC(mg_fill(&a, A, W, nullptr, who));
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
  THA_TRY_RC(mg_fill(&a, A, gated ? W_gate : W_up, gated ? W_up : nullptr, who));
  a.p.y = *out; a.p.act = act; a.p.limit = limit; a.p.alpha = alpha;
  return gated ? mg_run<MG_GATED>((cudaStream_t)stream, a) : mg_run<MG_UNGATED>((cudaStream_t)stream, a);
}
