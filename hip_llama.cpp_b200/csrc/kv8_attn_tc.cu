// Softmax attention of prompt portions over the cache in 8 bits on the 5th-generation tensor cores (tcgen05 + TMEM).  kv8_attn.cu keeps single rows and the portions that take longer
// here (k8_long_pays).
//
// Codes are fp16 numbers.  A step's visible keys and values are turned into fp16 once (kv8_stage_kernel), without scales, into scratch that holds tiles as they will lie in shared
// memory, from where bulk copies fetch them: warps of the block that did it themselves, tile by tile and again for every 256 rows, took half of the SM's issue slots (8000
// instructions of 32 lanes a tile instead of 3500).  K's scale belongs to 16 or more neighbouring keys and multiplies their scores, V's multiplies their weights, relative to a power of two
// that all of a row's weights share.  q is brought to [2^14, 2^15) by a power of two a row and rounded to one fp16 (bf16 results) or two (SPLIT: fp32 results or fp32 scores asked for, 22 bits; weights
// likewise), each product fp32.  A row's power of two is that of the scales that it sees itself: with one for the block's rows, a row lost as many bits as the scale of a block
// hidden from it was larger.
// A block takes 128 pairs of one key/value head (with two fp16 an operand and heads beyond 64 channels 256, two groups of 128 that share every tile) and a run of tiles of 64 keys.
// Ten warps (nineteen):
//   0 .. 7 (.. 15)   softmax of a group, a row for two threads of 32 keys each: scores out of TMEM, factor, mask, weights back into the same TMEM columns as the A operand of the
//                    second product.  With a thread a row (two warps on a scheduler) a tile's chain of waits, maximum, exponentials and stores took twice as long.
//   8 (16)           one thread asks for tiles
//   9 (17, 18)       one thread issues the products of a group: weights x values of tile j, then scores of tile j + 2 into the columns of those weights (with one
//                    thread for two groups, its waits and commits left the tensor cores idle for half of a tile's 2000 cycles); the first of them allocates TMEM
// The accumulator stays in TMEM.  The tensor cores cut off what their fp32 sums cannot hold, so that an error grows with the number of sums: 100 rows behind 3900 keys were 8.6e-6
// off with two fp16 an operand.  SPLIT therefore adds the accumulators of runs of 8 tiles (64 sums) in fp32, in local memory.  It is rescaled only where a row's maximum has grown
// by more than 2^8 since its reference was taken (weights are at most 2^15 then: fp16 holds them), or V's scales outgrow theirs.
//
// Bound: the tensor cores' shared-memory operand and the softmax together, 2100 cycles for 256 rows of a tile where the products alone are 1320 (a score product of 128 x 64 x 16 reads 6 KB of
// shared memory in 50 cycles, one of weights x values takes 65).  Two bf16 prompts of 777 and 2048 rows, 32 heads of 128: 92 us with 10 to 20 of staging, 430 TFLOP/s of the visible
// pairs; one fp32 prompt of 1024 (twice the products): 62 us.
#include "gemm_tc.h"
#include "kv8.cuh"
#include "tc_common.cuh"
#include "workspace.h"

namespace tha {

constexpr int KT_KEYS = 64, KT_ROWS = 128;
// Groups of 128 rows a block has: one, and two blocks share an SM, where shared memory allows that (one's beginning and end run under the other's tiles; with one block of two groups
// they were a fifth of the time), else two
__host__ __device__ constexpr int kt_groups(bool split, int DT) { return split && DT == 128 ? 2 : 1; }
__host__ __device__ constexpr int kt_threads(bool split, int DT) { return 32 * (9 * kt_groups(split, DT) + 1); }
constexpr float KT_UP = 7.0f, KT_SLACK = 8.0f;
constexpr int KT_RUN = 8;      // SPLIT: tiles that one accumulator sums
constexpr long long KT_MOST_STAGED = 1ll << 30;   // bytes of scratch beyond which a step takes the form that needs none
constexpr int KT_SCALES = 8;   // tiles whose scales are kept: K of tile j + 8 comes into a ring of four behind the scores of tile j + 4, those behind the weights of tile j + 2
// Staged keys: 32 at a time (a part), per part and head [K, V][64 channels][key][128 bytes swizzled] and the scales of its two 16 keys: (K, K, V, V), K's below 0: they do not exist
__host__ __device__ constexpr int kt_part(int DT) { return 2 * 32 * DT * 2; }

__host__ __device__ constexpr int kt_slots(bool split, int DT) { return DT == 64 ? 4 : split ? 3 : 2; }   // of the ring of K tiles, and of V's
__host__ __device__ constexpr int kt_smem(bool split, int DT) { return (split ? 2 : 1) * kt_groups(split, DT) * KT_ROWS * DT * 2 + 2 * kt_slots(split, DT) * KT_KEYS * DT * 2 + 1024; }

// tc_wait_ld where other work stands between: what is loaded is not touched ahead of it
__device__ __forceinline__ void kt_wait_ld32(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                 "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                 "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]) : : "memory");
}
// whether any thread of the 64 that meet at a barrier says so
__device__ __forceinline__ bool kt_any_of_pair(bool mine, int bar) {
  unsigned any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.aligned.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"((unsigned)mine), "r"(bar) : "memory");
  return any != 0;
}
// kind::f16, fp16 x fp16 -> fp32, M = 128; b_mn: the B operand's N runs along its rows
__device__ __forceinline__ uint32_t kt_idesc(int n, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// Shared-memory descriptors (tc_smem_desc) as their low words; all have the same high word.  What is added to them stays 32-bit arithmetic, and one register less to be made uniform
// for each operand of a product.
constexpr uint32_t KT_DESC_HI = (uint32_t)(1024 >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t kt_desc_k(uint32_t saddr) { return (saddr & 0x3FFFFu) >> 4 | 1u << 16; }
// MN-major B, SWIZZLE_128B: blocks of 64 columns (128 bytes) x 8 rows of K; K groups 1024 bytes apart, column blocks `block` bytes
__device__ __forceinline__ uint32_t kt_desc_mn(uint32_t saddr, uint32_t block) { return (saddr & 0x3FFFFu) >> 4 | (block >> 4) << 16; }
__device__ __forceinline__ void kt_mma(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"((uint32_t)accumulate), "n"(KT_DESC_HI) : "memory");
}
__device__ __forceinline__ void kt_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "r"(b_lo), "r"(idesc), "r"((uint32_t)accumulate), "n"(KT_DESC_HI) : "memory");
}
// Four codes as two fp16 pairs.  int8: channels (0, 2), (1, 3), what is cheapest to take apart: q's channels and the result's are in that order too.
template <int FMT>
__device__ __forceinline__ uint2 kt_half4(uint32_t w) {
  if (FMT == THA_KV8_INT8) return make_uint2(k8_bytes02(w), k8_bytes02(w >> 8));
  return make_uint2(k8_e4m3x2(w & 0xFFFFu), k8_e4m3x2(w >> 16));
}

// Rows, first and last position, and the parts of the keys that any row of sequence `seq` sees: none where it is not this form's.
struct KtSeq { int n, p0; HybTiles parts; };
__device__ __forceinline__ KtSeq kt_seq(const tha_attn_t& a, const tha_rows_t& rows, int seq, int min_rows) {
  const int r0 = rows.seq_first[seq], n = rows.seq_first[seq + 1] - r0;
  KtSeq q = {n, 0, {0, 0, 0, 0}};
  if (n < min_rows) return q;
  q.p0 = rows.pos[r0];
  q.parts = hyb_attn_tiles(a, a.chunk > 0 ? (q.p0 / a.chunk) * a.chunk : 0, q.p0, q.p0 + n - 1);
  return q;
}
// Staged parts ahead of those of `seq`
__device__ __forceinline__ int kt_stage_base(const tha_attn_t& a, const tha_rows_t& rows, int seq, int min_rows) {
  int sum = 0;
  for (int s = threadIdx.x & 31; s < seq; s += 32) sum += kt_seq(a, rows, s, min_rows).parts.n;
  return __reduce_add_sync(THA_FULL_MASK, sum);
}
// The staged part that holds `key`, one of those
__device__ __forceinline__ int kt_part_of(const HybTiles& t, int key) { return key < t.begin + 32 * t.n_a ? (key - t.begin) >> 5 : t.n_a + ((key - t.resume) >> 5); }

// grid (parts of all sequences or fewer, groups of KT_STAGE_HEADS heads), a thread: row t / 8 of a part, 16-byte piece t % 8, all heads' loads on their way at once
constexpr int KT_STAGE_HEADS = 4;
template <int DT, int FMT>
__device__ __forceinline__ bool kt_stage_part(const tha_attn_t& a, const tha_rows_t& rows, const tha_kv8_t& kv, int min_rows, int i, unsigned char* staged, float4* scales) {
  constexpr int PIECES = DT / 16;
  const Kv8Piece pc = kv8_find(rows.n_seqs, i, [&](int s) { return kt_seq(a, rows, s, min_rows).parts.n; });
  if (pc.seq < 0) return false;
  const KtSeq sq = kt_seq(a, rows, pc.seq, min_rows);
  const HybTiles& parts = sq.parts;
  const int slot = rows.seq_slot[pc.seq], last = sq.p0 + sq.n - 1, g0 = blockIdx.y * KT_STAGE_HEADS;
  const int r = threadIdx.x / PIECES, x = threadIdx.x % PIECES, key = (pc.at < parts.n_a ? parts.begin + 32 * pc.at : parts.resume + 32 * (pc.at - parts.n_a)) + (r & 16);
  const int id = key <= last ? kv8_block(kv, slot, key) : -1, in_block = (key & (kv.block_size - 1)) + (r & 15);
  uint4 c[KT_STAGE_HEADS][2];
#pragma unroll
  for (int h = 0; h < KT_STAGE_HEADS; h++) {
    const size_t row = id >= 0 ? kv8_tile(kv, id, a.cache_layer, g0 + h) * kv.block_size + in_block : 0;
    const bool there = id >= 0 && g0 + h < kv.kv_heads;
    c[h][0] = there && 16 * x < kv.dim ? *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(kv.k_pool) + row * kv.dim + 16 * x) : make_uint4(0u, 0u, 0u, 0u);
    c[h][1] = there && 16 * x < kv.vdim ? *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(kv.v_pool) + row * kv.vdim + 16 * x) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int h = 0; h < KT_STAGE_HEADS; h++) {
    if (g0 + h >= kv.kv_heads) break;
    const size_t at = (size_t)i * kv.kv_heads + g0 + h;
    unsigned char* d = staged + at * kt_part(DT) + (x >> 2) * (32 * 128) + r * 128;
#pragma unroll
    for (int side = 0; side < 2; side++) {
      const uint32_t w[4] = {c[h][side].x, c[h][side].y, c[h][side].z, c[h][side].w};
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const uint2 a0 = kt_half4<FMT>(w[2 * y]), a1 = kt_half4<FMT>(w[2 * y + 1]);
        *reinterpret_cast<uint4*>(d + side * (DT / 64) * (32 * 128) + (((2 * (x & 3) + y) ^ (r & 7)) << 4)) = make_uint4(a0.x, a0.y, a1.x, a1.y);
      }
    }
    if (x == 0 && (r & 15) == 0) {
      const size_t tile = id >= 0 ? kv8_tile(kv, id, a.cache_layer, g0 + h) : 0;
      float* s = reinterpret_cast<float*>(scales + at) + (r >> 4);
      s[0] = id >= 0 ? kv.k_scale[tile] : -1.f;
      s[2] = id >= 0 ? kv.v_scale[tile] : 0.f;
    }
  }
  return true;
}
// TURNS: a block may have several parts.  Its 57 registers for 48 are a block less on an SM: two prompts, 24 us for 20.
template <int DT, int FMT, bool TURNS>
__global__ void __launch_bounds__(2 * DT) kv8_stage_kernel(tha_attn_t a, tha_rows_t rows, tha_kv8_t kv, int min_rows, int parts, unsigned char* staged, float4* scales) {
  pdl_wait();
  pdl_trigger();                     // behind the wait: the kernel behind this one reads q without another
  if (!TURNS) {
    kt_stage_part<DT, FMT>(a, rows, kv, min_rows, (int)blockIdx.x, staged, scales);
  } else {
    for (int i = blockIdx.x; i < parts; i += gridDim.x)
      if (!kt_stage_part<DT, FMT>(a, rows, kv, min_rows, i, staged, scales)) return;
  }
}

// grid (kv_heads, tiles of pairs * splits)
template <int DT, int FMT, bool SPLIT, bool MORE, typename T>
__global__ void __launch_bounds__(kt_threads(SPLIT, DT), 3 - kt_groups(SPLIT, DT)) kv8_attn_tc_kernel(tha_attn_t a, tha_rows_t rows, const unsigned char* staged, const float4* scales, const float* q, T* out, int AP,
                                                                    int min_rows, int splits,
                                                                    float* partial, const float* gate, long long ldg, int* error_flag) {
  constexpr int GROUPS = kt_groups(SPLIT, DT), ROWS = GROUPS * KT_ROWS, THREADS = kt_threads(SPLIT, DT), KT_SOFTMAX = 8 * GROUPS, KT_LOAD = KT_SOFTMAX, KT_ISSUE = KT_LOAD + 1;
  constexpr int SLOTS = kt_slots(SPLIT, DT), KB = DT / 64, Q_PART = KB * KT_ROWS * 128, TILE = KT_KEYS * DT * 2;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ unsigned char kt_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(kt_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* Qs = smem;                          // [group][hi, lo][block][row][128 bytes]
  unsigned char* KVs = Qs + GROUPS * (SPLIT ? 2 : 1) * Q_PART;   // [K, V][slot][block][key][128 bytes]
  __shared__ uint64_t full[2][SLOTS], empty[2][SLOTS], s_full[2][2], p_full[2][2], pv_done[2][2], q_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_s;
  __shared__ float s_row[ROWS];               // per row: 1 / q's power of two times the scale, then what its two threads tell each other
  __shared__ alignas(16) float4 s_scales[KT_SCALES][2];   // of a tile's two parts

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int w = 0; w < 2; w++) {
      for (int i = 0; i < SLOTS; i++) { tc_mbar_init(&full[w][i], 1); tc_mbar_init(&empty[w][i], GROUPS); }
      for (int b = 0; b < 2; b++) { tc_mbar_init(&s_full[w][b], 1); tc_mbar_init(&p_full[w][b], 8); tc_mbar_init(&pv_done[w][b], 1); }
    }
    tc_mbar_init(&q_full, KT_SOFTMAX);
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == KT_ISSUE) {   // ahead of the trigger: what starts behind it takes what is left of the SM's TMEM
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(&tmem_slot)), "r"(256 * GROUPS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_trigger();                     // the kernel ahead has waited for those before it (kv8_stage_kernel): only what it stages is waited for, by the warp that fetches it
  auto release = [&]() {
    pdl_wait();                      // no kernel ends ahead of the one before it
    if (warp == KT_ISSUE) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256 * GROUPS));
  };
  const int D = a.dim, E = a.vdim, g = blockIdx.x, gsize = a.heads / a.kv_heads;
  const int sp = blockIdx.y % splits;
  int seq = -1, tile = 0;
  {
    // the last tiles of a prompt see the most keys: tile numbers in descending order over all sequences, so that the grid ends on short ones
    int i = (int)(blockIdx.y / splits);
    auto tiles_of = [&](int s) {
      const int n = rows.seq_first[s + 1] - rows.seq_first[s];
      return n >= min_rows ? (n + AP - 1) / AP : 0;
    };
    if (rows.n_seqs <= 32) {
      const int mine = lane < rows.n_seqs ? tiles_of(lane) : 0;
      for (int level = __reduce_max_sync(THA_FULL_MASK, mine) - 1; level >= 0; level--) {
        const unsigned has = __ballot_sync(THA_FULL_MASK, mine > level);
        if (i < __popc(has)) { seq = __fns(has, 0, i + 1); tile = level; break; }
        i -= __popc(has);
      }
    } else {
      const Kv8Piece pc = kv8_find(rows.n_seqs, i, tiles_of);
      seq = pc.seq;
      if (seq >= 0) tile = tiles_of(seq) - 1 - pc.at;
    }
  }
  if (seq < 0) { release(); return; }   // the same for the whole block
  const int seq_r0 = rows.seq_first[seq], r0 = seq_r0 + tile * AP, r_end = min(rows.seq_first[seq + 1], r0 + AP);
  const int p_first = rows.pos[seq_r0] + tile * AP, p_last = p_first + (r_end - r0) - 1;
  const int key_lo = a.chunk > 0 ? (p_first / a.chunk) * a.chunk : 0, last_first = a.chunk > 0 ? (p_last / a.chunk) * a.chunk : 0;
  const HybTiles tiles = hyb_attn_tiles(a, key_lo, p_first, p_last);   // of 32 keys: two to a tile here
  const int n_all = (tiles.n + 1) >> 1, per = (n_all + splits - 1) / splits, j0 = min(sp * per, n_all), n = min(j0 + per, n_all) - j0;   // tiles j0 .. j0 + n - 1
  auto part_key = [&](int ti) { return ti < tiles.n_a ? tiles.begin + 32 * ti : tiles.resume + 32 * (ti - tiles.n_a); };
  const size_t all = (size_t)rows.n_rows * a.heads;
  if (n < 1) {                           // a split behind the last tile: it has seen nothing
    for (int pr = threadIdx.x; pr < ROWS; pr += THREADS) {
      const int pp = pr / gsize;
      if (pp >= AP || r0 + pp >= r_end) continue;
      *reinterpret_cast<float2*>(partial + 2 * ((size_t)sp * all + (size_t)(r0 + pp) * a.heads + (size_t)g * gsize + (pr - pp * gsize))) = make_float2(-INFINITY, 0.f);
    }
    release();
    return;
  }

  int* abort_flag = &abort_s;
  if (warp < KT_SOFTMAX) {
    // q: eight lanes a row, sixteen rows a warp on their way at once; pairs past the block's positions are zeros.  A negative factor
    // of the scores goes into q.
    const int l8 = lane & 7;
#pragma unroll 1
    for (int b0 = 4 * warp + (lane >> 3); b0 < ROWS; b0 += 4 * 4 * KT_SOFTMAX) {
      float4 x[4][DT / 32];
      int h[4];
      bool ok[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int pr = b0 + u * 4 * KT_SOFTMAX, pp = pr / gsize;
        h[u] = g * gsize + (pr - pp * gsize);
        ok[u] = pp < AP && r0 + pp < r_end;
        const float* src = q + ((size_t)(r0 + pp) * a.heads + h[u]) * D;
#pragma unroll
        for (int i = 0; i < DT / 32; i++) {
          const int c = 32 * i + 4 * l8;
          x[u][i] = ok[u] && c < D ? *reinterpret_cast<const float4*>(src + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int pr = b0 + u * 4 * KT_SOFTMAX;
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < DT / 32; i++) top = fmaxf(top, fmaxf(fmaxf(fabsf(x[u][i].x), fabsf(x[u][i].y)), fmaxf(fabsf(x[u][i].z), fabsf(x[u][i].w))));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFu << (lane & 24), top, o));
        float inverse;
        const float up = split_scale<100>(top, 14, &inverse);
        const float f = ok[u] ? a.scale * (a.head_scale ? a.head_scale[h[u]] : 1.0f) : 0.f, s = f < 0.f ? -up : f == f ? up : f;   // no number stays none: below, the factor is held above 1e-30
        if (l8 == 0) s_row[pr] = inverse * fabsf(f) * (MORE ? 1.0f : LOG2E);
        unsigned char* row = Qs + (pr / KT_ROWS) * (SPLIT ? 2 : 1) * Q_PART + (pr % KT_ROWS) * 128;
#pragma unroll
        for (int i = 0; i < DT / 32; i++) {
          float4 v = x[u][i];
          if (FMT == THA_KV8_INT8) { const float y = v.y; v.y = v.z; v.z = y; }
          v.x *= s; v.y *= s; v.z *= s; v.w *= s;
          const uint2 hi = make_uint2(f16x2_of(make_float2(v.x, v.y)), f16x2_of(make_float2(v.z, v.w)));
          const int c = 32 * i + 4 * l8;
          unsigned char* dst = row + (c >> 6) * (KT_ROWS * 128) + ((((c & 63) >> 3) ^ (pr & 7)) << 4) + ((c & 7) << 1);
          *reinterpret_cast<uint2*>(dst) = hi;
          if (SPLIT) {   // what is left, in the same units: both parts go into one accumulator
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi.x)), z = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
            *reinterpret_cast<uint2*>(dst + Q_PART) = make_uint2(f16x2_of(make_float2(v.x - y.x, v.y - y.y)), f16x2_of(make_float2(v.z - z.x, v.w - z.y)));
          }
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) tc_mbar_arrive(&q_full);
  }

  if (warp < KT_SOFTMAX) {
    // ===== softmax: keys 32 hv .. 32 hv + 31 of a tile for a row of group w
    const int w = warp >> 3, hv = (warp >> 2) & 1, row = (warp & 3) * 32 + lane, pr = w * KT_ROWS + row;
    const int pair_bar = 1 + 4 * w + (warp & 3);      // the barrier of the two warps that share 32 rows
    const int pp = pr / gsize, h = g * gsize + (pr - pp * gsize);
    const bool row_ok = pp < AP && r0 + pp < r_end;
    const int pos = p_first + pp, first = a.chunk > 0 ? (pos / a.chunk) * a.chunk : 0;
    bool ok = tc_mbar_wait_warp(&q_full, 0u, abort_flag);
    const float fac = s_row[pr];
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + (uint32_t)(w * 2 * KT_KEYS + 32 * hv), t_o = tmem + lanes + (uint32_t)(GROUPS * 2 * KT_KEYS + w * DT + hv * (DT / 2));   // scores; this thread's half of the columns
    float m = -INFINITY, l = 0.f, ref = 0.f, down = 0.f, shift = 0.f;   // m: the reference, at most KT_SLACK below the largest score so far, the same in both threads of a row
    // every position of the block sees every one of 32 keys that begin at whole_lo .. whole_hi, or in the kept keys
    const int whole_hi = p_first - 31, whole_lo = a.window > 0 ? max(last_first, p_last - a.window + 1) : last_first, kept_hi = a.window > 0 ? a.keep_first - 32 : -1;
    alignas(16) float total[SPLIT ? DT / 2 : 1];
    float m_total = -INFINITY, ref_total = 0.f;       // the sum of the runs before this one, in its own units
    auto add_run = [&]() {                            // the accumulator into the total, in the present units
      const float f = m_total > -INFINITY ? hyb_ex2(m_total - m) * (ref > 0.f ? ref_total / ref : 0.f) : 0.f;
#pragma unroll 1
      for (int c = 0; c < DT / 2; c += 32) {          // columns from E on hold nothing, and nothing reads them
        float4 t[8];
        uint32_t o[32];
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = *reinterpret_cast<const float4*>(total + c + 4 * i);
        tc_tmem_ld32(t_o + (uint32_t)c, o);
        kt_wait_ld32(o);
#pragma unroll
        for (int i = 0; i < 8; i++)
          *reinterpret_cast<float4*>(total + c + 4 * i) =
              make_float4(fmaf(f, t[i].x, __uint_as_float(o[4 * i])), fmaf(f, t[i].y, __uint_as_float(o[4 * i + 1])), fmaf(f, t[i].z, __uint_as_float(o[4 * i + 2])),
                          fmaf(f, t[i].w, __uint_as_float(o[4 * i + 3])));
      }
      m_total = m; ref_total = ref;
    };
    if (SPLIT && n > KT_RUN) {
#pragma unroll 1
      for (int c = 0; c < DT / 2; c++) total[c] = 0.f;
    }
    auto both = [&](float mine, auto join) {          // join of the two threads' numbers, in both; one word a row is enough for it
      if (hv) s_row[pr] = mine;
      kt_any_of_pair(false, pair_bar);
      if (!hv) { mine = join(mine, s_row[pr]); s_row[pr] = mine; }
      kt_any_of_pair(false, pair_bar);
      return hv ? s_row[pr] : mine;                   // who joins reads it behind a barrier only, so that the other may write the next number at once
    };
    kt_any_of_pair(false, pair_bar);                  // both have read their factor
    for (int jl = 0; jl < n; jl++) {                  // to the end even where a wait has given up: the two warps meet at their barrier
      const int b = jl & 1;
      auto earlier = [&]() {                          // the products of earlier tiles are in the accumulator
        if (jl) ok = ok && tc_mbar_wait_warp(&pv_done[w][b ^ 1], (unsigned)((jl - 1) >> 1) & 1u, abort_flag);
        tc_fence_after();
      };
      const bool new_run = SPLIT && jl && jl % KT_RUN == 0;
      if (new_run) {
        earlier();
        add_run();
      }
      ok = ok && tc_mbar_wait_warp(&s_full[w][b], (unsigned)(jl >> 1) & 1u, abort_flag);   // the scales were there before the issuer saw the tile
      tc_fence_after();
      const uint32_t at = t_s + (uint32_t)(b * KT_KEYS);
      uint32_t x[32];
      tc_tmem_ld32(at, x);
      const float4 mine = s_scales[jl % KT_SCALES][hv];
      const float2 ks = make_float2(mine.x, mine.y);
      float vs0 = mine.z, vs1 = mine.w;               // of what this row sees: a weight of 0 under a scale far above the row's unit is no number
      const int ti = 2 * (j0 + jl) + hv;
      const bool there = ti < tiles.n;
      const int kt = part_key(there ? ti : tiles.n - 1);   // behind the last 32 their own keys again, as fetched
      const bool whole = there && kt <= whole_hi && (kt >= whole_lo || (kt <= kept_hi && kt >= last_first)) && fminf(ks.x, ks.y) >= 0.f;
      const float f0 = fmaxf(fac * ks.x, 1e-30f), f1 = fmaxf(fac * ks.y, 1e-30f);   // a hidden score is -inf under a scale of 0 as well
      kt_wait_ld32(x);
      if (MORE) {                                     // the score itself
#pragma unroll
        for (int i = 0; i < 32; i++) {
          float y = __uint_as_float(x[i]) * (i < 16 ? f0 : f1);
          if (a.softcap > 0.f) y = hyb_softcap(y, a.softcap);
          if (a.rel && row_ok) y += hyb_attn_rel(a, h, pos - (kt + i));
          x[i] = __float_as_uint(k8_log2_units(y));
        }
      }
      if (!whole) {
        uint32_t seen = row_ok && there ? kv8_sees32(a, kt, pos, first) : 0u;
        if (ks.x < 0.f) seen &= 0xFFFF0000u;
        if (ks.y < 0.f) seen &= 0xFFFFu;
#pragma unroll
        for (int i = 0; i < 32; i++) x[i] = seen >> i & 1u ? x[i] : 0xFF800000u;
        if (!(seen & 0xFFFFu)) vs0 = 0.f;
        if (!(seen >> 16)) vs1 = 0.f;
      }
      float mx;
      {
        float top[10];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int y = 0; y < 5; y++)
            top[5 * i + y] = k8_max3(__uint_as_float(x[16 * i + 3 * y]), __uint_as_float(x[16 * i + 3 * y + 1]), __uint_as_float(x[16 * i + 3 * y + 2]));
        const float m0 = k8_max3(k8_max3(top[0], top[1], top[2]), fmaxf(top[3], top[4]), __uint_as_float(x[15]));
        const float m1 = k8_max3(k8_max3(top[5], top[6], top[7]), fmaxf(top[8], top[9]), __uint_as_float(x[31]));
        mx = MORE ? fmaxf(m0, m1) : fmaxf(m0 * f0, m1 * f1);
      }
      bool grow = mx > m + KT_SLACK || (m == -INFINITY && mx > -INFINITY);
      float vtop = fmaxf(vs0, vs1);
      if (kt_any_of_pair(grow || vtop > ref, pair_bar)) {
        mx = both(mx, [](float a, float b) { return fmaxf(a, b); });
        vtop = both(vtop, [](float a, float b) { return fmaxf(a, b); });
        grow = mx > m + KT_SLACK || (m == -INFINITY && mx > -INFINITY);
        float corr = 1.f;
        if (grow) { corr = m > -INFINITY ? hyb_ex2(m - mx) : 0.f; m = mx; shift = MORE ? -m : KT_UP - m; }
        l *= corr;
        if (vtop > ref) {                             // the next power of two and a factor of 4 more, so that this is rare; lo ends at 2^-25 / 2^7 ref, below 2^-29 of the scale
          const float to = __uint_as_float(min(((__float_as_uint(vtop) + 0x7FFFFFu) & 0x7F800000u) + 0x1000000u, 0x7E800000u));
          corr *= ref / to;
          ref = to;
          down = 1.0f / ref;
        }
        if (jl && !new_run) {
          earlier();
#pragma unroll 1
          for (int c = 0; c < DT / 2; c += 16) {
            uint32_t o[16];
            tc_tmem_ld16(t_o + (uint32_t)c, o);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tc_tmem_st16(t_o + (uint32_t)c, o);
          }
        }
      }
      float2 sum = make_float2(0.f, 0.f);
      const float vr0 = vs0 * down, vr1 = vs1 * down;
      uint32_t hi[16], lo[16];
#pragma unroll
      for (int i = 0; i < 16; i++) {
        float2 y = make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
        const float f = i < 8 ? f0 : f1, vr = i < 8 ? vr0 : vr1;
        if (MORE) y = k8_add2(k8_add2(y, make_float2(shift, shift)), make_float2(KT_UP, KT_UP));   // next to a maximum of 2^127, 7 is nothing
        else y = f32x2_fma(y, make_float2(f, f), make_float2(shift, shift));
        const float2 p = make_float2(hyb_ex2(y.x), hyb_ex2(y.y));
        sum = k8_add2(sum, p);
        const float2 z = f32x2_mul(p, make_float2(vr, vr));
        hi[i] = f16x2_of(z);
        if (SPLIT) {
          const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
          lo[i] = f16x2_of(make_float2(z.x - u.x, z.y - u.y));
        }
      }
      tc_tmem_st16(at, hi);                                // over the scores that they come from
      if (SPLIT) tc_tmem_st16(at + 16u, lo);
      l += sum.x + sum.y;
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) tc_mbar_arrive(&p_full[w][b]);
    }
    if (ok) ok = tc_mbar_wait(&pv_done[w][(n - 1) & 1], (unsigned)((n - 1) >> 1) & 1u, abort_flag);
    tc_fence_after();
    ok = __all_sync(THA_FULL_MASK, ok);
    if (!ok) l = NAN;                                 // a wait has given up: the row, whichever of its threads it was, is no number rather than left as it was
    l = both(l, [](float a, float b) { return a + b; });
    const size_t at = row_ok ? (size_t)(r0 + pp) * a.heads + h : 0;
    float scale = exp2f(-KT_UP);                      // times ref, in this order: ref's smallest number times less is none that holds all bits
    l *= exp2f(-KT_UP);
    if (SPLIT && n > KT_RUN) add_run();
    if (l != l) m = l;                                // a NaN among the scores shows in the sum alone
    float* pd = splits > 1 ? partial + k8_sums_floats(splits, all) + ((size_t)sp * all + at) * E : nullptr;
    if (row_ok) {
      scale *= pd ? (l > 0.f ? 1.0f / l : l) : k8_final(a, h, m, l, gate ? gate + (size_t)(r0 + pp) * ldg : nullptr);   // a part is a mean
      if (pd && hv == 0) *reinterpret_cast<float2*>(partial + 2 * ((size_t)sp * all + at)) = make_float2(m, l);
    }
#pragma unroll 1
    for (int c = 0; c < DT / 2 && hv * (DT / 2) + c < E; c += 16) {
      uint32_t o[16];
      if (SPLIT && n > KT_RUN) {
#pragma unroll
        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(total[c + i]);
      } else {
        tc_tmem_ld16(t_o + (uint32_t)c, o);
        tc_wait_ld();
      }
      if (row_ok) {
        const int col = hv * (DT / 2) + c;
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int from = FMT == THA_KV8_INT8 && (i & 3) % 3 ? i ^ 3 : i;   // columns 1 and 2 of every four hold channels 2 and 1
          v[i] = __uint_as_float(o[from]) * scale * ref;
        }
        if (pd || sizeof(T) == 4 || a.out_f32) {
          float* dst = pd ? pd + col : reinterpret_cast<float*>(out) + at * E + col;
#pragma unroll
          for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
          __nv_bfloat162 y[8];
#pragma unroll
          for (int i = 0; i < 8; i++) y[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + at * E + col);
          dst[0] = reinterpret_cast<const uint4*>(y)[0];
          dst[1] = reinterpret_cast<const uint4*>(y)[1];
        }
      }
    }
    tc_fence_before();
  } else if (warp == KT_LOAD) {
    // ===== tiles: two parts each, behind the last the last again
    const int stage0 = kt_stage_base(a, rows, seq, min_rows);
    const HybTiles parts = kt_seq(a, rows, seq, min_rows).parts;
    pdl_wait();
    if (tc_elect()) {
      int at = 0;
      unsigned turn = 0;                            // how often the ring has come round
      bool ok = true;
      int sent[2] = {0, 0};
      for (int jl = 0; jl < n && ok; jl++) {
        size_t from[2];
#pragma unroll
        for (int hf = 0; hf < 2; hf++)
          from[hf] = (size_t)(stage0 + kt_part_of(parts, part_key(min(2 * (j0 + jl) + hf, tiles.n - 1)))) * a.kv_heads + g;
#pragma unroll
        for (int side = 0; side < 2; side++) {
          if (ok && turn) ok = tc_mbar_wait(&empty[side][at], (turn - 1) & 1u, abort_flag);
          if (!ok) break;
          tc_mbar_expect_tx(&full[side][at], TILE + (side ? 0 : 32));
          sent[side]++;
#pragma unroll
          for (int hf = 0; hf < 2; hf++) {
            if (side == 0) tc_bulk(&s_scales[jl % KT_SCALES][hf], scales + from[hf], 16, &full[0][at]);
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
              tc_bulk(KVs + (side * SLOTS + at) * TILE + kb * (KT_KEYS * 128) + hf * (32 * 128), staged + from[hf] * kt_part(DT) + (side * KB + kb) * (32 * 128), 32 * 128, &full[side][at]);
          }
        }
        if (++at == SLOTS) { at = 0; turn++; }
      }
      if (!ok) {                                    // copies in flight land before the block's shared memory is another's
        tc_drain(full[0], SLOTS, sent[0]);
        tc_drain(full[1], SLOTS, sent[1]);
      }
    }
  } else if (tc_elect()) {
    // ===== products of group w.  One thread's products run in the order of their issue, so that the scores of tile j + 2 may be asked for as soon as the weights of tile j, in whose
    // columns they go, are.
    const int w = warp - KT_ISSUE;
    const uint32_t id_s = kt_idesc(KT_KEYS, 0), id_o = kt_idesc(E, 1);
    const uint32_t q_desc = kt_desc_k(tc_smem_u32(Qs)) + (uint32_t)(w * ((SPLIT ? 2 : 1) * Q_PART >> 4)), k_desc = kt_desc_k(tc_smem_u32(KVs));
    const uint32_t v_desc = kt_desc_mn(tc_smem_u32(KVs) + SLOTS * TILE, KT_KEYS * 128);
    const uint32_t t_s = tmem + (uint32_t)(w * 2 * KT_KEYS), t_o = tmem + (uint32_t)(GROUPS * 2 * KT_KEYS + w * DT);
    const int k_steps = D / 16;
    int k_at = 0, v_at = 0;                         // the next slot of each ring
    unsigned k_turn = 0, v_turn = 0;
    auto scores = [&](int b) {
      const bool ok = tc_mbar_wait(&full[0][k_at], k_turn, abort_flag);
      if (!ok) return false;
      tc_fence_after();
      const uint32_t kd = k_desc + (uint32_t)(k_at * (TILE >> 4));
#pragma unroll
      for (int part = SPLIT ? 1 : 0; part >= 0; part--) {   // what is small first: sums are cut off at the size of what is there
#pragma unroll
        for (int s = 0; s < DT / 16; s++) {
          if (s < k_steps)
            kt_mma(t_s + (uint32_t)(b * KT_KEYS), q_desc + (uint32_t)((part * Q_PART + (s >> 2) * KT_ROWS * 128 >> 4) + 2 * (s & 3)),
                   kd + (uint32_t)(((s >> 2) * KT_KEYS * 128 >> 4) + 2 * (s & 3)), id_s, s != 0 || (SPLIT && part == 0));
        }
      }
      tc_commit(&s_full[w][b]);
      tc_commit(&empty[0][k_at]);
      if (++k_at == SLOTS) { k_at = 0; k_turn ^= 1u; }
      return true;
    };
    bool ok = tc_mbar_wait(&q_full, 0u, abort_flag);
    for (int jl = 0; jl < 2 && jl < n && ok; jl++) ok = scores(jl);
    for (int jl = 0; jl < n && ok; jl++) {
      const int b = jl & 1;
      const bool adds = (SPLIT ? jl % KT_RUN : jl) != 0;
      const uint32_t vd = v_desc + (uint32_t)(v_at * (TILE >> 4)), p = t_s + (uint32_t)(b * KT_KEYS);
      ok = tc_mbar_wait(&full[1][v_at], v_turn, abort_flag) && tc_mbar_wait(&p_full[w][b], (unsigned)(jl >> 1) & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int x = 0; x < KT_KEYS / 16; x++) {
        const uint32_t px = p + (uint32_t)(32 * (x >> 1) + 8 * (x & 1));
        kt_mma_ts(t_o, px, vd + (uint32_t)(x * (2048 >> 4)), id_o, x != 0 || adds);
        if (SPLIT) kt_mma_ts(t_o, px + 16u, vd + (uint32_t)(x * (2048 >> 4)), id_o, true);
      }
      tc_commit(&pv_done[w][b]);
      tc_commit(&empty[1][v_at]);
      if (++v_at == SLOTS) { v_at = 0; v_turn ^= 1u; }
      if (jl + 2 < n) ok = scores(b);
    }
  }
  __syncwarp();
  __syncthreads();
  tc_fence_after();
  release();
  if (threadIdx.x == 0 && abort_s && error_flag) *((volatile int*)error_flag) = 1;
}

static int kt_positions(const tha_attn_t* a, int dtype) {
  return kt_groups(kv8_exact(a, dtype), a->dim > 64 || a->vdim > 64 ? 128 : 64) * KT_ROWS / (a->heads / a->kv_heads);
}
// Sequences of at least min_rows rows that a step has at most.  (From the rows alone: the longest portion that a caller names may be one that no sequence has.)
static long long kt_sequences(const tha_rows_t* rows, int min_rows) { return rows->n_rows / min_rows < rows->n_seqs ? rows->n_rows / min_rows : rows->n_seqs; }
static long long kt_blocks(const tha_attn_t* a, const tha_rows_t* rows, int dtype, int min_rows) {
  return (long long)rows->n_rows / kt_positions(a, dtype) + kt_sequences(rows, min_rows);
}

// Parts of a context, most_tiles: of 32 keys.
int kv8_attn_tc_splits(const tha_attn_t* a, const tha_rows_t* rows, int dtype, int most_tiles) {
  const int each = 3 - kt_groups(kv8_exact(a, dtype), a->dim > 64 || a->vdim > 64 ? 128 : 64);   // blocks an SM
  const long long blocks = (long long)ceil_div(rows->n_rows, kt_positions(a, dtype)) * a->kv_heads;
  long long s = each * sm_budget() / blocks;
  if (s > most_tiles / 16) s = most_tiles / 16;       // eight tiles each at least
  return s < 1 ? 1 : s > 16 ? 16 : (int)s;
}

// Parts that a step's sequences of this form have at most, bytes of scratch for them (0: this form does not take the step): the parts, then their scales
static long long kt_part_bytes(const tha_attn_t* a) { return (long long)a->kv_heads * (kt_part(a->dim > 64 || a->vdim > 64 ? 128 : 64) + 16); }
static long long kt_parts(const tha_rows_t* rows, int most_tiles, int min_rows) { return kt_sequences(rows, min_rows) * most_tiles; }
size_t kv8_attn_tc_stage_bytes(const tha_attn_t* a, const tha_rows_t* rows, int most_tiles, int min_rows) {
  const long long parts = kt_parts(rows, most_tiles, min_rows), bytes = parts * kt_part_bytes(a);
  return parts > 0x7FFFFFFFll || bytes > KT_MOST_STAGED ? 0 : (size_t)bytes;
}
int kv8_attn_tc_room_for(const tha_attn_t* a, int most_tiles) { return (int)(KT_MOST_STAGED / (kt_part_bytes(a) * most_tiles)); }

template <int DT, int FMT, bool SPLIT, bool MORE, typename T>
static int kt_launch(cudaStream_t s, int dtype, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, T* out, int min_rows, int most_tiles, int splits,
                     unsigned char* staged, float* partial, const float* gate, long long ldg) {
  int* flag = nullptr;                               // allocated by a device's first call, which a capture allows in this mode
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  THA_CUDA_OK(cudaThreadExchangeStreamCaptureMode(&mode));
  const int st = gemm_tc_init(&flag);
  THA_CUDA_OK(cudaThreadExchangeStreamCaptureMode(&mode));
  THA_TRY_RC(st);
  const long long parts = kt_parts(rows, most_tiles, min_rows);
  float4* scales = reinterpret_cast<float4*>(staged + (size_t)parts * a->kv_heads * kt_part(DT));
  // A step of a prompt and many single rows has far fewer parts than it might: blocks for those of one sequence, or for sixteen on an SM, take all of them in turn.
  const int groups = ceil_div(a->kv_heads, KT_STAGE_HEADS), at_once = ceil_div(16 * sm_budget(), groups);
  const long long blocks = at_once > most_tiles ? at_once : most_tiles;
  THA_CUDA_OK(launch(parts > blocks ? kv8_stage_kernel<DT, FMT, true> : kv8_stage_kernel<DT, FMT, false>, dim3((unsigned)(parts > blocks ? blocks : parts), groups), dim3(32 * DT / 16), 0, s,
                     pdl_enabled() != 0, *a, *rows, *kv, min_rows, (int)parts, staged, scales));
  auto k = kv8_attn_tc_kernel<DT, FMT, SPLIT, MORE, T>;
  THA_CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kt_smem(SPLIT, DT)));
  THA_CUDA_OK(launch(k, dim3(a->kv_heads, (unsigned)(kt_blocks(a, rows, dtype, min_rows) * splits)), dim3(kt_threads(SPLIT, DT)), kt_smem(SPLIT, DT), s, pdl_enabled() != 0, *a, *rows,
                     (const unsigned char*)staged, (const float4*)scales, q, out, kt_positions(a, dtype), min_rows, splits, partial, gate, ldg, flag));
  return THA_STATUS_SUCCESS;
}
template <int DT, bool SPLIT, typename T>
static int kt_form(cudaStream_t s, int dtype, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, T* out, int min_rows, int most_tiles, int splits,
                   unsigned char* staged, float* partial, const float* gate, long long ldg) {
  const bool more = a->softcap > 0.f || a->rel;
  if (kv->format == THA_KV8_INT8)
    return more ? kt_launch<DT, THA_KV8_INT8, SPLIT, true>(s, dtype, a, rows, kv, q, out, min_rows, most_tiles, splits, staged, partial, gate, ldg)
                : kt_launch<DT, THA_KV8_INT8, SPLIT, false>(s, dtype, a, rows, kv, q, out, min_rows, most_tiles, splits, staged, partial, gate, ldg);
  return more ? kt_launch<DT, THA_KV8_E4M3, SPLIT, true>(s, dtype, a, rows, kv, q, out, min_rows, most_tiles, splits, staged, partial, gate, ldg)
              : kt_launch<DT, THA_KV8_E4M3, SPLIT, false>(s, dtype, a, rows, kv, q, out, min_rows, most_tiles, splits, staged, partial, gate, ldg);
}

// staged: as many bytes as kv8_attn_tc_stage_bytes says, on a 16-byte boundary
int kv8_attn_tc_launch(cudaStream_t s, int dtype, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, void* out, int min_rows, int most_tiles,
                       int splits, void* staged, float* partial, const float* gate, long long ldg) {
  if (!aligned16(out) || kt_blocks(a, rows, dtype, min_rows) * splits > 65535) return THA_STATUS_NOT_SUPPORTED;
  const bool wide = a->dim > 64 || a->vdim > 64;
  auto st = (unsigned char*)staged;
  if (dtype == THA_DT_BF16) {
    auto o = (__nv_bfloat16*)out;
    if (kv8_exact(a, dtype)) return wide ? kt_form<128, true>(s, dtype, a, rows, kv, q, o, min_rows, most_tiles, splits, st, partial, gate, ldg)
                                         : kt_form<64, true>(s, dtype, a, rows, kv, q, o, min_rows, most_tiles, splits, st, partial, gate, ldg);
    return wide ? kt_form<128, false>(s, dtype, a, rows, kv, q, o, min_rows, most_tiles, splits, st, partial, gate, ldg)
                : kt_form<64, false>(s, dtype, a, rows, kv, q, o, min_rows, most_tiles, splits, st, partial, gate, ldg);
  }
  auto o = (float*)out;
  return wide ? kt_form<128, true>(s, dtype, a, rows, kv, q, o, min_rows, most_tiles, splits, st, partial, gate, ldg)
              : kt_form<64, true>(s, dtype, a, rows, kv, q, o, min_rows, most_tiles, splits, st, partial, gate, ldg);
}

}  // namespace tha
