// Softmax attention of prompt portions over the cache in 8 bits on the 5th-generation tensor cores (tcgen05 + TMEM): sequences whose (position, head) pairs fill
// tiles of 256.  kv8_attn.cu keeps single rows and short portions.
//
// Codes are fp16 numbers, so a tile of 64 keys goes from the cache through registers of converter warps to fp16 tiles in shared memory, without scales: K's scale
// belongs to 16 or more neighbouring keys and multiplies their scores, V's multiplies their weights, relative to a power of two that all of a row's weights share.  q is brought to
// [2^14, 2^15) by a power of two a row and rounded to one fp16 (bf16 results) or two (SPLIT: fp32 results, 22 bits; weights likewise), each product fp32.
// A block takes 256 pairs of one key/value head, two groups of 128 rows that share every tile, and a run of tiles.  Four groups of four warps (registers a thread 168, 168, 112, 64 of the
// 512 that four threads have at launch):
//   0 .. 3, 4 .. 7  softmax of group 0 and 1, a thread a row: 64 scores out of TMEM, factor, mask, weights back into the same TMEM columns as the A operand of the second product
//   8 .. 11         tiles, 16 keys a warp: the next tile's codes are on their way into registers while this one's are converted
//   12              allocates TMEM; one elected thread issues the products, scores of tile j + 1 ahead of weights x values of tile j
// The accumulator stays in TMEM.  The tensor cores cut off what their fp32 sums cannot hold, so that an error grows with the number of sums: 100 rows behind 3900 keys were 8.6e-6
// off with two fp16 an operand.  SPLIT therefore adds the accumulators of runs of 16 tiles (128 sums) in fp32, in local memory.  It is rescaled only where a row's maximum has grown by more than 2^8 since its reference was taken (weights are at most 2^15 then:
// fp16 holds them), or V's scales outgrow theirs.
#include "gemm_tc.h"
#include "kv8.cuh"
#include "tc_common.cuh"

namespace tha {

constexpr int KT_KEYS = 64, KT_ROWS = 128, KT_THREADS = 512, KT_CONV = 8, KT_ISSUE = 12;
constexpr float KT_UP = 7.0f, KT_SLACK = 8.0f;
constexpr int KT_RUN = 16;   // SPLIT: tiles that one accumulator sums

__host__ __device__ constexpr int kt_stages(bool split, int DT) { return split && DT == 128 ? 3 : 4; }
__host__ __device__ constexpr int kt_smem(bool split, int DT) { return (split ? 2 : 1) * 2 * KT_ROWS * DT * 2 + kt_stages(split, DT) * 2 * KT_KEYS * DT * 2 + 1024; }

__device__ __forceinline__ void kt_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
        "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]),
        "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void kt_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void kt_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void kt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// kind::f16, fp16 x fp16 -> fp32, M = 128; b_mn: the B operand's N runs along its rows
__device__ __forceinline__ uint32_t kt_idesc(int n, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// MN-major B, SWIZZLE_128B: blocks of 64 columns (128 bytes) x 8 rows of K; K groups 1024 bytes apart, column blocks `block` bytes
__device__ __forceinline__ uint64_t kt_desc_mn(uint32_t saddr, uint32_t block) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(block >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Four codes as two fp16 pairs.  int8: channels (0, 2), (1, 3), what is cheapest to take apart: q's channels and the result's are in that order too.
template <int FMT>
__device__ __forceinline__ uint2 kt_half4(uint32_t w) {
  if (FMT == THA_KV8_INT8) return make_uint2(k8_bytes02(w), k8_bytes02(w >> 8));
  return make_uint2(k8_e4m3x2(w & 0xFFFFu), k8_e4m3x2(w >> 16));
}

// grid (kv_heads, tiles of pairs * splits)
template <int DT, int FMT, bool SPLIT, bool MORE, typename T>
__global__ void __launch_bounds__(KT_THREADS, 1) kv8_attn_tc_kernel(tha_attn_t a, tha_rows_t rows, tha_kv8_t kv, const float* q, T* out, int AP, int min_rows, int splits,
                                                                    float* partial, const float* gate, long long ldg, int* error_flag) {
  constexpr int STAGES = kt_stages(SPLIT, DT), KB = DT / 64, Q_PART = KB * KT_ROWS * 128, K_STAGE = KT_KEYS * DT * 2, KV_STAGE = 2 * K_STAGE;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ unsigned char kt_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(kt_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* Qs = smem;                          // [group][hi, lo][block][row][128 bytes]
  unsigned char* KVs = Qs + 2 * (SPLIT ? 2 : 1) * Q_PART;   // [stage][K | V][block][key][128 bytes]
  __shared__ uint64_t kv_full[STAGES], kv_empty[STAGES], s_full[2][2], p_full[2][2], pv_done[2][2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_s;
  __shared__ float s_fac[2 * KT_ROWS];               // per row: 1 / q's power of two times the scale
  __shared__ float4 s_ks[STAGES], s_vs[STAGES];      // per 16 keys of a tile; K's below 0: the keys do not exist

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; i++) { tc_mbar_init(&kv_full[i], 4); tc_mbar_init(&kv_empty[i], 1); }
    for (int w = 0; w < 2; w++)
      for (int b = 0; b < 2; b++) { tc_mbar_init(&s_full[w][b], 1); tc_mbar_init(&p_full[w][b], 4); tc_mbar_init(&pv_done[w][b], 1); }
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == KT_ISSUE) {   // ahead of the trigger: what starts behind it takes what is left of the SM's TMEM
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(&tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  kt_fence_before();
  __syncthreads();
  kt_fence_after();
  const uint32_t tmem = tmem_slot;
  hyb_pdl_enter();
  auto release = [&]() {
    if (warp == KT_ISSUE) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  };
  const int D = a.dim, E = a.vdim, g = blockIdx.x, gsize = a.heads / a.kv_heads, layer = a.cache_layer;
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
  const int seq_r0 = rows.seq_first[seq], r0 = seq_r0 + tile * AP, r_end = min(rows.seq_first[seq + 1], r0 + AP), slot = rows.seq_slot[seq];
  const int p_first = rows.pos[seq_r0] + tile * AP, p_last = p_first + (r_end - r0) - 1;
  const int key_lo = a.chunk > 0 ? (p_first / a.chunk) * a.chunk : 0, last_first = a.chunk > 0 ? (p_last / a.chunk) * a.chunk : 0;
  const HybTiles tiles = hyb_attn_tiles(a, key_lo, p_first, p_last);   // of 32 keys: two to a tile here
  const int n_all = (tiles.n + 1) >> 1, per = (n_all + splits - 1) / splits, j0 = min(sp * per, n_all), n = min(j0 + per, n_all) - j0;   // tiles j0 .. j0 + n - 1
  auto half_key = [&](int ti) { return ti < tiles.n_a ? tiles.begin + 32 * ti : tiles.resume + 32 * (ti - tiles.n_a); };
  const size_t all = (size_t)rows.n_rows * a.heads;
  if (n < 1) {                           // a split behind the last tile: it has seen nothing
    for (int pr = threadIdx.x; pr < 2 * KT_ROWS; pr += KT_THREADS) {
      const int pp = pr / gsize;
      if (pp >= AP || r0 + pp >= r_end) continue;
      *reinterpret_cast<float2*>(partial + 2 * ((size_t)sp * all + (size_t)(r0 + pp) * a.heads + (size_t)g * gsize + (pr - pp * gsize))) = make_float2(-INFINITY, 0.f);
    }
    release();
    return;
  }

  // q: warp w takes rows w, w + 16, .., eight on their way at a time; pairs past the block's positions are zeros.  A negative factor of the scores goes into q.
#pragma unroll 1
  for (int b0 = warp; b0 < 2 * KT_ROWS; b0 += 8 * (KT_THREADS / 32)) {
    const int c = 4 * lane;
    float4 rows4[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int pr = b0 + i * (KT_THREADS / 32), pp = pr / gsize, h = g * gsize + (pr - pp * gsize);
      rows4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (pp < AP && r0 + pp < r_end && c < D) rows4[i] = *reinterpret_cast<const float4*>(q + ((size_t)(r0 + pp) * a.heads + h) * D + c);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int pr = b0 + i * (KT_THREADS / 32), pp = pr / gsize, h = g * gsize + (pr - pp * gsize);
      const bool ok = pp < AP && r0 + pp < r_end;
      float4 v = rows4[i];
      const float top = warp_max(fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
      float inverse;
      const float up = split_scale<100>(top, 14, &inverse);
      const float f = ok ? a.scale * (a.head_scale ? a.head_scale[h] : 1.0f) : 0.f;
      if (lane == 0) s_fac[pr] = inverse * fabsf(f) * (MORE ? 1.0f : LOG2E);
      if (c < DT) {
        const float s = f < 0.f ? -up : up;
        if (FMT == THA_KV8_INT8) { const float y = v.y; v.y = v.z; v.z = y; }
        v.x *= s; v.y *= s; v.z *= s; v.w *= s;
        const uint2 hi = make_uint2(f16x2_of(make_float2(v.x, v.y)), f16x2_of(make_float2(v.z, v.w)));
        unsigned char* dst = Qs + (pr / KT_ROWS) * (SPLIT ? 2 : 1) * Q_PART + (c >> 6) * (KT_ROWS * 128) + (pr % KT_ROWS) * 128 + ((((c & 63) >> 3) ^ (pr & 7)) << 4) + ((c & 7) << 1);
        *reinterpret_cast<uint2*>(dst) = hi;
        if (SPLIT) {   // what is left, in the same units: both parts go into one accumulator
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&hi.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
          *reinterpret_cast<uint2*>(dst + Q_PART) = make_uint2(f16x2_of(make_float2(v.x - x.x, v.y - x.y)), f16x2_of(make_float2(v.z - y.x, v.w - y.y)));
        }
      }
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  int* abort_flag = &abort_s;

  if (warp < KT_CONV) {
    // ===== softmax of group w
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const int w = warp >> 2, row = (warp & 3) * 32 + lane, pr = w * KT_ROWS + row;
    const int pp = pr / gsize, h = g * gsize + (pr - pp * gsize);
    const bool row_ok = pp < AP && r0 + pp < r_end;
    const int pos = p_first + pp, first = a.chunk > 0 ? (pos / a.chunk) * a.chunk : 0;
    const float fac = s_fac[pr];
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + (uint32_t)(w * 2 * KT_KEYS), t_o = tmem + lanes + (uint32_t)(4 * KT_KEYS + w * DT);
    float m = -INFINITY, l = 0.f, ref = 0.f;         // m: the reference, at most KT_SLACK below the largest score so far
    bool ok = true;
    float total[SPLIT ? DT : 1], m_total = -INFINITY, ref_total = 0.f;   // the sum of the runs before this one, in its own units
    auto add_run = [&]() {                            // the accumulator into the total; both end in the present units
      const float f = m_total > -INFINITY ? k8_ex2(m_total - m) * (ref > 0.f ? ref_total / ref : 0.f) : 0.f;
#pragma unroll 1
      for (int c = 0; c < DT; c += 16) {
        uint32_t o[16];
        tc_tmem_ld16(t_o + (uint32_t)c, o);
        kt_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; i++) total[c + i] = fmaf(f, total[c + i], __uint_as_float(o[i]));
      }
      m_total = m; ref_total = ref;
    };
    if (SPLIT && n > KT_RUN) {
#pragma unroll 1
      for (int c = 0; c < DT; c++) total[c] = 0.f;
    }
    for (int jl = 0; jl < n && ok; jl++) {
      const int b = jl & 1, st = jl % STAGES;
      ok = tc_mbar_wait(&kv_full[st], (unsigned)(jl / STAGES) & 1u, abort_flag);   // the scales
      ok = ok && tc_mbar_wait(&s_full[w][b], (unsigned)(jl >> 1) & 1u, abort_flag);
      ok = __all_sync(THA_FULL_MASK, ok);
      kt_fence_after();
      uint32_t sr[KT_KEYS];
      kt_ld32(t_s + (uint32_t)(b * KT_KEYS), sr);
      kt_ld32(t_s + (uint32_t)(b * KT_KEYS + 32), sr + 32);
      const float4 ks4 = s_ks[st], vs4 = s_vs[st];
      const float ks[4] = {ks4.x, ks4.y, ks4.z, ks4.w}, vs[4] = {vs4.x, vs4.y, vs4.z, vs4.w};
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = fmaxf(fac * ks[i], 1e-30f);   // a hidden score is -inf under a scale of 0 as well
      kt_wait_ld();
      float mx = -INFINITY;
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        const int ti = 2 * (j0 + jl) + hf;
        const bool there = ti < tiles.n;
        const int kt = half_key(there ? ti : tiles.n - 1);   // behind the last half its own keys again, as fetched
        if (MORE) {
#pragma unroll
          for (int i = 0; i < 32; i++) {
            float x = __uint_as_float(sr[32 * hf + i]) * f[2 * hf + (i >> 4)];
            if (a.softcap > 0.f) x = hyb_softcap(x, a.softcap);
            if (a.rel && row_ok) x += hyb_attn_rel(a, h, pos - (kt + i));
            sr[32 * hf + i] = __float_as_uint(x * LOG2E);
          }
        }
        // every position of the block sees every key of this half
        const bool whole = there && kt + 31 <= p_first && kt >= last_first && (a.window <= 0 || p_last - kt < a.window || kt + 32 <= a.keep_first) && ks[2 * hf] >= 0.f &&
                           ks[2 * hf + 1] >= 0.f;
        if (!whole) {
          uint32_t seen = row_ok && there ? kv8_sees32(a, kt, pos, first) : 0u;
          if (ks[2 * hf] < 0.f) seen &= 0xFFFF0000u;
          if (ks[2 * hf + 1] < 0.f) seen &= 0xFFFFu;
#pragma unroll
          for (int i = 0; i < 32; i++) sr[32 * hf + i] = seen >> i & 1u ? sr[32 * hf + i] : 0xFF800000u;
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float top = __uint_as_float(sr[32 * hf + 16 * i]);
#pragma unroll
          for (int x = 1; x < 16; x++) top = fmaxf(top, __uint_as_float(sr[32 * hf + 16 * i + x]));
          mx = fmaxf(mx, MORE ? top : top * f[2 * hf + i]);
        }
      }
      const float vtop = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
      const bool grow = mx > m + KT_SLACK || (m == -INFINITY && mx > -INFINITY);
      const bool wider = vtop > ref;                  // the same for the whole block
      if (wider || __any_sync(THA_FULL_MASK, grow)) {
        float corr = 1.f;
        if (grow) { corr = m > -INFINITY ? k8_ex2(m - mx) : 0.f; m = mx; }
        l *= corr;
        if (wider) {                                  // the next power of two and a factor of 4 more, so that this is rare
          const float to = __uint_as_float(min(((__float_as_uint(vtop) + 0x7FFFFFu) & 0x7F800000u) + 0x1000000u, 0x7E800000u));
          corr *= ref / to;
          ref = to;
        }
        if (jl > 0) {                                 // all products of earlier tiles are in the accumulator
          ok = __all_sync(THA_FULL_MASK, tc_mbar_wait(&pv_done[w][b ^ 1], (unsigned)((jl - 1) >> 1) & 1u, abort_flag) && ok);
          kt_fence_after();
#pragma unroll
          for (int c = 0; c < DT; c += 32) {
            uint32_t o[32];
            kt_ld32(t_o + (uint32_t)c, o);
            kt_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tc_tmem_st32(t_o + (uint32_t)c, o);
          }
        }
      }
      if (SPLIT && jl && jl % KT_RUN == 0) {          // in the units of the run that has ended or already in this tile's: they are what the accumulator has
        ok = __all_sync(THA_FULL_MASK, tc_mbar_wait(&pv_done[w][b ^ 1], (unsigned)((jl - 1) >> 1) & 1u, abort_flag) && ok);
        kt_fence_after();
        add_run();
      }
      const float shift = m > -INFINITY ? KT_UP - m : 0.f, down = ref > 0.f ? 1.0f / ref : 0.f;
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < KT_KEYS / 2; c += 16) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int k = 2 * (c + i), qd = k >> 4;
          float2 x = make_float2(__uint_as_float(sr[k]), __uint_as_float(sr[k + 1]));
          if (MORE) { x.x += shift; x.y += shift; }
          else x = f32x2_fma(x, make_float2(f[qd], f[qd]), make_float2(shift, shift));
          const float2 p = make_float2(k8_ex2(x.x), k8_ex2(x.y));
          sum.x += p.x; sum.y += p.y;
          const float vr = vs[qd] * down;
          const float2 y = f32x2_mul(p, make_float2(vr, vr));
          hi[i] = f16x2_of(y);
          if (SPLIT) {
            const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
            lo[i] = f16x2_of(make_float2(y.x - z.x, y.y - z.y));
          }
        }
        kt_st16(t_s + (uint32_t)(b * KT_KEYS + c), hi);
        if (SPLIT) kt_st16(t_s + (uint32_t)(b * KT_KEYS + 32 + c), lo);
      }
      l += sum.x + sum.y;
      kt_wait_st();
      kt_fence_before();
      __syncwarp();
      if (lane == 0) tc_mbar_arrive(&p_full[w][b]);
    }
    if (ok) ok = tc_mbar_wait(&pv_done[w][(n - 1) & 1], (unsigned)((n - 1) >> 1) & 1u, abort_flag);
    kt_fence_after();
    ok = __all_sync(THA_FULL_MASK, ok);
    const size_t at = row_ok ? (size_t)(r0 + pp) * a.heads + h : 0;
    float scale = ref * exp2f(-KT_UP);
    l *= exp2f(-KT_UP);
    if (SPLIT && n > KT_RUN) add_run();
    if (l != l) m = l;                                // a NaN among the scores shows in the sum alone
    float* pd = splits > 1 ? partial + 2 * all * splits + ((size_t)sp * all + at) * E : nullptr;
    if (row_ok) {
      if (pd) *reinterpret_cast<float2*>(partial + 2 * ((size_t)sp * all + at)) = make_float2(m, l);
      else scale *= k8_final(a, h, m, l, gate ? gate + (size_t)(r0 + pp) * ldg : nullptr);
    }
#pragma unroll 1
    for (int c = 0; c < E; c += 16) {
      uint32_t o[16];
      if (SPLIT && n > KT_RUN) {
#pragma unroll
        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(total[c + i]);
      } else {
        tc_tmem_ld16(t_o + (uint32_t)c, o);
        kt_wait_ld();
      }
      if (row_ok && ok) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int from = FMT == THA_KV8_INT8 && (i & 3) % 3 ? i ^ 3 : i;   // columns 1 and 2 of every four hold channels 2 and 1
          v[i] = __uint_as_float(o[from]) * scale;
        }
        if (pd || sizeof(T) == 4 || a.out_f32) {
          float* dst = pd ? pd + c : reinterpret_cast<float*>(out) + at * E + c;
#pragma unroll
          for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
          __nv_bfloat162 x[8];
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + at * E + c);
          dst[0] = reinterpret_cast<const uint4*>(x)[0];
          dst[1] = reinterpret_cast<const uint4*>(x)[1];
        }
      }
    }
    kt_fence_before();
  } else if (warp < KT_ISSUE) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    // ===== tiles: 16 keys of one block a warp; lane: row lane / 4 of eight, 16-byte piece lane % 4 of four
    const int cw = warp - KT_CONV, rl = lane >> 2, cl = lane & 3, B = kv.block_size;
    const uint8_t *kpool = static_cast<const uint8_t*>(kv.k_pool), *vpool = static_cast<const uint8_t*>(kv.v_pool);
    auto key_of = [&](int jl) {   // this warp's first key of a tile; behind the last half that half again
      const int ti = 2 * (j0 + jl) + (cw >> 1);
      return half_key(ti < tiles.n ? ti : tiles.n - 1) + 16 * (cw & 1);
    };
    auto id_of = [&](int jl) {
      if (jl >= n) return -1;
      const int key = key_of(jl);
      return key <= p_last ? kv8_block(kv, slot, key) : -1;
    };
    uint4 ck[4], cv[4];
    float ks, vs;
    auto fetch = [&](int jl, int id) {
      const size_t at = id >= 0 ? kv8_tile(kv, id, layer, g) : 0;
      const size_t row = at * B + (id >= 0 ? key_of(jl) % B : 0);
      const uint8_t *k0 = kpool + row * D, *v0 = vpool + row * E;
#pragma unroll
      for (int i = 0; i < 4; i++) {               // rows rl, rl + 8; pieces cl, cl + 4
        const int r = rl + 8 * (i & 1), c = 16 * (cl + 4 * (i >> 1));
        ck[i] = id >= 0 && c < D ? __ldg(reinterpret_cast<const uint4*>(k0 + r * D + c)) : make_uint4(0u, 0u, 0u, 0u);
        cv[i] = id >= 0 && c < E ? __ldg(reinterpret_cast<const uint4*>(v0 + r * E + c)) : make_uint4(0u, 0u, 0u, 0u);
      }
      ks = id >= 0 ? __ldg(kv.k_scale + at) : -1.f;
      vs = id >= 0 ? __ldg(kv.v_scale + at) : 0.f;
    };
    int id_next = id_of(1);
    fetch(0, id_of(0));
    bool ok = true;
    for (int jl = 0; jl < n && ok; jl++) {
      const int st = jl % STAGES;
      uint4 k[4], v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) { k[i] = ck[i]; v[i] = cv[i]; }
      const float ks_now = ks, vs_now = vs;
      if (jl + 1 < n) fetch(jl + 1, id_next);
      id_next = id_of(jl + 2);
      if (jl >= STAGES) ok = tc_mbar_wait_warp(&kv_empty[st], (unsigned)(jl / STAGES - 1) & 1u, abort_flag);
      if (!ok) break;
      unsigned char* d = KVs + st * KV_STAGE;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = 16 * cw + rl + 8 * (i & 1), block = i >> 1;
        if (block >= KB) continue;
        unsigned char* at = d + block * (KT_KEYS * 128) + r * 128;
        const int u = 2 * cl;
        const uint32_t kw[4] = {k[i].x, k[i].y, k[i].z, k[i].w}, vw[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const uint2 a0 = kt_half4<FMT>(kw[2 * x]), a1 = kt_half4<FMT>(kw[2 * x + 1]);
          *reinterpret_cast<uint4*>(at + (((u + x) ^ (r & 7)) << 4)) = make_uint4(a0.x, a0.y, a1.x, a1.y);
          const uint2 b0 = kt_half4<FMT>(vw[2 * x]), b1 = kt_half4<FMT>(vw[2 * x + 1]);
          *reinterpret_cast<uint4*>(at + K_STAGE + (((u + x) ^ (r & 7)) << 4)) = make_uint4(b0.x, b0.y, b1.x, b1.y);
        }
      }
      if (lane == 0) { reinterpret_cast<float*>(&s_ks[st])[cw] = ks_now; reinterpret_cast<float*>(&s_vs[st])[cw] = vs_now; }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) tc_mbar_arrive(&kv_full[st]);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == KT_ISSUE && tc_elect()) {
    // ===== products
    const uint32_t id_s = kt_idesc(KT_KEYS, 0), id_o = kt_idesc(E, 1);
    const uint32_t q_addr = tc_smem_u32(Qs), kv_addr = tc_smem_u32(KVs);
    const int k_steps = D / 16;
    bool ok = true;
    auto scores = [&](int jl, int w) {
      const uint32_t d = tmem + (uint32_t)(w * 2 * KT_KEYS + (jl & 1) * KT_KEYS), k = kv_addr + (uint32_t)((jl % STAGES) * KV_STAGE);
#pragma unroll
      for (int part = SPLIT ? 1 : 0; part >= 0; part--) {   // what is small first: sums are cut off at the size of what is there
#pragma unroll
        for (int s = 0; s < DT / 16; s++) {
          if (s >= k_steps) break;
          const uint64_t ad = tc_smem_desc(q_addr + (uint32_t)((w * (SPLIT ? 2 : 1) + part) * Q_PART + (s >> 2) * KT_ROWS * 128)) + (uint64_t)(2 * (s & 3));
          const uint64_t bd = tc_smem_desc(k + (uint32_t)((s >> 2) * KT_KEYS * 128)) + (uint64_t)(2 * (s & 3));
          tc_mma_f16(d, ad, bd, id_s, (uint32_t)(s != 0 || (SPLIT && part == 0)));
        }
      }
      tc_commit(&s_full[w][jl & 1]);
    };
    ok = tc_mbar_wait(&kv_full[0], 0u, abort_flag);
    kt_fence_after();
    if (ok) { scores(0, 0); scores(0, 1); }
    for (int jl = 0; jl < n && ok; jl++) {
      if (jl + 1 < n) {
        ok = tc_mbar_wait(&kv_full[(jl + 1) % STAGES], (unsigned)((jl + 1) / STAGES) & 1u, abort_flag);
        for (int w = 0; w < 2 && ok; w++) {
          if (jl > 0) ok = tc_mbar_wait(&pv_done[w][(jl + 1) & 1], (unsigned)((jl - 1) >> 1) & 1u, abort_flag);   // the buffer's weights have been used
          kt_fence_after();
          if (ok) scores(jl + 1, w);
        }
      }
      for (int w = 0; w < 2 && ok; w++) {
        ok = tc_mbar_wait(&p_full[w][jl & 1], (unsigned)(jl >> 1) & 1u, abort_flag);
        kt_fence_after();
        if (!ok) break;
        const uint32_t d = tmem + (uint32_t)(4 * KT_KEYS + w * DT), p = tmem + (uint32_t)(w * 2 * KT_KEYS + (jl & 1) * KT_KEYS);
        const uint64_t vd = kt_desc_mn(kv_addr + (uint32_t)((jl % STAGES) * KV_STAGE + K_STAGE), KT_KEYS * 128);
#pragma unroll
        for (int x = 0; x < KT_KEYS / 16; x++) {
          tc_mma_f16_ts(d, p + (uint32_t)(8 * x), vd + (uint64_t)(x * (2048 >> 4)), id_o, (uint32_t)(((SPLIT ? jl % KT_RUN : jl) | x) != 0));
          if (SPLIT) tc_mma_f16_ts(d, p + (uint32_t)(32 + 8 * x), vd + (uint64_t)(x * (2048 >> 4)), id_o, 1u);
        }
        tc_commit(&pv_done[w][jl & 1]);
      }
      tc_commit(&kv_empty[jl % STAGES]);
    }
    }
  }
  __syncwarp();
  __syncthreads();
  kt_fence_after();
  release();
  if (threadIdx.x == 0 && abort_s && error_flag) *((volatile int*)error_flag) = 1;
}

static int kt_positions(const tha_attn_t* a) { return 2 * KT_ROWS / (a->heads / a->kv_heads); }
static long long kt_blocks(const tha_attn_t* a, const tha_rows_t* rows) { return (long long)rows->n_rows / kt_positions(a) + rows->n_seqs; }

// Parts of a context, most_tiles: of 32 keys.
int kv8_attn_tc_splits(const tha_attn_t* a, const tha_rows_t* rows, int most_tiles) {
  const long long blocks = (long long)ceil_div(rows->n_rows, kt_positions(a)) * a->kv_heads;
  long long s = 148 / blocks;
  if (s > most_tiles / 16) s = most_tiles / 16;       // eight tiles each at least
  return s < 1 ? 1 : s > 16 ? 16 : (int)s;
}

template <int DT, int FMT, bool SPLIT, bool MORE, typename T>
static int kt_launch(cudaStream_t s, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, T* out, int min_rows, int splits, float* partial,
                     const float* gate, long long ldg) {
  int* flag = nullptr;                               // allocated by a device's first call, which a capture allows in this mode
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  THA_CUDA_OK(cudaThreadExchangeStreamCaptureMode(&mode));
  const int st = gemm_tc_init(&flag);
  THA_CUDA_OK(cudaThreadExchangeStreamCaptureMode(&mode));
  THA_TRY_RC(st);
  auto k = kv8_attn_tc_kernel<DT, FMT, SPLIT, MORE, T>;
  THA_CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kt_smem(SPLIT, DT)));
  THA_CUDA_OK(launch(k, dim3(a->kv_heads, (unsigned)(kt_blocks(a, rows) * splits)), dim3(KT_THREADS), kt_smem(SPLIT, DT), s, pdl_enabled() != 0, *a, *rows, *kv, q, out,
                     kt_positions(a), min_rows, splits, partial, gate, ldg, flag));
  return THA_STATUS_SUCCESS;
}
template <int DT, bool SPLIT, typename T>
static int kt_form(cudaStream_t s, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, T* out, int min_rows, int splits, float* partial,
                   const float* gate, long long ldg) {
  const bool more = a->softcap > 0.f || a->rel;
  if (kv->format == THA_KV8_INT8)
    return more ? kt_launch<DT, THA_KV8_INT8, SPLIT, true>(s, a, rows, kv, q, out, min_rows, splits, partial, gate, ldg)
                : kt_launch<DT, THA_KV8_INT8, SPLIT, false>(s, a, rows, kv, q, out, min_rows, splits, partial, gate, ldg);
  return more ? kt_launch<DT, THA_KV8_E4M3, SPLIT, true>(s, a, rows, kv, q, out, min_rows, splits, partial, gate, ldg)
              : kt_launch<DT, THA_KV8_E4M3, SPLIT, false>(s, a, rows, kv, q, out, min_rows, splits, partial, gate, ldg);
}

int kv8_attn_tc_launch(cudaStream_t s, int dtype, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, void* out, int min_rows, int splits,
                       float* partial, const float* gate, long long ldg) {
  if (!aligned16(out) || kt_blocks(a, rows) * splits > 65535) return THA_STATUS_NOT_SUPPORTED;
  const bool wide = a->dim > 64 || a->vdim > 64;
  if (dtype == THA_DT_BF16) {
    auto o = (__nv_bfloat16*)out;
    return wide ? kt_form<128, false>(s, a, rows, kv, q, o, min_rows, splits, partial, gate, ldg) : kt_form<64, false>(s, a, rows, kv, q, o, min_rows, splits, partial, gate, ldg);
  }
  auto o = (float*)out;
  return wide ? kt_form<128, true>(s, a, rows, kv, q, o, min_rows, splits, partial, gate, ldg) : kt_form<64, true>(s, a, rows, kv, q, o, min_rows, splits, partial, gate, ldg);
}

}  // namespace tha
