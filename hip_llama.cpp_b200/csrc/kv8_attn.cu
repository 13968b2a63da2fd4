// Softmax attention over the cache in 8 bits (include/tha_hybrid.h, tha_hyb_kv8_attn): single rows, and portions of few (position, head) pairs.
//
// The bytes of the cache bound a decoded token, so a byte goes from memory to the tensor cores with as little as possible in between.  Every int8 and e4m3 code is an fp16
// number, so codes are one operand as they are; the other operand, q or the softmax weights, is fp32 and becomes two fp16, hi + lo 2^-11, that carry 22 bits of it
// (split_f16.cuh).  mma.m16n8k16 has 16 rows: eight (position, query head) pairs of one key/value head, hi in rows 0 .. 7, lo in rows 8 .. 15, so that one instruction makes
// both products and a thread finds a pair's two sums in its own registers.  The scores' layout is the one the weights enter the second product with:
// nothing of them is exchanged.
//
// A block takes eight pairs of one key/value head and a run of tiles of 32 keys, its warps every fourth tile.  A warp's tiles come through a ring in shared memory of its own
// (cp.async).  Channels of K and the order of channels in V's column groups are free, as long as both operands agree, and chosen so that
// a lane reads 16 bytes at a time and the eight lanes of a shared-memory phase meet 32 different banks (16-byte pieces of a row are stored at piece ^ (row mod 8)).
// V's scale belongs to a block of keys, the accumulator to all of them: a weight is multiplied by scale / (largest scale that its pair and warp have seen, rounded up to a
// power of two) ahead of the split; scales that a mask hides from a pair cost it nothing.  Weights have the factor 2^15, so that the 22 bits reach down to 2^-28 of the largest.
//
// Bound: the cache's bytes where nothing else is; here the instructions that turn them into fp16 pairs (int8: five for four codes of K, six of V) and the chain of a tile, which
// three blocks on an SM (168 registers at most, a ring of two tiles a warp) hide better than two (217 registers, three tiles: 15 % more on the 64 contexts below).  One context of 131072
// keys, 8 heads of 128: 66 us, 4.1 of 6.55 TB/s; 64 contexts of 3 to 2047 keys, 32 heads: 131 us, 4.1 TB/s; 16 of 501 to 8190, 8 heads, e4m3: 52 us, 2.8 TB/s (the longest are the tail).
// A unit for each pair, compared with every tile's scales, costs 1 % of that; one for a block's pairs let the scales of hidden keys take bits from a row.
#include <math.h>

#include "kv8.cuh"
#include "workspace.h"

namespace tha {

constexpr int K8_WARPS = 4, K8_THREADS = 32 * K8_WARPS, K8_PAIRS = 8, K8_KEYS = 32, K8_SEG = 256, K8_MAX_SPLITS = 64;
constexpr float K8_UP = 15.0f;   // weights: 2^(score log2(e) - maximum + 15)

template <int DT>
struct Kv8Ring {
  static constexpr int TILE = K8_KEYS * DT;                 // bytes of a tile's K, and of its V
  static constexpr int STAGES = DT == 128 ? 2 : 4;
  static constexpr int WARP = STAGES * 2 * TILE;
  static constexpr int BYTES = K8_WARPS * WARP;
};
// byte offset of 16-byte piece c of row r of a tile with DT-byte rows
template <int DT>
__device__ __forceinline__ int k8_piece(int r, int c) { return r * DT + ((DT == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4); }

__device__ __forceinline__ void k8_mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// The channels of a word of K that go to the two registers of the B operand: (0, 2) and (1, 3), or (0, 1) and (2, 3) -- what is cheapest to take apart
template <int FMT>
__device__ __forceinline__ void k8_keys(uint32_t w, uint32_t& b0, uint32_t& b1) {
  if (FMT == THA_KV8_INT8) { b0 = k8_bytes02(w); b1 = k8_bytes02(w >> 8); }
  else { b0 = k8_e4m3x2(w & 0xFFFFu); b1 = k8_e4m3x2(w >> 16); }
}
// byte i of x and of y as fp16
template <int FMT, int I>
__device__ __forceinline__ uint32_t k8_values(uint32_t x, uint32_t y) {
  if (FMT == THA_KV8_INT8) return k8_bytes02(__byte_perm(x, y, I | I << 4 | (4 + I) << 8 | (4 + I) << 12));
  return k8_e4m3x2(__byte_perm(x, y, I | (4 + I) << 4));
}

// Tiles of eight pairs of sequence s: none where it has more than `most` rows.
__device__ __forceinline__ int k8_tiles_of(const tha_rows_t& rows, int s, int gsize, int most) {
  const int n = rows.seq_first[s + 1] - rows.seq_first[s];
  return n <= most ? (n * gsize + K8_PAIRS - 1) / K8_PAIRS : 0;
}
// grid (tiles of pairs * splits, kv_heads).  Partial results of a split: sums and maxima [split][row * heads + head][2], then weighted means [..][vdim].
// FULL: heads have DT channels, keys and values alike.
template <int DT, int FMT, bool MORE, bool FULL>
__global__ void __launch_bounds__(K8_THREADS, 3) kv8_attn_kernel(tha_attn_t a, tha_rows_t rows, tha_kv8_t kv, const float* q, void* out, int out_bf16, int most_rows, int splits, int run,
                                                                 float* partial, const float* gate, long long ldg) {
  using Ring = Kv8Ring<DT>;
  constexpr float LOG2E = 1.4426950408889634f;
  constexpr int KS = DT / 16;                               // k steps of the scores
  constexpr int NV = DT / 8;                                // column groups of the accumulator
  extern __shared__ __align__(128) unsigned char k8_ring[];
  __shared__ uint4 s_q[KS][32];                             // q as the A operand of every step, a lane's registers together
  __shared__ int s_tile[2 * K8_SEG];                        // per 16 keys of a segment's tiles: (block, layer, head), -1 where they do not exist, and the scales
  __shared__ float s_ks[2 * K8_SEG], s_vs[2 * K8_SEG];
  __shared__ float s_ml[K8_WARPS][K8_PAIRS][3];             // maximum, sum, unit
  const int D = FULL ? DT : a.dim, E = FULL ? DT : a.vdim, gsize = a.heads / a.kv_heads, B = kv.block_size, layer = a.cache_layer;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  hyb_pdl_enter();
  const int kvh = blockIdx.y, sp = blockIdx.x % splits;
  int seq, tile;
  {
    const int i = blockIdx.x / splits, per = (gsize + K8_PAIRS - 1) / K8_PAIRS;
    if (rows.max_seq_rows == 1) {
      seq = i / per; tile = i - seq * per;
    } else {
      const Kv8Piece pc = kv8_find(rows.n_seqs, i, [&](int s) { return k8_tiles_of(rows, s, gsize, most_rows); });
      seq = pc.seq; tile = pc.at;
    }
  }
  if (seq < 0) return;
  // What a block waits for ahead of its first tile is a chain of loads: positions, block ids, codes.  With every sequence a row the first row of one is its number, and the
  // scales and q's parts are made while the first codes are on their way.
  const bool singles = rows.max_seq_rows == 1;
  const int r0 = singles ? seq : rows.seq_first[seq], n_rows = singles ? 1 : rows.seq_first[seq + 1] - r0, slot = rows.seq_slot[seq];
  const int pairs = min(K8_PAIRS, n_rows * gsize - tile * K8_PAIRS);
  if (pairs < 1) return;
  const int pr = tile * K8_PAIRS + min(g, pairs - 1), pp = pr / gsize, head = kvh * gsize + (pr - pp * gsize);   // this lane's pair (behind the last: the last again)
  const int p_seq = rows.pos[r0];
  if (!FULL)                                                // channels past the head's are zeros that no copy touches
    for (int i = threadIdx.x; i < Ring::BYTES / 16; i += K8_THREADS) reinterpret_cast<uint4*>(k8_ring)[i] = make_uint4(0u, 0u, 0u, 0u);
  const int p_first = p_seq + (tile * K8_PAIRS) / gsize, p_last = p_seq + (tile * K8_PAIRS + pairs - 1) / gsize, pos = p_seq + pp;
  const int key_lo = a.chunk > 0 ? (p_first / a.chunk) * a.chunk : 0, last_lo = a.chunk > 0 ? (p_last / a.chunk) * a.chunk : 0;
  const int my_lo = a.chunk > 0 ? (pos / a.chunk) * a.chunk : 0;
  HybTiles tiles = {0, 0, 0, 0};
  if (p_seq >= 0) tiles = hyb_attn_tiles(a, key_lo, p_first, p_last);
  const int ti0 = min(sp * run, tiles.n), ti1 = sp == splits - 1 ? tiles.n : min(ti0 + run, tiles.n);
  auto tile_key = [&](int ti) { return ti < tiles.n_a ? tiles.begin + 32 * ti : tiles.resume + 32 * (ti - tiles.n_a); };

  // q's parts as operands, and the factor of its scores: a lane's channels of its pair are those it reads of a key
  float fac = 0.f;
  auto make_q = [&]() {
    const float* qr = q + ((size_t)(r0 + pp) * a.heads + head) * D;
    float v[KS][4], top = 0.f;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const int c = (DT == 128 ? 2 * t + (s >> 2) : t) * 16 + (s & 3) * 4;
      const float4 x = c < D ? *reinterpret_cast<const float4*>(qr + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[s][0] = x.x; v[s][1] = x.y; v[s][2] = x.z; v[s][3] = x.w;
    }
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(v[s][i]));
    top = fmaxf(top, __shfl_xor_sync(THA_FULL_MASK, top, 1));
    top = fmaxf(top, __shfl_xor_sync(THA_FULL_MASK, top, 2));
    float inverse;
    const float up = split_scale<100>(top, 14, &inverse);
    constexpr int X = FMT == THA_KV8_INT8 ? 2 : 1, Y = FMT == THA_KV8_INT8 ? 1 : 2;   // k8_keys
    if (warp == 0) {                                        // all warps have the same
#pragma unroll
      for (int s = 0; s < KS; s++) {
        uint4 f;
        split_f16x2(make_float2(v[s][0], v[s][X]), up, f.x, f.y);
        split_f16x2(make_float2(v[s][Y], v[s][3]), up, f.z, f.w);
        s_q[s][lane] = f;
      }
    }
    fac = inverse * a.scale * (a.head_scale ? a.head_scale[head] : 1.0f) * (MORE ? 1.0f : LOG2E);
  };

  float acc[NV][4];
#pragma unroll
  for (int i = 0; i < NV; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  float m = -INFINITY, l = 0.f, ref = 0.f, down = 0.f;      // l: this lane's keys only; ref: the unit of this lane's pair and its warp, 1 / down
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(k8_ring) + warp * Ring::WARP;
  const int lane_r = lane / (DT / 16), lane_c = lane % (DT / 16);   // the row and piece of 512 bytes of a tile that this lane copies
  const uint32_t lane_to = (uint32_t)k8_piece<DT>(lane_r, lane_c);
  const bool k_there = 16 * lane_c < D, v_there = 16 * lane_c < E;
  const size_t k_tile = (size_t)B * D, v_tile = (size_t)B * E;
  const uint8_t *kpool = static_cast<const uint8_t*>(kv.k_pool) + lane_r * D + 16 * lane_c, *vpool = static_cast<const uint8_t*>(kv.v_pool) + lane_r * E + 16 * lane_c;

  // The tensor cores cut off what their fp32 sums cannot hold: an accumulator sums a segment's tiles, 128 sums a warp, and the segments' are added here.
  float seg_total[2 * NV], m_total = -INFINITY, ref_total = 0.f;
  float* total = seg_total;
  asm volatile("" : "+l"(total));                           // local memory: few contexts have a second segment
  auto add_segment = [&]() {
    const float f = m_total > -INFINITY ? hyb_ex2(m_total - m) * (ref > 0.f ? ref_total / ref : 0.f) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int x = 0; x < 2; x++) {
        acc[i][x] = fmaf(acc[i][2 + x], SPLIT_DOWN, acc[i][x]);
        if (f != 0.f) acc[i][x] = fmaf(f, total[2 * i + x], acc[i][x]);
        acc[i][2 + x] = 0.f;
      }
  };
  for (int s0 = ti0; s0 < ti1; s0 += K8_SEG) {
    const int s1 = min(s0 + K8_SEG, ti1);
    if (s0 > ti0) {
      add_segment();
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int x = 0; x < 2; x++) { total[2 * i + x] = acc[i][x]; acc[i][x] = 0.f; }
      m_total = m; ref_total = ref;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * (s1 - s0); e += K8_THREADS) {
      const int key = tile_key(s0 + (e >> 1)) + 16 * (e & 1);
      const int id = key <= p_last ? kv8_block(kv, slot, key) : -1;
      s_tile[e] = id >= 0 ? (int)kv8_tile(kv, id, layer, kvh) : -1;   // a tile has 256 bytes at least: they are below 2^31 in any memory
    }
    __syncthreads();
    auto fetch = [&](int ti, int stage) {                   // every lane's share of a tile; nothing behind the segment's last
      if (ti >= s1) return;
      const int e = 2 * (ti - s0), in_block = tile_key(ti) & (B - 1);
      const uint32_t dst = ring + stage * 2 * Ring::TILE;
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        const int tile = s_tile[e + hf], row = (in_block + 16 * hf) & (B - 1);
        const bool there = tile >= 0;
        const uint8_t *ks = kpool + (there ? (size_t)(unsigned)tile * k_tile + row * D : 0), *vs = vpool + (there ? (size_t)(unsigned)tile * v_tile + row * E : 0);
#pragma unroll
        for (int i = 0; i < DT / 32; i++) {                 // rows lane_r, lane_r + STEP, ..: the piece's place turns with the row
          constexpr int STEP = 512 / DT;
          const int turn = DT == 128 ? (i & 1) * 64 : 0;
          const uint32_t to = dst + (16 * hf + STEP * i) * DT + (lane_to ^ turn);
          if (FULL || k_there) hyb_copy16(to, ks + STEP * i * D, there ? 16 : 0);
          if (FULL || v_there) hyb_copy16(to + Ring::TILE, vs + STEP * i * E, there ? 16 : 0);
        }
      }
    };
#pragma unroll
    for (int i = 0; i < Ring::STAGES - 1; i++) { fetch(s0 + warp + i * K8_WARPS, i); hyb_copies_end(); }
    for (int e = threadIdx.x; e < 2 * (s1 - s0); e += K8_THREADS) {
      const int at = s_tile[e];
      s_ks[e] = at >= 0 ? kv.k_scale[at] : 0.f;
      s_vs[e] = at >= 0 ? kv.v_scale[at] : 0.f;
    }
    if (s0 == ti0) make_q();
    __syncthreads();

    int stage = 0;
    for (int ti = s0 + warp; ti < s1; ti += K8_WARPS) {
      fetch(ti + (Ring::STAGES - 1) * K8_WARPS, stage == 0 ? Ring::STAGES - 1 : stage - 1);
      hyb_copies_end();
      hyb_copies_await<Ring::STAGES - 1>();
      __syncwarp();
      const unsigned char* st = k8_ring + warp * Ring::WARP + stage * 2 * Ring::TILE;
      const int e = 2 * (ti - s0), kt = tile_key(ti);
      // scores: 16 bytes of each of the lane's four keys at a time, q of a step read once for them
      float sc[4][4];
#pragma unroll
      for (int j = 0; j < 4; j++) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
      for (int pcs = 0; pcs < DT / 64; pcs++) {
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = *reinterpret_cast<const uint4*>(st + k8_piece<DT>(8 * j + g, DT == 128 ? 2 * t + pcs : t));
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const uint4 qf = s_q[4 * pcs + x][lane];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            uint32_t b0, b1;
            k8_keys<FMT>(x == 0 ? w[j].x : x == 1 ? w[j].y : x == 2 ? w[j].z : w[j].w, b0, b1);
            k8_mma(sc[j], qf, b0, b1);
          }
        }
      }
      const float f0 = fac * s_ks[e], f1 = fac * s_ks[e + 1];
      const bool there0 = s_tile[e] >= 0, there1 = s_tile[e + 1] >= 0;
      const bool whole = there0 && there1 && kt + 31 <= p_first && kt >= last_lo && (a.window <= 0 || p_last - kt < a.window || kt + 32 <= a.keep_first);
      float2 x[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float f = j < 2 ? f0 : f1;
        x[j] = f32x2_mul(f32x2_fma(make_float2(sc[j][2], sc[j][3]), make_float2(SPLIT_DOWN, SPLIT_DOWN), make_float2(sc[j][0], sc[j][1])), make_float2(f, f));
        if (MORE) {
          const int key = kt + 8 * j + 2 * t;
          if (a.softcap > 0.f) { x[j].x = hyb_softcap(x[j].x, a.softcap); x[j].y = hyb_softcap(x[j].y, a.softcap); }
          if (a.rel) { x[j].x += hyb_attn_rel(a, head, pos - key); x[j].y += hyb_attn_rel(a, head, pos - key - 1); }
          x[j].x = k8_log2_units(x[j].x); x[j].y = k8_log2_units(x[j].y);
        }
      }
      float v0 = s_vs[e], v1 = s_vs[e + 1];                  // of what this lane's pair sees: a weight of 0 under a scale far above the pair's unit is no number
      if (!whole) {
        uint32_t seen = kv8_sees32(a, kt, pos, my_lo);
        if (!there0) seen &= 0xFFFF0000u;
        if (!there1) seen &= 0xFFFFu;
        if (!(seen & 0xFFFFu)) v0 = 0.f;
        if (!(seen >> 16)) v1 = 0.f;
        seen >>= 2 * t;                                      // bits 8 j, 8 j + 1 are this lane's
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (!(seen >> (8 * j) & 1u)) x[j].x = -INFINITY;
          if (!(seen >> (8 * j + 1) & 1u)) x[j].y = -INFINITY;
        }
      }
      float top_x = k8_max3(k8_max3(x[0].x, x[0].y, x[1].x), k8_max3(x[1].y, x[2].x, x[2].y), fmaxf(x[3].x, x[3].y));
      top_x = fmaxf(top_x, __shfl_xor_sync(THA_FULL_MASK, top_x, 1));
      top_x = fmaxf(top_x, __shfl_xor_sync(THA_FULL_MASK, top_x, 2));
      const float top_v = fmaxf(v0, v1);
      const bool grow = top_x > m, wider = top_v > ref;
      if (__any_sync(THA_FULL_MASK, grow || wider)) {
        const float to = grow ? top_x : m;
        float corr = m > -INFINITY ? hyb_ex2(m - to) : grow ? 0.f : 1.f;
        m = to;
        l *= corr;
        if (wider) {                                         // up to the next power of two: what is there changes units exactly
          const float unit = __uint_as_float(min((__float_as_uint(top_v) + 0x7FFFFFu) & 0x7F800000u, 0x7E800000u));
          corr *= ref / unit;
          ref = unit;
          down = 1.0f / unit;
        }
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
          for (int y = 0; y < 4; y++) acc[i][y] *= corr;
      }
      const float shift = m > -INFINITY ? (MORE ? -m : K8_UP - m) : 0.f;   // nothing seen so far: weights are 2^-inf; MORE: next to a maximum of 2^127, 15 is nothing
      v0 *= down; v1 *= down;
      uint4 pf[2];
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        float2 y = k8_add2(x[j], make_float2(shift, shift));
        if (MORE) y = k8_add2(y, make_float2(K8_UP, K8_UP));
        const float2 w = make_float2(hyb_ex2(y.x), hyb_ex2(y.y));
        sum = k8_add2(sum, w);
        split_f16x2(f32x2_mul(w, j < 2 ? make_float2(v0, v0) : make_float2(v1, v1)), 1.0f, j & 1 ? pf[j >> 1].z : pf[j >> 1].x, j & 1 ? pf[j >> 1].w : pf[j >> 1].y);
      }
      l += sum.x + sum.y;
      // weights x values: 16 keys at a time
      const unsigned char* sv = st + Ring::TILE;
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        const int k0 = 16 * kk + 2 * t;
        if (DT == 128) {
          const uint4 wa = *reinterpret_cast<const uint4*>(sv + k8_piece<DT>(k0, g)), wb = *reinterpret_cast<const uint4*>(sv + k8_piece<DT>(k0 + 1, g));
          const uint4 wc = *reinterpret_cast<const uint4*>(sv + k8_piece<DT>(k0 + 8, g)), wd = *reinterpret_cast<const uint4*>(sv + k8_piece<DT>(k0 + 9, g));
          const uint32_t A[4] = {wa.x, wa.y, wa.z, wa.w}, Bw[4] = {wb.x, wb.y, wb.z, wb.w}, C[4] = {wc.x, wc.y, wc.z, wc.w}, Dw[4] = {wd.x, wd.y, wd.z, wd.w};
#pragma unroll
          for (int w = 0; w < NV / 4; w++) {
            k8_mma(acc[4 * w], pf[kk], k8_values<FMT, 0>(A[w], Bw[w]), k8_values<FMT, 0>(C[w], Dw[w]));
            k8_mma(acc[4 * w + 1], pf[kk], k8_values<FMT, 1>(A[w], Bw[w]), k8_values<FMT, 1>(C[w], Dw[w]));
            k8_mma(acc[4 * w + 2], pf[kk], k8_values<FMT, 2>(A[w], Bw[w]), k8_values<FMT, 2>(C[w], Dw[w]));
            k8_mma(acc[4 * w + 3], pf[kk], k8_values<FMT, 3>(A[w], Bw[w]), k8_values<FMT, 3>(C[w], Dw[w]));
          }
        } else {
          auto two = [&](int r) { return *reinterpret_cast<const uint2*>(sv + k8_piece<DT>(r, g >> 1) + 8 * (g & 1)); };
          const uint2 wa = two(k0), wb = two(k0 + 1), wc = two(k0 + 8), wd = two(k0 + 9);
          const uint32_t A[2] = {wa.x, wa.y}, Bw[2] = {wb.x, wb.y}, C[2] = {wc.x, wc.y}, Dw[2] = {wd.x, wd.y};
#pragma unroll
          for (int w = 0; w < NV / 4; w++) {
            k8_mma(acc[4 * w], pf[kk], k8_values<FMT, 0>(A[w], Bw[w]), k8_values<FMT, 0>(C[w], Dw[w]));
            k8_mma(acc[4 * w + 1], pf[kk], k8_values<FMT, 1>(A[w], Bw[w]), k8_values<FMT, 1>(C[w], Dw[w]));
            k8_mma(acc[4 * w + 2], pf[kk], k8_values<FMT, 2>(A[w], Bw[w]), k8_values<FMT, 2>(C[w], Dw[w]));
            k8_mma(acc[4 * w + 3], pf[kk], k8_values<FMT, 3>(A[w], Bw[w]), k8_values<FMT, 3>(C[w], Dw[w]));
          }
        }
      }
      __syncwarp();                                          // the stage has been read
      stage = stage + 1 == Ring::STAGES ? 0 : stage + 1;
    }
    hyb_copies_await<0>();
  }

  add_segment();

  // The warps meet: accumulators over the ring, [warp][column group][pair][8 columns], the groups two words apart in the banks: neither a warp's pairs of columns nor a pair's
  // channels meet in one.  (As [pair][channel] all 32 lanes met in a bank, and a block took 5 us beside its keys.)
  constexpr int GROUP = 8 * K8_PAIRS + 2;
  l += __shfl_xor_sync(THA_FULL_MASK, l, 1);
  l += __shfl_xor_sync(THA_FULL_MASK, l, 2);
  __syncthreads();
  float* s_acc = reinterpret_cast<float*>(k8_ring);
  if (t == 0) { s_ml[warp][g][0] = l == l ? m : l; s_ml[warp][g][1] = l; s_ml[warp][g][2] = ref; }   // a NaN among the scores shows in the sum alone
#pragma unroll
  for (int i = 0; i < NV; i++)                               // columns 2 t, 2 t + 1 of group i are channels 2 t * DT / 8 + i, (2 t + 1) * DT / 8 + i
    *reinterpret_cast<float2*>(s_acc + (warp * NV + i) * GROUP + g * 8 + 2 * t) = make_float2(acc[i][0], acc[i][1]);
  __syncthreads();
  for (int w = warp; w < pairs; w += K8_WARPS) {
    const int pr2 = tile * K8_PAIRS + w, pp2 = pr2 / gsize, h2 = kvh * gsize + (pr2 - pp2 * gsize), r = r0 + pp2;
    float M = -INFINITY, L = 0.f, f[K8_WARPS];
#pragma unroll
    for (int x = 0; x < K8_WARPS; x++) M = s_ml[x][w][0] > M || s_ml[x][w][0] != s_ml[x][w][0] ? s_ml[x][w][0] : M;
#pragma unroll
    for (int x = 0; x < K8_WARPS; x++) {
      f[x] = s_ml[x][w][0] > -INFINITY ? exp2f(s_ml[x][w][0] - M) : 0.f;
      L += f[x] * s_ml[x][w][1];
    }
    L *= exp2f(-K8_UP);
    float scale = exp2f(-K8_UP);
    const size_t at = (size_t)r * a.heads + h2, all = (size_t)rows.n_rows * a.heads;
    float* pd = splits > 1 ? partial + k8_sums_floats(splits, all) + ((size_t)sp * all + at) * E : nullptr;
    scale *= pd ? (L > 0.f ? 1.0f / L : L) : k8_final(a, h2, M, L, gate ? gate + (size_t)r * ldg : nullptr);   // a part is a mean: sums of values beyond 2^118 are not finite
    if (pd && lane == 0) { float* ml = partial + 2 * ((size_t)sp * all + at); ml[0] = M; ml[1] = L; }
#pragma unroll
    for (int x = 0; x < K8_WARPS; x++) f[x] *= scale;
    for (int c = lane; c < E; c += 32) {
      float o = 0.f;
#pragma unroll
      for (int x = 0; x < K8_WARPS; x++) o += s_acc[(x * NV + c % NV) * GROUP + w * 8 + c / NV] * f[x] * s_ml[x][w][2];
      if (pd) pd[c] = o;
      else if (out_bf16) reinterpret_cast<__nv_bfloat16*>(out)[at * E + c] = __float2bfloat16_rn(o);
      else reinterpret_cast<float*>(out)[at * E + c] = o;
    }
  }
}

// The parts of a (row, head), of sequences of least .. most rows, four channels a lane.  WARPS 1: a warp has them all, in order; 4: a block, every fourth to a warp (many parts of few rows:
// one after the other they took 12 us).  grid (rows * heads * WARPS / 4)
template <int WARPS, typename T>
__global__ void __launch_bounds__(128) kv8_merge_kernel(T* out, const float* partial, tha_rows_t rows, int least, int most, int splits, tha_attn_t a, const float* gate, long long ldg) {
  hyb_pdl_enter();
  __shared__ float4 s_o[WARPS][32];
  const int warp = threadIdx.x >> 5, w0 = WARPS == 1 ? 0 : warp;
  const size_t at = (size_t)blockIdx.x * (4 / WARPS) + (WARPS == 1 ? warp : 0), all = (size_t)rows.n_rows * a.heads;
  if (at >= all) return;
  const int E = a.vdim, lane = threadIdx.x & 31, row = (int)(at / a.heads), h = (int)(at - (size_t)row * a.heads);
  const int seq = rows.row_seq[row], n = rows.seq_first[seq + 1] - rows.seq_first[seq];
  if (n < least || n > most) return;
  static_assert(K8_MAX_SPLITS == 64, "two parts a lane");
  float m[2], l[2], w[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int s = lane + 32 * i;
    const float2 ml = s < splits ? *reinterpret_cast<const float2*>(partial + 2 * ((size_t)s * all + at)) : make_float2(-INFINITY, 0.f);
    m[i] = ml.x; l[i] = ml.y;
  }
  const float* p = partial + k8_sums_floats(splits, all) + at * E + 4 * lane;
  const bool mine = 4 * lane < E, nan = __any_sync(THA_FULL_MASK, m[0] != m[0] || m[1] != m[1]);
  const float M = warp_max(fmaxf(m[0], m[1]));
#pragma unroll
  for (int i = 0; i < 2; i++) w[i] = m[i] > -INFINITY ? exp2f(m[i] - M) : 0.f;
  const float L = warp_sum(w[0] * l[0] + w[1] * l[1]), inv = L > 0.f ? 1.0f / L : 0.f;
#pragma unroll
  for (int i = 0; i < 2; i++) w[i] *= l[i] * inv;           // of the parts' means
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = w0; s < splits; s += WARPS) {
    const float ws = __shfl_sync(THA_FULL_MASK, s < 32 ? w[0] : w[1], s & 31);
    if (ws > 0.f && mine) {                                 // parts that saw nothing hold nothing
      const float4 v = *reinterpret_cast<const float4*>(p + (size_t)s * all * E);
      o.x = fmaf(v.x, ws, o.x); o.y = fmaf(v.y, ws, o.y); o.z = fmaf(v.z, ws, o.z); o.w = fmaf(v.w, ws, o.w);
    }
  }
  if (WARPS > 1) {                                          // the whole block is one (row, head): it comes here as one
    s_o[w0][lane] = o;
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int i = 1; i < WARPS; i++) {
      const float4 v = s_o[i][lane];
      o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
    }
  }
  if (!mine) return;
  const float f = k8_final(a, h, nan ? NAN : M, L, gate ? gate + (size_t)row * ldg : nullptr) * L;
  const float v[4] = {o.x * f, o.y * f, o.z * f, o.w * f};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (a.out_f32) reinterpret_cast<float*>(out)[at * E + 4 * lane + i] = v[i];
    else k8_store(out + at * E + 4 * lane + i, v[i]);
  }
}

// Keys that the row of the longest context sees at most, as tiles of 32.
static int k8_most_tiles(const tha_attn_t* a, const tha_rows_t* rows) {
  const long long seen = rows->max_pos + 1ll;
  long long keys = a->chunk > 0 ? (long long)a->chunk + rows->max_seq_rows : seen;
  if (a->window > 0 && (long long)a->window + a->keep_first + rows->max_seq_rows + 64 < keys) keys = (long long)a->window + a->keep_first + rows->max_seq_rows + 64;
  if (keys > seen) keys = seen;
  return (int)((keys + 31) / 32) + 1;
}
// Pair tiles of the sequences of up to `most` rows, at most.
static int k8_pair_tiles(const tha_attn_t* a, const tha_rows_t* rows, int most) {
  const int gsize = a->heads / a->kv_heads;
  if (rows->max_seq_rows == 1) return rows->n_seqs * ceil_div(gsize, K8_PAIRS);
  const long long by_rows = (long long)rows->n_rows * gsize / K8_PAIRS + rows->n_seqs;
  const long long by_seqs = (long long)rows->n_seqs * (((long long)(most < rows->max_seq_rows ? most : rows->max_seq_rows) * gsize + K8_PAIRS - 1) / K8_PAIRS);
  return (int)(by_rows < by_seqs ? by_rows : by_seqs);
}
// Parts of a context.  Three blocks run at once on an SM, 444 on 148; a block takes the time of six tiles of 32 keys (4 us) beside its own, the meeting of the parts as much.  One context:
// rounds of whole parts.  Several: their lengths are between nothing and the longest, blocks follow one another as they end, and the last of them is the tail.  us (of an
// earlier state, 2 % less than now) with 1 / 2 / 4 / 6 / 10 / 20 parts, heads of 128: 64 contexts up to 2048 of 32 heads 125 / 136 / 162 / 192; 16 up to 8192 of 8 heads (3 parts: 69) 56 (4) / 50 / 51 / 59; one of 131072 of 8 heads with 18 /
// 37 / 55 / 64 parts 145 / 83 / 63 / 74.
static int k8_splits(const tha_attn_t* a, const tha_rows_t* rows, int most_rows) {
  const int SLOTS = 3 * sm_budget();
  constexpr float BESIDE = 6.f;
  const int most = k8_most_tiles(a, rows);
  const long long blocks = (long long)k8_pair_tiles(a, rows, most_rows) * a->kv_heads;
  // kv8_merge_kernel passes every row of the step: 2700 (row, head) a tile's time.  Rows of longer sequences, which it leaves as they are, count here: two prompts of 777 and 2048
  // rows, 32 heads, whose step may hold short portions but does not, took 115 us with such a pass and take 91 without.
  const long long rows_short = (long long)rows->n_seqs * (most_rows < rows->max_seq_rows ? most_rows : rows->max_seq_rows);
  const float passed = rows->n_rows > rows_short ? (float)(rows->n_rows - rows_short) * a->heads / 2700.f : 0.f;
  int best = 1;
  float least = 0.f;
  for (int s = 1; s <= K8_MAX_SPLITS && (s == 1 || s * 4 <= most); s++) {   // a tile for each warp at least
    const float run = (float)ceil_div(most, s) + BESIDE;
    float cost;
    if (rows->n_seqs == 1) {
      cost = (float)((blocks * s + SLOTS - 1) / SLOTS) * run;
    } else {
      cost = (float)blocks * (0.5f * most + BESIDE * s) / SLOTS + 0.5f * run;
      if (cost < run) cost = run;
    }
    if (s > 1) cost += BESIDE + passed;
    if (s == 1 || cost < least) { least = cost; best = s; }
  }
  return best;
}

template <typename T>
static int k8_merge(cudaStream_t s, const tha_attn_t* a, const tha_rows_t* rows, T* out, int least, int most, int splits, const float* partial, const float* gate, long long ldg) {
  const unsigned all = (unsigned)rows->n_rows * a->heads;
  if (splits > 8)
    THA_CUDA_OK(launch(kv8_merge_kernel<4, T>, dim3(all), dim3(128), 0, s, pdl_enabled() != 0, out, partial, *rows, least, most, splits, *a, gate, ldg));
  else if (splits > 1)
    THA_CUDA_OK(launch(kv8_merge_kernel<1, T>, dim3((all + 3) / 4), dim3(128), 0, s, pdl_enabled() != 0, out, partial, *rows, least, most, splits, *a, gate, ldg));
  return THA_STATUS_SUCCESS;
}
template <int DT, int FMT, bool MORE, bool FULL>
static int k8_launch(cudaStream_t s, int dtype, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, void* out, int most_rows, int splits,
                     float* partial, const float* gate, long long ldg) {
  auto k = kv8_attn_kernel<DT, FMT, MORE, FULL>;
  THA_CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Kv8Ring<DT>::BYTES));
  const int run = ceil_div(k8_most_tiles(a, rows), splits);
  THA_CUDA_OK(launch(k, dim3((unsigned)k8_pair_tiles(a, rows, most_rows) * splits, a->kv_heads), dim3(K8_THREADS), Kv8Ring<DT>::BYTES, s, pdl_enabled() != 0, *a, *rows, *kv, q,
                     out, (int)(dtype == THA_DT_BF16 && !a->out_f32), most_rows, splits, run, partial, gate, ldg));
  return THA_STATUS_SUCCESS;
}
template <int DT, int FMT>
static int k8_form(cudaStream_t s, int dtype, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, void* out, int most_rows, int splits,
                   float* partial, const float* gate, long long ldg) {
  const bool more = a->softcap > 0.f || a->rel, full = a->dim == DT && a->vdim == DT;
  if (more) return full ? k8_launch<DT, FMT, true, true>(s, dtype, a, rows, kv, q, out, most_rows, splits, partial, gate, ldg)
                        : k8_launch<DT, FMT, true, false>(s, dtype, a, rows, kv, q, out, most_rows, splits, partial, gate, ldg);
  return full ? k8_launch<DT, FMT, false, true>(s, dtype, a, rows, kv, q, out, most_rows, splits, partial, gate, ldg)
              : k8_launch<DT, FMT, false, false>(s, dtype, a, rows, kv, q, out, most_rows, splits, partial, gate, ldg);
}
// Which sequences take which form.  short_rows: up to so many rows take kv8_attn_kernel; has_short, has_long: whether the step may hold any.
struct Kv8Forms { int short_rows; bool has_short, has_long; };
// The two forms' times, in us, for n_seqs sequences of n rows that see `keys` keys at most, as both were measured over 1136 steps of 1 to 16 portions of 4 to 512 rows behind 0 to 70000 keys,
// 2 to 64 heads on 1 to 32, 64 and 128 channels, both result types.  kv8_attn_kernel: 14.5, and 0.72 (heads up to 64 channels: 0.41) for a tile of 32 keys of one of 444 blocks, six of them
// beside its keys.  kv8_attn_tc_kernel: 17, 1.45 for 10000 staged keys of a head, 8 where contexts are cut, and for a tile of 64 keys of a block on one of 148 SMs 1.0 (128 pairs, one fp16 an
// operand) or 3.1 (256 pairs, two), but 0.5 or 1.2 for each of a block's own tiles at least; with 64 channels 0.64 and 1.15 (128 pairs).  What is chosen so is 0.6 % slower than the faster
// form on the geometric mean, more than 10 % for 33 of the 1136, 48 % at worst (12 heads of 64, 256 rows, fp32: 38 for 26).  Model / measured, short and long: 32 heads of 128, 128 rows 22 / 22
// and 18 / 17, 512 rows 64 / 65 and 23 / 28, 128 rows behind 4000 keys 126 / 140 and 58 / 60; 16 on 4, 64 rows behind 4000 keys 42 / 46 and 31 / 34; 256 rows 24 / 24 and 18 / 20.
static bool k8_long_pays(const tha_attn_t* a, const tha_rows_t* rows, int dtype, long long keys, int n) {
  const int gsize = a->heads / a->kv_heads;
  const bool wide = a->dim > 64 || a->vdim > 64, exact = kv8_exact(a, dtype);
  const float seqs = (float)rows->n_seqs, pairs = (float)n * gsize, seen = keys > n ? (float)keys - 0.5f * n : 0.5f * keys, sms = (float)sm_budget();
  const float as_short = 14.5f + (wide ? 0.72f : 0.41f) * ceilf(pairs / K8_PAIRS) * a->kv_heads * seqs * (seen / 32.f + 6.f) / (3.f * sms);
  const float blocks = ceilf(pairs / (wide && exact ? 256.f : 128.f)) * a->kv_heads * seqs;
  float cut = floorf((wide && exact ? 1.f : 2.f) * sms / blocks);   // kv8_attn_tc_splits
  cut = fmaxf(1.f, fminf(fminf(cut, (float)(keys / (32 * 16))), 16.f));
  const float tiles = (wide ? (exact ? 3.1f : 1.0f) : (exact ? 1.15f : 0.64f)) * blocks * (seen / 64.f) / sms, alone = wide ? (exact ? 1.2f : 0.5f) * ceilf(seen / 64.f / cut) : 0.f;
  const float as_long = 17.f + 1.45e-4f * (wide ? 1.f : 0.5f) * keys * a->kv_heads * seqs + (cut > 1.f ? 8.f : 0.f) + fmaxf(tiles, alone);
  return as_long < as_short;
}
static Kv8Forms k8_forms(const tha_attn_t* a, const tha_rows_t* rows, int dtype) {
  Kv8Forms f = {0x7FFFFFFF, true, false};
  if (a->heads / a->kv_heads > 128 || rows->max_seq_rows < 2) return f;
  const long long keys = 32ll * k8_most_tiles(a, rows);
  for (int n = 2;; n = n + n / 4 + 1) {
    if (n > rows->max_seq_rows) n = rows->max_seq_rows;
    if (k8_long_pays(a, rows, dtype, keys, n)) { f.short_rows = n - 1; f.has_long = true; break; }
    if (n == rows->max_seq_rows) break;
  }
  if (f.has_long) {   // all sequences that might be long have to find room: where they do not, the shorter of them are short
    const int room = kv8_attn_tc_room_for(a, (int)(keys / 32));
    if (rows->n_seqs > room && rows->n_rows / (f.short_rows + 1) > room) f.short_rows = rows->n_rows / (room + 1);
    if (room < 1 || f.short_rows >= rows->max_seq_rows) { f.short_rows = 0x7FFFFFFF; f.has_long = false; }
  }
  f.has_short = !(f.has_long && (long long)rows->n_seqs * rows->max_seq_rows == rows->n_rows);   // all sequences are as long as the longest
  return f;
}
template <typename T>
static int k8_attend(cudaStream_t s, int dtype, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, T* out, float* scratch, size_t room,
                     const float* gate, long long ldg) {
  const Kv8Forms f = k8_forms(a, rows, dtype);
  const size_t all = (size_t)rows->n_rows * a->heads;
  auto fit = [&](int splits, size_t room) {
    while (splits > 1 && k8_partial_floats(splits, all, a->vdim) > room) splits--;
    return splits;
  };
  int short_rows = f.short_rows;
  if (f.has_long) {
    // tiles in fp16 first, partial results behind them
    const int most = k8_most_tiles(a, rows);
    const size_t stage = kv8_attn_tc_stage_bytes(a, rows, most, short_rows + 1) / sizeof(float);
    int st = THA_STATUS_NOT_SUPPORTED;
    if (scratch && stage && stage <= room) {
      const int splits = fit(kv8_attn_tc_splits(a, rows, dtype, most), room - stage);
      st = kv8_attn_tc_launch(s, dtype, a, rows, kv, q, out, short_rows + 1, most, splits, scratch, scratch + stage, gate, ldg);
      if (st == THA_STATUS_SUCCESS) {
        THA_TRY_RC(k8_merge(s, a, rows, out, short_rows + 1, 0x7FFFFFFF, splits, scratch + stage, gate, ldg));
        if (!f.has_short) return THA_STATUS_SUCCESS;
      }
    }
    if (st == THA_STATUS_NOT_SUPPORTED) short_rows = 0x7FFFFFFF;
    else if (st != THA_STATUS_SUCCESS) return st;
  }
  const int splits = scratch ? fit(k8_splits(a, rows, short_rows), room) : 1;
  const bool wide = a->dim > 64 || a->vdim > 64;
  if (kv->format == THA_KV8_INT8)
    THA_TRY_RC((wide ? k8_form<128, THA_KV8_INT8> : k8_form<64, THA_KV8_INT8>)(s, dtype, a, rows, kv, q, out, short_rows, splits, scratch, gate, ldg));
  else
    THA_TRY_RC((wide ? k8_form<128, THA_KV8_E4M3> : k8_form<64, THA_KV8_E4M3>)(s, dtype, a, rows, kv, q, out, short_rows, splits, scratch, gate, ldg));
  return k8_merge(s, a, rows, out, 0, short_rows, splits, scratch, gate, ldg);
}
static int k8_check(const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const char* who) {
  THA_TRY_RC(kv8_check(rows, kv, a->cache_layer, who));
  if (a->kv_heads != kv->kv_heads || a->dim != kv->dim || a->vdim != kv->vdim) return kv8_refuse(who, "heads or channels are not the cache's");
  if (a->heads < 1 || a->heads % a->kv_heads) return kv8_refuse(who, "query heads are a multiple of the key/value heads");
  if (a->window < 0 || a->keep_first < 0 || a->chunk < 0) return kv8_refuse(who, "a mask's extent is below 0");
  if (a->rel && a->rel_n < 1) return kv8_refuse(who, "distance biases without an extent");
  if (a->values_in_keys || a->v_share > 1 || a->diff) {
    kv8_refuse(who, "values_in_keys, v_share and diff are not for this cache");
    return THA_STATUS_NOT_SUPPORTED;
  }
  if ((long long)rows->n_rows * a->heads > 1ll << 30) return kv8_refuse(who, "too many rows");
  return THA_STATUS_SUCCESS;
}

}  // namespace tha

using namespace tha;

extern "C" size_t tha_hyb_kv8_attn_scratch(int dtype, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv) {
  if (rows->n_rows < 1 || k8_check(a, rows, kv, "tha_hyb_kv8_attn_scratch") != THA_STATUS_SUCCESS) return 0;
  const Kv8Forms f = k8_forms(a, rows, dtype);
  const size_t all = (size_t)rows->n_rows * a->heads;
  const int most = k8_most_tiles(a, rows);
  const size_t stage = f.has_long ? kv8_attn_tc_stage_bytes(a, rows, most, f.short_rows + 1) / sizeof(float) : 0;
  size_t need = 0;
  if (f.has_short || !stage) {
    const int splits = k8_splits(a, rows, stage ? f.short_rows : 0x7FFFFFFF);
    if (splits > 1) need = k8_partial_floats(splits, all, a->vdim);
  }
  if (stage) {
    const int splits = kv8_attn_tc_splits(a, rows, dtype, most);
    const size_t with = stage + (splits > 1 ? k8_partial_floats(splits, all, a->vdim) : 0);
    if (with > need) need = with;
  }
  return need;
}

extern "C" int tha_hyb_kv8_attn(void* stream, int dtype, const tha_attn_t* a, const tha_rows_t* rows, const tha_kv8_t* kv, const float* q, void* out, float* scratch,
                                size_t scratch_floats, const float* proj, long long ldp) {
  if (rows->n_rows < 1) return THA_STATUS_SUCCESS;
  THA_TRY_RC(k8_check(a, rows, kv, "tha_hyb_kv8_attn"));
  if (dtype != THA_DT_BF16 && dtype != THA_DT_F32) return kv8_refuse("tha_hyb_kv8_attn", "unknown dtype");
  if (!q || !out || !aligned16(q)) return kv8_refuse("tha_hyb_kv8_attn", "q on a 16-byte boundary and a result are needed");
  if (scratch && !aligned16(scratch)) return kv8_refuse("tha_hyb_kv8_attn", "scratch on a 16-byte boundary");
  const float* gate = a->head_gate && proj ? proj + a->o_g : nullptr;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == THA_DT_BF16) return k8_attend(s, dtype, a, rows, kv, q, (__nv_bfloat16*)out, scratch, scratch_floats, gate, ldp);
  return k8_attend(s, dtype, a, rows, kv, q, (float*)out, scratch, scratch_floats, gate, ldp);
}
