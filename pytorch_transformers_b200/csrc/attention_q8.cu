// Attention over a paged cache in 8 bits (q8.cuh), straight from the codes.
//
//   score_j = ((q . code_j) * 2^exp_k + bias_j) * scale      exp_k, exp_v: of the page and K/V head that key j lies in
//   out     = sum_j softmax(score)_j * code'_j * 2^exp_v
//
// Two uses: a step of single tokens (FUSED: rotate the token's queries and key, append key and value to the page, attend, in one
// launch; a block's rows are the query heads of one K/V head), and prompts or chunks whose queries are given (rows: tokens x heads).
//
// Numbers. A code becomes a float16 number exactly (cvt.rn.f16x2.e4m3x2) and meets float16 operands in mma.m16n8k16: queries of 11
// bits, their row brought to [1, 2) by a power of two, and softmax weights of 11 bits (of bfloat16's 8 they would cost as much as
// the output's own rounding). Sums, maxima and the output are float32. Keys' exponents go into the factor of a page's scores; values'
// are the unit of the float32 output, which is multiplied by a power of two (exactly) where the unit changes. The unit is
// a warp's, for all of its rows, and stays within 2^60 of the largest exponent that it has met, so that the output cannot overflow in
// small units; products with smaller pages are scaled in float32 before they are added. So a row that does not see (or weigh) the large
// page keeps the small ones' values: those of pages after it to 2^190 below, those of pages before it to 2^140; smaller ones are lost to
// it. The running maximum moves only when a score exceeds it by 2^4 (one vote a tile instead of shuffles for each row).
//
// A weight's range is float16's: the sum of the weights is float32 and loses none, so a weight too small for float16 would be missing
// from the output. The largest is therefore at the top, 2^11 to 2^15, and never below 2^5 in a page of values 2^6 below the unit's: 11
// bits down to 2^-25 of the largest, half a step of 2^-36 below. Beside one key whose score stands out and whose value is zero (an attention
// sink), the output of 8,191 others is as far off as without it (0.0015 of its norm, the output's own rounding) to the 2^-19 of the
// weights that they have at 22 to 24 above them; with the largest weight at 1 they lost 0.4 of it at 18 above and all at 20. It costs 0.4 % at
// the sizes below (a pass of the large batch 181.4 against 180.6 us), and 6 % where a warp has 32 rows, of which one or another moves
// (chunks of 17 tokens: 54.7 against 51.7); with 2^8 before a maximum moves, and four bits less below it, 181.1 and 52.8.
//
// Products. The codes are the larger operand: S^T = K Q^T of 16 keys by 8 rows, O^T = V^T P^T of 16 entries by 8 rows, since few query
// heads read a K/V head (as the smaller one, four heads of 128 on each K/V head wasted three quarters of the products and twice the
// registers). The weights' way from one to the other is a transposition of 8 x 8 (movmatrix). Which key and which entry an index of the
// instruction stands for is free as long as both operands agree: a thread's share of a key's row is 16 codes in a row (a 16-byte load
// gives four k-steps of fragments), and its share of a value's row likewise (the output's rows are named accordingly, pairs of keys are
// put together with byte permutes). The copies' swizzle and an order of keys within eight (kappa) keep both ways of reading free of bank
// conflicts.
//
// Copies. Pages land whole, keys and values, in rings that the tensor memory accelerator fills, two requests a page; a block's warps
// have a part of the keys of a ring's pages each, for one group of rows or another, and take turns to ask for the page that comes into
// the place of one that all have read. No warp waits for another, but through a ring of pages, before the end. Before: cp.async by
// each warp for itself (a tile's copies a quarter of its time), boxes of 16 or 32 rows asked for by the reading warp or by one warp for
// all (the requests alone 175 us where memory allows 150).
//
// What bounds it: 64 sequences of up to 8,192 keys, 32 heads of 128 on 8, 1 GB of codes: 174 us, 5.6 TB/s; without the arithmetic
// the same copies take 150, the rate of a plain copy. The ALU pipe is at 44 % of its peak: 176 of 361 instructions for 16 keys, of which
// unpacking and putting pairs together are 80 by the source's count; the rest are maxima, factors and the loop. Few rows and short
// contexts: the shortest walks measured take 9 us in all, a chain of look-ups (position, page, exponents, codes), queries and the join.
// 71 heads on one K/V head: 64 sequences of 4,096 keys are slower here than over bfloat16 pages on the tcgen05 kernel (a step of six
// layers 1.09 against 0.87 ms).
#include <cooperative_groups.h>

#include <type_traits>

#include "q8.cuh"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace {

// A weight beside a fresh maximum is 2^WEIGHT_TOP, and float16's largest, 2^15, beside one that has not moved yet.
constexpr int MOVE_LOG2 = 4, WEIGHT_TOP = 15 - MOVE_LOG2;
constexpr int UNIT_RANGE = 60, UNIT_SLACK = 6;
constexpr int MAX_CLUSTER = 8;

struct AttnQ8 {
  const __nv_bfloat16* rows;           // FUSED: the projection; else queries [tokens, heads, dim]
  uint8_t *k_pool, *v_pool;
  int8_t *k_exp, *v_exp;
  __nv_bfloat16* out;
  const float *rope_cos, *rope_sin, *slopes;
  const int *tile_seq, *tile_q0;       // not FUSED
  int tile_tokens;
  int heads, kv_heads, dim, pool_pages, rot_pairs, interleaved, write_cache, window;
  int n_splits, cluster, teams;        // blocks that share a row's pages = cluster (one thread-block cluster) * teams
  int row_groups, page_parts, rings, stages;      // warps at work = row_groups * page_parts * rings
  int ring_bytes;                      // of shared memory before the queries
  float scale;
  float* parts;                        // [grid x][grid y][teams][rows][dim + 2] where teams > 1
  int* error_flag;
};

// DP: 64, 128 or 256 entries that a head of `dim` is padded to; NH: eights of rows that a warp holds (a code is unpacked once for all
// of them).
constexpr int WARPS = 8, MAX_STAGES = 8;
template <int DP, int NH> struct Q8Shape {
  static constexpr int TILE = DP == 64 ? 32 : 16;        // keys of a warp's step
  static constexpr int BLOCKS = DP == 256 || NH >= 4 ? 1 : 2;   // on an SM
  static constexpr int STAGE_BYTES = 2 * PTB_PAGE * DP;  // a page of one K/V head: keys, then values
  static constexpr int PITCH = DP + 4;                   // floats of a row of the join
  static constexpr bool ONE = DP == 64 || (DP == 128 && NH <= 2);      // a warp's part of a page is one tile; the launch checks it
};

// The order of a tile's keys: column c of eight stands for key kappa(c). A quarter-warp's 16-byte reads of keys touch columns 2 t and
// 2 t + 1, of values columns 2 t + b for four t: both sets have to lie in different banks under the copies' swizzle.
template <int DP> __device__ __forceinline__ int kappa(int c) {
  const int t = c >> 1;
  if (DP == 64) return (c & 1) ? ((t & 1) + ((t & 2) << 1)) ^ 3 : (t & 1) + ((t & 2) << 1);      // 0 3 1 2 4 7 5 6
  return (c & 1) ? ((2 * t) ^ 4) + 1 : 2 * t;                                                    // 0 5 2 7 4 1 6 3
}
// where the 16-byte chunk `c` of the page's row `key` lies: the 64- and 128-byte swizzles of the copies (boxes of 128 bytes side by side)
template <int DP> __device__ __forceinline__ int place(int key, int c) {
  if (DP == 64) return key * 64 + ((c ^ ((key >> 1) & 3)) << 4);
  return (c >> 3) * (PTB_PAGE * 128) + key * 128 + (((c & 7) ^ (key & 7)) << 4);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// an 8 x 8 matrix of 16-bit numbers, a thread two of row lane / 4, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  uint32_t h;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(h) : "f"(hi), "f"(lo));
  return h;
}
template <int DP, int NH, bool FUSED>
__global__ void __launch_bounds__(WARPS * 32, Q8Shape<DP, NH>::BLOCKS)
attention_q8_kernel(StepBatch sb, AttnQ8 p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using Shape = Q8Shape<DP, NH>;
  constexpr int TILE = Shape::TILE, KS = DP / 16, ST = TILE / 16;      // steps of 16 entries, of 16 keys
  constexpr bool Q_REGS = NH * DP <= 128;      // else the queries' fragments come from shared memory, tile by tile
  extern __shared__ unsigned char smem_dyn[];
  __shared__ __align__(8) uint64_t bars[WARPS][2][MAX_STAGES];      // ring, stage: the page has landed; its warps have read it
  __shared__ __align__(16) unsigned char new_rows[2][DP];      // FUSED: the new token's codes, the page's exponents and whether one rose
  __shared__ int new_exp[2], new_rose[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthreads = blockDim.x;
  const int g4 = lane >> 2, t4 = lane & 3;
  // this warp's eights of rows, its part of every page that lands in its ring, and the ring
  const int rg = warp % p.row_groups, part = warp / p.row_groups % p.page_parts, ring_no = warp / (p.row_groups * p.page_parts);
  const bool idle = ring_no >= p.rings;
  const int key_groups = p.page_parts * p.rings, kg = ring_no * p.page_parts + part;
  const int rows_pad = p.row_groups * 8 * NH;
  // shared memory, by offsets from a base of 1,024 bytes: rings (later the join), queries, their exponents, maxima and sums
  unsigned char* smem = smem_dyn + ((1024 - (smem_u32(smem_dyn) & 1023)) & 1023);
  const int ring = ring_no * p.stages * Shape::STAGE_BYTES;
  const int q_s = p.ring_bytes;      // [8 rows][two steps][lane]: a thread's B fragments, 16 bytes
  int* row_exp = reinterpret_cast<int*>(smem + q_s + rows_pad * DP * 2);
  float* merged_ml = reinterpret_cast<float*>(row_exp + rows_pad);                  // [row][2]
  const int D = p.dim, qpk = p.heads / p.kv_heads;
  const uint32_t bar0 = smem_u32(&bars[ring_no < WARPS ? ring_no : 0][0][0]);      // 8 * MAX_STAGES on: read
  const bool leads = !idle && warp == ring_no * p.row_groups * p.page_parts;      // its first lane asks for the first pages
  pdl_entry();

  // this block's rows: row r of the block is head (row0 + r) % qpk of the group and token (row0 + r) / qpk of the tile
  int seq, q0 = 0, g, row0 = 0, tokens = 1;
  if (FUSED) {
    seq = blockIdx.x;
    g = blockIdx.y;
  } else {
    seq = p.tile_seq[blockIdx.x];
    q0 = p.tile_q0[blockIdx.x];
    g = blockIdx.y % p.kv_heads;
    row0 = int(blockIdx.y / p.kv_heads) * rows_pad;
    tokens = min(p.tile_tokens, sb.seq_new[seq] - q0);
  }
  const int n_rows = min(rows_pad, tokens * qpk - row0);
  if (n_rows <= 0) return;      // all blocks of a cluster alike
  const int past = sb.seq_past[seq], start = sb.seq_start[seq];
  if (FUSED && sb.seq_new[seq] != 1) {      // as many tokens as sequences, but not one each: `start` may lie past the last row
    if (tid == 0) atomicExch(p.error_flag, 54);
    return;
  }
  const int first_pos = FUSED ? past : past + q0 + row0 / qpk, last_pos = FUSED ? past : past + q0 + (row0 + n_rows - 1) / qpk;
  const int low = p.window > 0 ? max(0, first_pos - p.window + 1) : 0;      // the first key that a row sees
  const int* pages = sb.pages + size_t(seq) * sb.pages_stride;
  const int split = blockIdx.z;
  // pages of this block (whole ones: the page that a step appends to has one reader), and of them this warp's tiles
  const int pg0 = low / PTB_PAGE, n_pages = last_pos / PTB_PAGE + 1 - pg0;
  auto up_to = [&](int i) {
    return n_pages < (1 << 21) ? i * n_pages / p.n_splits : int((long long)i * n_pages / p.n_splits);      // n_splits <= 512
  };
  const int pg_begin = pg0 + (p.n_splits == 1 ? 0 : up_to(split)), pg_end = pg0 + (p.n_splits == 1 ? n_pages : up_to(split + 1));
  const bool appends = FUSED && p.write_cache && pg_end == pg0 + n_pages && pg_begin < pg_end;
  const int fused_width = p.kv_heads * (qpk + 2) * D;

  const int n_mine = !idle && pg_begin + ring_no < pg_end && rg * 8 * NH < n_rows ? (pg_end - pg_begin - ring_no + p.rings - 1) / p.rings : 0;
  const int sharers = p.page_parts * min(p.row_groups, (n_rows + 8 * NH - 1) / (8 * NH));      // warps that read a page of the ring
  // what a lane knows of page `lane` of a stretch of 32 of the ring's: its number and its exponents
  auto look_up = [&](int stretch, int& page, int& exps) {
    const int i = stretch * 32 + lane;
    page = 0;
    exps = 0;
    if (i < n_mine) {
      const int at = pg_begin + ring_no + i * p.rings;
      page = at < sb.pages_stride ? pages[at] : -1;
      if (page < 0 || page >= p.pool_pages) {
        atomicExch(p.error_flag, 51);
        page = 0;
      }
      const size_t block = size_t(page) * p.kv_heads + g;
      exps = int(__ldcg(reinterpret_cast<const signed char*>(p.k_exp) + block)) * 256 +
             (int(__ldcg(reinterpret_cast<const signed char*>(p.v_exp) + block)) & 255);
    }
  };
  int page_now, exps_now, page_next = 0, exps_next = 0;
  look_up(0, page_now, exps_now);
  auto ask = [&](int page, int st) {      // by one thread
    const uint32_t bar = bar0 + 8 * st, to = smem_u32(smem) + ring + st * Shape::STAGE_BYTES;
    const int y = (page * p.kv_heads + g) * PTB_PAGE;
    mbar_expect_tx(bar, Shape::STAGE_BYTES);
#pragma unroll
    for (int x = 0; x < DP; x += 128) tma_load_2d(to + x * PTB_PAGE, &k_map, x, y, bar);
#pragma unroll
    for (int x = 0; x < DP; x += 128) tma_load_2d(to + PTB_PAGE * DP + x * PTB_PAGE, &v_map, x, y, bar);
  };
  auto ask_first = [&]() {
    if (lane < p.stages && lane < n_mine) ask(page_now, lane);      // a lane a stage
  };
  if (leads) {      // on their way while the queries are made
    if (lane < p.stages) {
      mbar_init(bar0 + 8 * lane, 1);
      mbar_init(bar0 + 8 * (MAX_STAGES + lane), sharers);
      asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncwarp();
    ask_first();
  }
  if (appends) {
    const int page = pg_end <= sb.pages_stride ? pages[pg_end - 1] : -1;
    const __nv_bfloat16* frow = p.rows + size_t(start) * fused_width + size_t(g) * (qpk + 2) * D;
    if (warp == 5 || warp == 7) {      // never the ones that ask for the first pages
      const int which = warp == 7;
      bool rose = false;
      int e = 0;
      if (page >= 0 && page < p.pool_pages) {
        const size_t block = size_t(page) * p.kv_heads + g;
        e = append_row(frow + size_t(qpk + which) * D, p.rope_cos + size_t(start) * p.rot_pairs, p.rope_sin + size_t(start) * p.rot_pairs,
                       which == 0 ? p.rot_pairs : 0, p.interleaved, (which == 0 ? p.k_pool : p.v_pool) + block * PTB_PAGE * D,
                       (which == 0 ? p.k_exp : p.v_exp) + block, past % PTB_PAGE, D, new_rows[which], rose);
      }
      if (lane == 0) {
        new_exp[which] = e;
        new_rose[which] = rose;
      }
    }
  }

  // queries: rotated (FUSED), brought to [1, 2) by a power of two, float16. A group of lanes holds a row, eight entries each; the
  // loads of four rows are out before the first is used.
  {
    constexpr int GL = DP / 8, PER = 32 / GL, AHEAD = 4;
    const int c = lane % GL, step = WARPS * PER;
    Angles angles;
    angles.mode = 0;
    angles.other = c;
    const float *rc = p.rope_cos + size_t(start) * p.rot_pairs, *rs = p.rope_sin + size_t(start) * p.rot_pairs;
    if (FUSED && c * 8 < D) angles = angles_of(c, rc, rs, p.rot_pairs, p.interleaved);
    auto row_at = [&](int r) {
      if (FUSED) return p.rows + size_t(start) * fused_width + (size_t(g) * (qpk + 2) + r) * D;
      const size_t t = start + q0 + (row0 + r) / qpk;
      return p.rows + (t * p.heads + g * qpk + (row0 + r) % qpk) * D;
    };
    for (int r0 = warp * PER + lane / GL; r0 < rows_pad; r0 += step * AHEAD) {
      uint4 own[AHEAD], other[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int r = r0 + k * step;
        own[k] = other[k] = make_uint4(0, 0, 0, 0);
        if (r < n_rows && c * 8 < D) {
          const uint4* row = reinterpret_cast<const uint4*>(row_at(r));
          own[k] = row[c];
          if (FUSED && angles.mode == 2) other[k] = row[angles.other];
        }
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int r = r0 + k * step;
        if (r >= rows_pad) break;      // rows_pad and r0 - lane / GL are multiples of PER: a warp leaves as one
        float x[8];
        if (FUSED && angles.mode == 3 && r < n_rows) load_rotated8(row_at(r), c, rc, rs, p.rot_pairs, 0, x);
        else rotate8(angles, own[k], other[k], x);
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, finite_abs(x[e]));
#pragma unroll
        for (int o = GL / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const int e = min(max((__float_as_int(most) >> 23) - 127, -100), 126);      // most = 2^e * [1, 2)
        const float by = power_of_two(-e);
        uint4 w;
        w.x = pack_half(x[0] * by, x[1] * by);
        w.y = pack_half(x[2] * by, x[3] * by);
        w.z = pack_half(x[4] * by, x[5] * by);
        w.w = pack_half(x[6] * by, x[7] * by);
        // entries 8 c and on: two steps of the thread that holds this row and these 16 entries
        *reinterpret_cast<uint4*>(smem + q_s + (((r >> 3) * (KS / 2) + (c >> 3) * 2 + (c & 1)) * 32 + (r & 7) * 4 + ((c >> 1) & 3)) * 16) = w;
        if (c == 0) row_exp[r] = e;
      }
    }
  }
  __syncthreads();
  // Waits are bounded: one that runs out raises the error flag, and the block goes on to its end.
  bool alive = true;
  int turn = 0;      // of the barriers: whether the first pages came twice
  auto landed = [&](int st, int parity) {
    const uint32_t bar = bar0 + 8 * st;
    if (!__all_sync(0xffffffffu, mbar_test(bar, parity))) alive = __all_sync(0xffffffffu, mbar_wait(bar, parity, p.error_flag, 52));
  };
  if (appends) {
    if (new_rose[0] || new_rose[1]) {      // the page's earlier codes have changed: the first pages once more
      for (int st = 0; st < p.stages && st < n_mine && alive; ++st) landed(st, 0);
      __syncthreads();
      if (leads && alive) ask_first();
      turn = 1;
    }
    if (lane < n_mine && pg_begin + ring_no + lane * p.rings == pg_end - 1) exps_now = new_exp[0] * 256 + (new_exp[1] & 255);
  }

  const float sl2 = p.scale * 1.4426950408889634f;
  float row_fac[NH][2];      // a thread's rows: 8 n + 2 t4 and the next, of its warp's
#pragma unroll
  for (int n = 0; n < NH; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      row_fac[n][i] = power_of_two(row_exp[(rg * NH + n) * 8 + 2 * t4 + i]);
      if (!p.slopes) row_fac[n][i] *= sl2;
    }
  const int q_at = q_s + rg * NH * (KS / 2) * 512 + lane * 16;
  auto q_frag = [&](int n, int step) { return *reinterpret_cast<const uint4*>(smem + q_at + (n * (KS / 2) + step / 2) * 512); };      // of steps `step`, step + 1
  uint4 qb[Q_REGS ? NH : 1][Q_REGS ? KS / 2 : 1];
  if (Q_REGS) {
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int s = 0; s < KS / 2; ++s) qb[Q_REGS ? n : 0][Q_REGS ? s : 0] = q_frag(n, 2 * s);
  }

  float o[NH][KS][4];
#pragma unroll
  for (int n = 0; n < NH; ++n)
#pragma unroll
    for (int j = 0; j < KS; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
  float m_run[NH][2], l_run[NH][2];
#pragma unroll
  for (int n = 0; n < NH; ++n) m_run[n][0] = m_run[n][1] = -INFINITY, l_run[n][0] = l_run[n][1] = 0.f;
  int unit = Q8_EXP_MIN, largest = Q8_EXP_MIN;      // of the output; of the values' exponents so far
  constexpr int VW = DP == 64 ? 2 : 4, VR = (DP + 127) / 128;      // words of a key's row a thread takes at a time, and times
  // where in a stage a thread reads: its key of eight (the other eights 8 rows on, under the same swizzle), its keys of a value pair
  int k_at[DP / 64], v_at[2];
#pragma unroll
  for (int r = 0; r < DP / 64; ++r) k_at[r] = ring + place<DP>(kappa<DP>(g4), t4 + 4 * r);
#pragma unroll
  for (int u = 0; u < 2; ++u)
    v_at[u] = ring + PTB_PAGE * DP + (DP == 64 ? place<DP>(kappa<DP>(2 * t4 + u), g4 >> 1) + (g4 & 1) * 8 : place<DP>(kappa<DP>(2 * t4 + u), g4));
  constexpr int EIGHT = 8 * (DP == 64 ? 64 : 128);      // bytes from a row to that of eight keys on
  constexpr bool ONE = Shape::ONE;
  const int part_keys = ONE ? TILE : PTB_PAGE / p.page_parts;
  int st = 0, reads_turn = 0;

  int i = 0;
  for (; i < n_mine && alive; ++i) {
    if ((i & 31) == 0 && i > 0) {
      page_now = page_next;
      exps_now = exps_next;
    }
    if ((i & 31) == 8 && (i & ~31) + 32 < n_mine) look_up((i >> 5) + 1, page_next, exps_next);
    const int both = __shfl_sync(0xffffffffu, exps_now, i & 31);
    const int page_key0 = (pg_begin + ring_no + i * p.rings) * PTB_PAGE;
    landed(st, turn & 1);
    if (!alive) break;
    // page `stages` on from the one before, into its place: its warps take turns to ask, a page late, when all have read it
    if (i > 0 && i - 1 + p.stages < n_mine && rg == 0 && ((i - 1) & (p.page_parts - 1)) == part) {      // page_parts is a power of two
      const int j = i - 1 + p.stages, before = st == 0 ? p.stages - 1 : st - 1;
      const int page = __shfl_sync(0xffffffffu, (j ^ i) < 32 ? page_now : page_next, j & 31);
      const uint32_t bar = bar0 + 8 * (MAX_STAGES + before), parity = (st == 0 ? reads_turn - 1 : reads_turn) & 1;
      if (!__all_sync(0xffffffffu, mbar_test(bar, parity))) alive = __all_sync(0xffffffffu, mbar_wait(bar, parity, p.error_flag, 53));
      if (!alive) break;
      if (lane == 0) ask(page, before);
    }
    const int first_key = page_key0 + part * part_keys;
    if (FUSED && appends && past - first_key >= 0 && past - first_key < part_keys) {
      // the new token's codes from this block rather than from the page, where they may have come after the copy; all who read them
      // write the same
      if (lane < 2 * D / 16) {
        const int which = lane >= D / 16, c = which ? lane - D / 16 : lane;
        *reinterpret_cast<uint4*>(smem + ring + st * Shape::STAGE_BYTES + which * PTB_PAGE * DP + place<DP>(past - page_key0, c)) =
            *reinterpret_cast<const uint4*>(new_rows[which] + c * 16);
        proxy_fence_async();      // before the accelerator may write there again
      }
      __syncwarp();
    }
    const int ev = int(int8_t(both & 255)), ek = both >> 8;
    for (int sub = 0; sub < (ONE ? TILE : part_keys); sub += TILE) {
      const int key0 = first_key + sub;
      if (key0 > last_pos || key0 + TILE <= low) continue;
      const int kt = st * Shape::STAGE_BYTES + (key0 - page_key0) * (DP == 64 ? 64 : 128);

      // scores
      float s[NH][ST][4];      // of row 2 t4, 2 t4 + 1 with key kappa(g4), then with key 8 + kappa(g4)
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int j = 0; j < ST; ++j) s[n][j][0] = s[n][j][1] = s[n][j][2] = s[n][j][3] = 0.f;
#pragma unroll
      for (int r = 0; r < DP / 64; ++r) {
        uint4 w[2 * ST];
#pragma unroll
        for (int j = 0; j < 2 * ST; ++j) w[j] = *reinterpret_cast<const uint4*>(smem + k_at[r] + kt + j * EIGHT);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
          for (int j = 0; j < ST; ++j) {
            uint32_t a[4];
            q8_halves(word_of(w[2 * j], kk), a[0], a[2]);
            q8_halves(word_of(w[2 * j + 1], kk), a[1], a[3]);
#pragma unroll
            for (int n = 0; n < NH; ++n) {
              const uint4 q = Q_REGS ? qb[Q_REGS ? n : 0][Q_REGS ? r * 2 + kk / 2 : 0] : q_frag(n, r * 4 + kk);
              mma_f16(s[n][j], a, (kk & 1) ? q.z : q.x, (kk & 1) ? q.w : q.y);
            }
          }
        }
      }
      // The unit of the output: that of the tile's values, but where these are smaller by up to 2^6, which the weights carry instead (a
      // weight of fewer bits then belongs to a smaller value), and for pages 2^60 below the largest.
      bool new_unit = false;
      int far = 0, shift = 0, old_unit = unit;
      if (ev != unit) {
        largest = max(largest, ev);
        const int floor_unit = largest - UNIT_RANGE;
        new_unit = (ev > unit || ev < unit - UNIT_SLACK) && !(ev < floor_unit && unit == floor_unit);
        if (new_unit) unit = max(ev > unit ? ev : ev + UNIT_SLACK / 2, floor_unit);
        far = ev - unit;      // 0 to -185
        shift = far < -UNIT_SLACK ? 0 : far;      // 2^shift comes with the exponential
      }
      // score - running maximum + WEIGHT_TOP + shift, in powers of two; a tile that all rows see whole needs no mask
      const float fk = power_of_two(ek), fshift = float(WEIGHT_TOP + shift);
      const bool whole = key0 + TILE - 1 <= first_pos && (p.window == 0 || key0 > last_pos - p.window);
      float over = -INFINITY;      // by how much the tile exceeds the running maxima
      if (whole && !p.slopes) {
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const bool fresh = m_run[n][h] == -INFINITY;
            const float f = row_fac[n][h] * fk, m = fresh ? fshift : fshift - m_run[n][h];
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < ST; ++j) {
              s[n][j][h] = fmaf(s[n][j][h], f, m);
              s[n][j][2 + h] = fmaf(s[n][j][2 + h], f, m);
              top = fmaxf(top, fmaxf(s[n][j][h], s[n][j][2 + h]));
            }
            over = fmaxf(over, fresh ? INFINITY : top);
          }
      } else {
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = (rg * NH + n) * 8 + 2 * t4 + h;
            const bool ok = r < n_rows;
            const int pos = !ok ? -1 : FUSED ? past : past + q0 + (row0 + r) / qpk;
            const float slope = ok && p.slopes ? p.slopes[g * qpk + (FUSED ? r : (row0 + r) % qpk)] : 0.f;
            const bool fresh = m_run[n][h] == -INFINITY;
            const float f = row_fac[n][h] * fk, m = fresh ? fshift : fshift - m_run[n][h];
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 2 * ST; ++j) {
              const int key = key0 + j * 8 + kappa<DP>(g4);
              float v = s[n][j >> 1][(j & 1) * 2 + h] * f;
              if (p.slopes) v = (v + alibi_bias(slope, key)) * sl2;
              v += m;
              if (!whole && (key > pos || (p.window > 0 && key <= pos - p.window))) v = -INFINITY;
              s[n][j >> 1][(j & 1) * 2 + h] = v;
              top = fmaxf(top, v);
            }
            over = fmaxf(over, fresh && top != -INFINITY ? INFINITY : top);
          }
      }
      if (__any_sync(0xffffffffu, over > float(MOVE_LOG2) + fshift) || new_unit) {
        // a unit may rise by 2^245: more than one power of two holds
        const float change = power_of_two(max((old_unit - unit) / 2, -126)), change2 = power_of_two(max(old_unit - unit - (old_unit - unit) / 2, -126));
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float up = -INFINITY;
#pragma unroll
            for (int j = 0; j < ST; ++j) up = fmaxf(up, fmaxf(s[n][j][h], s[n][j][2 + h]));
#pragma unroll
            for (int lanes = 4; lanes < 32; lanes *= 2) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, lanes));
            up -= fshift;
            const bool fresh = m_run[n][h] == -INFINITY;      // then `up` is the maximum itself
            if (!fresh) up = fmaxf(up, 0.f);
            const float corr = fresh ? 0.f : exp2f(-up), by = up == -INFINITY ? 0.f : up;
            m_run[n][h] = fresh ? up : m_run[n][h] + up;
            l_run[n][h] *= corr;
#pragma unroll
            for (int j = 0; j < ST; ++j) {
              s[n][j][h] -= by;
              s[n][j][2 + h] -= by;
            }
            const float f = corr * change;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
              o[n][j][h] = o[n][j][h] * f * change2;
              o[n][j][2 + h] = o[n][j][2 + h] * f * change2;
            }
          }
      }
      uint32_t pb[NH][ST][2];
      const float back = power_of_two(-shift);      // the sums are of the weights without it
#pragma unroll
      for (int n = 0; n < NH; ++n) {
#pragma unroll
        for (int j = 0; j < ST; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][j][e] = fast_exp2(s[n][j][e]);
          l_run[n][0] = fmaf(s[n][j][0] + s[n][j][2], back, l_run[n][0]);
          l_run[n][1] = fmaf(s[n][j][1] + s[n][j][3], back, l_run[n][1]);
        }
#pragma unroll
        for (int j = 0; j < ST; ++j) {
          pb[n][j][0] = transposed(pack_half(s[n][j][0], s[n][j][1]));
          pb[n][j][1] = transposed(pack_half(s[n][j][2], s[n][j][3]));
        }
      }
      // output. Keys that no row of the block sees are taken as zero: their codes may be anything.
      const bool edge = key0 + TILE - 1 > last_pos || key0 < low;
      // apart: a page 2^60 below the largest, whose products are scaled in float32 before they are added. Large batch 185.0 us a pass with this
      // second copy of the products, 181.0 without; one copy, the sums waiting in local memory: 189.4
      auto add_values = [&](auto apart) {
#pragma unroll
        for (int ks = 0; ks < ST; ++ks)
#pragma unroll
          for (int rr = 0; rr < VR; ++rr) {
            uint32_t v[4][VW];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int at = v_at[u & 1] + kt + rr * (PTB_PAGE * 128) + (2 * ks + (u >> 1)) * EIGHT;
              if (DP == 64) {
                const uint2 x = *reinterpret_cast<const uint2*>(smem + at);
                v[u][0] = x.x; v[u][1] = x.y;
              } else {
                const uint4 x = *reinterpret_cast<const uint4*>(smem + at);
                v[u][0] = x.x; v[u][1] = x.y; v[u][VW - 2] = x.z; v[u][VW - 1] = x.w;
              }
            }
            if (edge) {
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int key = key0 + (2 * ks + (u >> 1)) * 8 + kappa<DP>(2 * t4 + (u & 1));
#pragma unroll
                for (int q = 0; q < VW; ++q) v[u][q] = key > last_pos || key < low ? 0u : v[u][q];
              }
            }
#pragma unroll
            for (int q = 0; q < VW; ++q) {
              uint32_t a[4], b[4];      // entries 4 q, 4 q + 1 and 4 q + 2, 4 q + 3 of the thread's
              q8_halves(__byte_perm(v[0][q], v[1][q], 0x5140), a[0], a[1]);
              q8_halves(__byte_perm(v[2][q], v[3][q], 0x5140), a[2], a[3]);
              q8_halves(__byte_perm(v[0][q], v[1][q], 0x7362), b[0], b[1]);
              q8_halves(__byte_perm(v[2][q], v[3][q], 0x7362), b[2], b[3]);
#pragma unroll
              for (int n = 0; n < NH; ++n) {
                if constexpr (decltype(apart)::value) {
                  float x[4] = {}, y[4] = {};
                  mma_f16(x, a, pb[n][ks][0], pb[n][ks][1]);
                  mma_f16(y, b, pb[n][ks][0], pb[n][ks][1]);
                  const float f = power_of_two(max(far, -126)), f2 = power_of_two(min(far + 126, 0));
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    o[n][rr * 8 + q * 2][e] += x[e] * f2 * f;
                    o[n][rr * 8 + q * 2 + 1][e] += y[e] * f2 * f;
                  }
                } else {
                  mma_f16(o[n][rr * 8 + q * 2], a, pb[n][ks][0], pb[n][ks][1]);
                  mma_f16(o[n][rr * 8 + q * 2 + 1], b, pb[n][ks][0], pb[n][ks][1]);
                }
              }
            }
          }
      };
      if (far == shift) add_values(std::false_type{});
      else add_values(std::true_type{});
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(bar0 + 8 * (MAX_STAGES + st));
    if (++st == p.stages) st = 0, ++turn, ++reads_turn;
  }
  if (!alive)      // a wait ran out: what is in flight lands before the block ends (bounded waits again)
    for (int k = 0; k < p.stages && i + k < n_mine; ++k) {
      landed(st, turn & 1);
      if (++st == p.stages) st = 0, ++turn;
    }

  // Parts of a row into one, always in the same order: of the key groups here, of a cluster's blocks through their shared memory,
  // of the teams of clusters by join_q8_kernel. Every part is a mean under its own weights times its share of the sum: the shares come
  // before the sums of values, which may be as large as float32 holds.
  float* join = reinterpret_cast<float*>(smem);                 // [key group][row][PITCH], in the rings' place
  float* join_ml = merged_ml + 2 * rows_pad;                    // [key group][row][2]
#pragma unroll
  for (int n = 0; n < NH; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float l = l_run[n][h];
#pragma unroll
      for (int lanes = 4; lanes < 32; lanes *= 2) l += __shfl_xor_sync(0xffffffffu, l, lanes);
      l_run[n][h] = l;
      const int r = kg * rows_pad + (rg * NH + n) * 8 + 2 * t4 + h;
      if (g4 == 0 && !idle) *reinterpret_cast<float2*>(join_ml + 2 * r) = make_float2(m_run[n][h], l);
    }
  __syncthreads();      // and the rings are done with
  for (int r = tid; r < n_rows; r += WARPS * 32) {
    float m = -INFINITY, l = 0.f;
    for (int k = 0; k < key_groups; ++k) m = fmaxf(m, join_ml[2 * (k * rows_pad + r)]);
    for (int k = 0; k < key_groups; ++k) {
      const float2 ml = *reinterpret_cast<const float2*>(join_ml + 2 * (k * rows_pad + r));
      l += ml.x == -INFINITY && ml.y == 0.f ? 0.f : ml.y * exp2f(ml.x - m);
    }
    *reinterpret_cast<float2*>(merged_ml + 2 * r) = make_float2(m, l);
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NH; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = (rg * NH + n) * 8 + 2 * t4 + h;
      if (r >= n_rows || idle) continue;
      const float2 ml = *reinterpret_cast<const float2*>(merged_ml + 2 * r);
      const bool none = m_run[n][h] == -INFINITY && l_run[n][h] == 0.f;
      const float share = none ? 0.f : exp2f(m_run[n][h] - ml.x) / ml.y, in_unit = power_of_two(unit);      // one after the other: their product may be too small a number
      constexpr int COLS = DP == 64 ? 8 : 16;      // entries of a row of the output that a thread holds: [g4][COLS]
      float* to = join + size_t(kg * rows_pad + r) * Shape::PITCH + g4 * COLS;
#pragma unroll
      for (int rr = 0; rr < VR; ++rr)
#pragma unroll
        for (int c = 0; c < COLS / 2; c += 2) {
          const float(&x)[4] = o[n][rr * 8 + c], (&y)[4] = o[n][rr * 8 + c + 1];
          *reinterpret_cast<float4*>(to + rr * 128 + 2 * c) =
              none ? make_float4(0.f, 0.f, 0.f, 0.f)
                   : make_float4(x[h] * share * in_unit, x[2 + h] * share * in_unit, y[h] * share * in_unit, y[2 + h] * share * in_unit);
        }
    }
  __syncthreads();
  const int quads = D / 4;
  auto write = [&](int r, int d, const float4& acc, float m, float l) {
    if (p.teams > 1) {
      float* to = p.parts + (((size_t(blockIdx.x) * gridDim.y + blockIdx.y) * p.teams + split / p.cluster) * rows_pad + r) * size_t(D + 2);
      *reinterpret_cast<float2*>(to + d) = make_float2(acc.x, acc.y);
      *reinterpret_cast<float2*>(to + d + 2) = make_float2(acc.z, acc.w);
      if (d == 0) *reinterpret_cast<float2*>(to + D) = make_float2(m, l);
    } else {
      const size_t t = start + q0 + (FUSED ? 0 : (row0 + r) / qpk);
      *reinterpret_cast<uint2*>(p.out + (t * p.heads + g * qpk + (FUSED ? r : (row0 + r) % qpk)) * D + d) =
          make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
    }
  };
  for (int i = tid; i < n_rows * quads; i += nthreads) {
    const int r = i / quads, d = (i - r * quads) * 4;
    float4 acc = *reinterpret_cast<const float4*>(join + size_t(r) * Shape::PITCH + d);
    for (int k = 1; k < key_groups; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(join + size_t(k * rows_pad + r) * Shape::PITCH + d);
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    }
    if (p.cluster > 1) *reinterpret_cast<float4*>(join + size_t(r) * Shape::PITCH + d) = acc;      // this thread alone reads and writes here
    else write(r, d, acc, merged_ml[2 * r], merged_ml[2 * r + 1]);
  }
  if (p.cluster == 1) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int n = p.cluster;
  for (int i = tid * n + split % n; i < n_rows * quads; i += nthreads * n) {
    const int r = i / quads, d = (i - r * quads) * 4;
    float ms[MAX_CLUSTER], w[MAX_CLUSTER];
    float4 v[MAX_CLUSTER];
#pragma unroll
    for (int k = 0; k < MAX_CLUSTER; ++k) {      // all on their way before the first is used
      const int rank = k < n ? k : 0;
      const float2 ml = *reinterpret_cast<const float2*>(cluster.map_shared_rank(merged_ml, rank) + 2 * r);
      v[k] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(join, rank) + size_t(r) * Shape::PITCH + d);
      ms[k] = k < n ? ml.x : -INFINITY;
      w[k] = k < n ? ml.y : 0.f;
    }
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < MAX_CLUSTER; ++k) m = fmaxf(m, ms[k]);
#pragma unroll
    for (int k = 0; k < MAX_CLUSTER; ++k) {
      w[k] = ms[k] == -INFINITY && w[k] == 0.f ? 0.f : w[k] * exp2f(ms[k] - m);
      l += w[k];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int k = 0; k < MAX_CLUSTER; ++k) {
      const float u = w[k] * inv;
      if (u != 0.f) { acc.x += v[k].x * u; acc.y += v[k].y * u; acc.z += v[k].z * u; acc.w += v[k].w * u; }
    }
    write(r, d, acc, m, l);
  }
  cluster.sync();      // no block leaves while another may still read its shared memory
}

// The teams' parts of a row into its output, always in their order.
template <bool FUSED>
__global__ void __launch_bounds__(256) join_q8_kernel(StepBatch sb, AttnQ8 p, int rows_pad, int grid_y) {
  pdl_entry();
  const int x = blockIdx.x, y = blockIdx.y, D = p.dim, qpk = p.heads / p.kv_heads;
  const int g = FUSED ? y : y % p.kv_heads, row0 = FUSED ? 0 : y / p.kv_heads * rows_pad;
  const int seq = FUSED ? x : p.tile_seq[x], q0 = FUSED ? 0 : p.tile_q0[x];
  if (FUSED && sb.seq_new[seq] != 1) return;      // the attention kernel has said so and left no parts; the row may lie past the last
  const int tokens = FUSED ? 1 : min(p.tile_tokens, sb.seq_new[seq] - q0);
  const int n_rows = min(rows_pad, tokens * qpk - row0), quads = D / 4;
  const float* parts = p.parts + (size_t(x) * grid_y + y) * p.teams * size_t(rows_pad) * (D + 2);
  const size_t pitch = size_t(rows_pad) * (D + 2);
  for (int i = blockIdx.z * blockDim.x + threadIdx.x; i < n_rows * quads; i += gridDim.z * blockDim.x) {
    const int r = i / quads, d = (i - r * quads) * 4;
    const float* at = parts + size_t(r) * (D + 2);
    float m = -INFINITY;
    for (int s = 0; s < p.teams; ++s) m = fmaxf(m, at[s * pitch + D]);
    float l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    auto weight = [&](int s) {
      const float2 ml = *reinterpret_cast<const float2*>(at + s * pitch + D);
      return ml.x == -INFINITY && ml.y == 0.f ? 0.f : ml.y * exp2f(ml.x - m);
    };
    for (int s = 0; s < p.teams; ++s) l += weight(s);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int s = 0; s < p.teams; ++s) {
      const float w = weight(s) * inv;
      const float2 a = *reinterpret_cast<const float2*>(at + s * pitch + d), b = *reinterpret_cast<const float2*>(at + s * pitch + d + 2);
      if (w != 0.f) { acc[0] += a.x * w; acc[1] += a.y * w; acc[2] += b.x * w; acc[3] += b.y * w; }
    }
    const size_t t = size_t(sb.seq_start[seq]) + q0 + (row0 + r) / qpk;
    *reinterpret_cast<uint2*>(p.out + (t * p.heads + g * qpk + (row0 + r) % qpk) * D + d) =
        make_uint2(pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3]));
  }
}

struct Plan {
  int dp, nh, row_groups, page_parts, rings, stages, rows_pad;
};
// rows: of a block's tile at most (more are divided among blocks)
Plan plan_of(int dim, int rows) {
  Plan q;
  q.dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  // heads of 64: fives of eights where they waste less, as for 71 rows: two warps of 40 in place of three of 32, which left two idle
  const bool fives = q.dp == 64 && ((rows > 32 && rows <= 40) || (rows > 64 && rows <= 80));
  q.nh = rows <= 8 ? 1 : rows <= 16 || q.dp == 256 ? 2 : fives ? 5 : 4;
  const int groups = (rows + 8 * q.nh - 1) / (8 * q.nh), most = q.dp == 256 ? 8 : 4;
  q.row_groups = groups < most ? groups : most;
  q.rows_pad = q.row_groups * 8 * q.nh;
  const int keys = WARPS / q.row_groups, parts = q.dp == 64 ? 2 : 4;      // a part is a tile at least
  q.page_parts = keys >= parts ? parts : keys >= 2 ? 2 : 1;
  q.rings = keys / q.page_parts;
  // about 96 KB of rings where two blocks are to fit on an SM, else 128
  const int pages = (q.nh >= 4 || q.dp == 256 ? 131072 : 98304) / (2 * PTB_PAGE * q.dp);
  q.stages = pages / q.rings < MAX_STAGES ? pages / q.rings : MAX_STAGES;
  return q;
}

// The codes of a pool as rows of `dim` bytes: boxes of a page's rows, 64 bytes or 128 wide (zeros past dim), under the swizzle of that width.
bool codes_map(CUtensorMap* map, const void* pool, int pool_pages, int kv_heads, int dim, int dp) {
  static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> known{nullptr};
  PFN_cuTensorMapEncodeTiled_v12000 encode = known.load(std::memory_order_acquire);
  if (encode == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qr) != cudaSuccess || qr != cudaDriverEntryPointSuccess)
      return false;
    encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    known.store(encode, std::memory_order_release);
  }
  const cuuint64_t dims[2] = {cuuint64_t(dim), cuuint64_t(pool_pages) * kv_heads * PTB_PAGE};
  const cuuint64_t strides[1] = {cuuint64_t(dim)};
  const cuuint32_t box[2] = {dp == 64 ? 64u : 128u, cuuint32_t(PTB_PAGE)};
  const cuuint32_t elem[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pool), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                dp == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int NH, bool FUSED>
int launch_attn(const StepBatch& sb, AttnQ8 p, const Plan& q, dim3 grid, cudaStream_t stream) {
  using Shape = Q8Shape<DP, NH>;
  const int key_groups = q.page_parts * q.rings;
  if (Shape::ONE && PTB_PAGE / q.page_parts != Shape::TILE) return PTB_ERR_SIZE;      // keys would be left out
  const size_t ring = size_t(q.rings) * q.stages * Shape::STAGE_BYTES;
  const size_t join = size_t(key_groups) * q.rows_pad * Shape::PITCH * sizeof(float);
  p.ring_bytes = int(ring > join ? ring : (join + 15) / 16 * 16);
  const size_t smem = 1024 + p.ring_bytes + size_t(q.rows_pad) * (DP * 2 + sizeof(int) + 2 * sizeof(float) * (1 + key_groups));
  static SharedLimit limit;
  if (!limit.allows(attention_q8_kernel<DP, NH, FUSED>, smem)) return PTB_ERR_LAUNCH;
  CUtensorMap k_map, v_map;
  if (!codes_map(&k_map, p.k_pool, p.pool_pages, p.kv_heads, p.dim, DP) ||
      !codes_map(&v_map, p.v_pool, p.pool_pages, p.kv_heads, p.dim, DP))
    return PTB_ERR_LAUNCH;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  bool captured = true;      // launch_pdl's rule
  if (cudaStreamIsCapturing(stream, &capture) == cudaSuccess) captured = capture != cudaStreamCaptureStatusNone;
  else (void)cudaGetLastError();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = captured ? 0 : 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = unsigned(p.cluster);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = captured ? attr + 1 : attr;
  cfg.numAttrs = (captured ? 0 : 1) + (p.cluster > 1 ? 1 : 0);
  cudaLaunchKernelEx(&cfg, attention_q8_kernel<DP, NH, FUSED>, sb, p, k_map, v_map);
  int status = launch_status();
  if (status == PTB_OK && p.teams > 1) {
    const int z = max(1, min(8, q.rows_pad * (p.dim / 4) / 512));
    launch_pdl(join_q8_kernel<FUSED>, dim3(grid.x, grid.y, z), dim3(256), 0, stream, sb, p, q.rows_pad, int(grid.y));
    status = launch_status();
  }
  return status;
}
template <bool FUSED>
int launch_any(const StepBatch& sb, const AttnQ8& p, const Plan& q, dim3 grid, cudaStream_t stream) {
#define PTB_Q8(DD, NN) return launch_attn<DD, NN, FUSED>(sb, p, q, grid, stream)
  if (q.dp == 64) {
    if (q.nh == 1) PTB_Q8(64, 1);
    if (q.nh == 2) PTB_Q8(64, 2);
    if (q.nh == 5) PTB_Q8(64, 5);
    PTB_Q8(64, 4);
  }
  if (q.dp == 128) {
    if (q.nh == 1) PTB_Q8(128, 1);
    if (q.nh == 2) PTB_Q8(128, 2);
    PTB_Q8(128, 4);
  }
  if (q.nh == 1) PTB_Q8(256, 1);
  PTB_Q8(256, 2);
#undef PTB_Q8
}
bool known(int heads, int kv_heads, int dim, int pool_pages) {
  return heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && kv_heads <= 65535 && dim >= 16 && dim <= 256 && dim % 16 == 0 && pool_pages > 0 &&
         (long long)pool_pages * kv_heads * PTB_PAGE < (1ll << 31);      // rows of codes, as the copies count them
}
// Blocks that share a row's pages: as many as the SMs take at a time, two pages each at least. Up to eight form a cluster and join
// through its shared memory; more are a multiple of eight, of eight pages each at least, whose clusters join through a workspace.
// `beside` a weight stream on another branch of a graph the blocks' shared memory keeps the stream's blocks off their SMs, and they are as many as half
// of the SMs at most, below eight a power of two for each row's pages. Six layers of 32 heads of 128 on 8, ms a step by blocks: 2 sequences of 2,048 tokens 0.519 with
// 64, 0.526 with 96, 0.655 with 128 and 0.619 on one branch; 4 of 500 0.523, 0.579 (three for a row), 0.661 and 0.615. 71 heads of 64 on one, a block
// an SM: 8 of 16,384 0.78 with 32, 0.90 with 64 and 0.85 with 24; 16 of 2,048 0.68 with 64, 0.90 with 128.
int splits_of(long long blocks, int pages, int dp, int nh, bool beside) {
  const long long slots = beside ? sm_count() / 2 : (nh >= 4 || dp == 256 ? 1ll : 2ll) * sm_count();
  long long want = blocks > 0 ? slots / blocks : 1;
  if (want > pages / 2) want = pages / 2;
  if (beside && want < MAX_CLUSTER) want = want >= 4 ? 4 : want >= 2 ? 2 : 1;
  if (want > MAX_CLUSTER) {
    const long long wide = (want < pages / 8 ? want : pages / 8) / MAX_CLUSTER * MAX_CLUSTER;
    want = wide > MAX_CLUSTER ? wide : MAX_CLUSTER;
  }
  return int(want < 1 ? 1 : want > 512 ? 512 : want);
}
enum { PTB_NEEDS_WORKSPACE = -1 };
int teams_of(int n_splits) { return n_splits <= MAX_CLUSTER ? 1 : n_splits / MAX_CLUSTER; }
bool splits_known(int n_splits) { return n_splits >= 1 && n_splits <= 512 && (n_splits <= MAX_CLUSTER || n_splits % MAX_CLUSTER == 0); }
}  // namespace

// Blocks that share a row's pages where the caller leaves it open (n_splits 0). rows: query heads of a K/V head times tokens of a tile, at most;
// pages: that a row may see, at most. Prompts' last tiles are seldom full: as many chunks of rows are counted as the step's tokens fill.
static int splits_or(int n_splits, int tiles, int kv_heads, int rows, int tile_tokens, int pages, int tokens, const Plan& q, bool beside = false) {
  if (n_splits > 0) return n_splits;
  const long long chunks = ((long long)rows / tile_tokens * tokens + q.rows_pad - 1) / q.rows_pad;
  return splits_of(kv_heads * (chunks > tiles ? chunks : tiles), pages, q.dp, q.nh, beside);
}

// The choice for a step of single tokens that runs beside a weight stream.
PTB_API int ptb_attention_decode_q8_splits_beside(int seqs, int kv_heads, int rows, int dim, int pages) {
  return splits_or(0, seqs, kv_heads, rows, 1, pages, seqs, plan_of(dim, rows), true);
}

// Floats of workspace (`parts` below) of a call that answered PTB_NEEDS_WORKSPACE, for the same sizes; tokens: of the step.
PTB_API long long ptb_attention_q8_floats(int tiles, int kv_heads, int rows, int tile_tokens, int dim, int n_splits, int pages, int tokens) {
  const Plan q = plan_of(dim, rows);
  const long long chunks = (rows + q.rows_pad - 1) / q.rows_pad;
  const int teams = teams_of(splits_or(n_splits, tiles, kv_heads, rows, tile_tokens, pages, tokens, q));
  return teams > 1 ? (long long)tiles * kv_heads * chunks * teams * q.rows_pad * (dim + 2) : 0;
}

// A step of single tokens. fused [n_seqs, kv_heads * (heads / kv_heads + 2) * dim] bfloat16, out [n_seqs, heads * dim]; pools and exponents as
// in cache_q8.cu. At most 128 query heads a K/V head. n_splits: 1 to 8, a multiple of 8, or 0 for a choice by the sizes and
// `pages`, the most that a sequence spans. PTB_NEEDS_WORKSPACE: nothing was launched, and `parts` has to have ptb_attention_q8_floats floats.
PTB_API int ptb_attention_decode_q8(const void* fused, void* k_pool, void* k_exp, void* v_pool, void* v_exp, int pool_pages, void* out,
                                    const StepBatch* sb, const float* rope_cos, const float* rope_sin, int rot_pairs, int interleaved,
                                    const float* slopes, int heads, int kv_heads, int dim, float scale, int window, int write_cache,
                                    int n_splits, int pages, float* parts, long long part_floats, int* error_flag, cudaStream_t stream) {
  if (sb->n_seqs <= 0) return PTB_OK;
  if (!known(heads, kv_heads, dim, pool_pages) || heads / kv_heads > 128 || sb->n_tokens != sb->n_seqs || rot_pairs < 0 || 2 * rot_pairs > dim ||
      window < 0 || error_flag == nullptr || (rot_pairs > 0 && (rope_cos == nullptr || rope_sin == nullptr)))
    return PTB_ERR_SIZE;
  if (!aligned16(fused) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out) || (reinterpret_cast<uintptr_t>(parts) & 15)) return PTB_ERR_ALIGN;
  const int rows = heads / kv_heads;
  const Plan q = plan_of(dim, rows);
  n_splits = splits_or(n_splits, sb->n_seqs, kv_heads, rows, 1, pages, sb->n_tokens, q);
  if (!splits_known(n_splits)) return PTB_ERR_SIZE;
  if (ptb_attention_q8_floats(sb->n_seqs, kv_heads, rows, 1, dim, n_splits, pages, sb->n_tokens) > part_floats) return PTB_NEEDS_WORKSPACE;
  AttnQ8 p = {};
  p.rows = (const __nv_bfloat16*)fused; p.k_pool = (uint8_t*)k_pool; p.v_pool = (uint8_t*)v_pool; p.k_exp = (int8_t*)k_exp;
  p.v_exp = (int8_t*)v_exp; p.out = (__nv_bfloat16*)out; p.rope_cos = rope_cos; p.rope_sin = rope_sin; p.slopes = slopes;
  p.heads = heads; p.kv_heads = kv_heads; p.dim = dim; p.pool_pages = pool_pages; p.rot_pairs = rot_pairs; p.interleaved = interleaved;
  p.write_cache = write_cache; p.window = window; p.n_splits = n_splits; p.scale = scale; p.parts = parts; p.error_flag = error_flag;
  p.row_groups = q.row_groups; p.page_parts = q.page_parts; p.rings = q.rings; p.stages = q.stages;
  p.teams = teams_of(n_splits); p.cluster = n_splits / p.teams;
  return launch_any<true>(*sb, p, q, dim3(sb->n_seqs, kv_heads, n_splits), stream);
}

// Prompts and chunks whose keys and values are in the pages already: q [tokens, heads, dim] bfloat16, out [tokens, heads * dim]; tiles of at most
// tile_tokens consecutive new tokens of one sequence.
PTB_API int ptb_attention_q8(const void* q_rows, const void* k_pool, const void* k_exp, const void* v_pool, const void* v_exp, int pool_pages,
                             void* out, const StepBatch* sb, const int* tile_seq, const int* tile_q0, int n_tiles, int tile_tokens,
                             const float* slopes, int heads, int kv_heads, int dim, float scale, int window, int n_splits, int pages, float* parts,
                             long long part_floats, int* error_flag, cudaStream_t stream) {
  if (n_tiles <= 0) return PTB_OK;
  if (!known(heads, kv_heads, dim, pool_pages) || window < 0 || error_flag == nullptr || tile_tokens < 1 ||
      (long long)tile_tokens * (heads / kv_heads) > (1 << 24))
    return PTB_ERR_SIZE;
  if (!aligned16(q_rows) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out) || (reinterpret_cast<uintptr_t>(parts) & 15)) return PTB_ERR_ALIGN;
  const int rows = tile_tokens * (heads / kv_heads);
  const Plan q = plan_of(dim, rows);
  n_splits = splits_or(n_splits, n_tiles, kv_heads, rows, tile_tokens, pages, sb->n_tokens, q);
  const long long chunks = (rows + q.rows_pad - 1) / q.rows_pad;
  if (!splits_known(n_splits) || chunks * kv_heads > 65535) return PTB_ERR_SIZE;
  if (ptb_attention_q8_floats(n_tiles, kv_heads, rows, tile_tokens, dim, n_splits, pages, sb->n_tokens) > part_floats) return PTB_NEEDS_WORKSPACE;
  AttnQ8 p = {};
  p.rows = (const __nv_bfloat16*)q_rows; p.k_pool = (uint8_t*)k_pool; p.v_pool = (uint8_t*)v_pool; p.k_exp = (int8_t*)k_exp;
  p.v_exp = (int8_t*)v_exp; p.out = (__nv_bfloat16*)out; p.slopes = slopes; p.tile_seq = tile_seq; p.tile_q0 = tile_q0;
  p.tile_tokens = tile_tokens; p.heads = heads; p.kv_heads = kv_heads; p.dim = dim; p.pool_pages = pool_pages; p.window = window;
  p.n_splits = n_splits; p.scale = scale; p.parts = parts; p.error_flag = error_flag;
  p.row_groups = q.row_groups; p.page_parts = q.page_parts; p.rings = q.rings; p.stages = q.stages;
  p.teams = teams_of(n_splits); p.cluster = n_splits / p.teams;
  return launch_any<false>(*sb, p, q, dim3(n_tiles, unsigned(chunks * kv_heads), n_splits), stream);
}
