// Attention over a paged cache in 8 bits (q8.cuh), straight from the codes.
//
//   score_j = ((q . code_j) * 2^exp_k + bias_j) * scale      exp_k, exp_v: of the page and K/V head that key j lies in
//   out     = sum_j softmax(score)_j * code'_j * 2^exp_v
//
// Two uses: a step of single tokens (FUSED: rotate the token's queries and key, append key and value to the page, attend, in one
// launch; a block's rows are the query heads of one K/V head), and prompts or chunks whose queries are given (rows: tokens x heads).
//
// What bounds it is the codes' way from memory, so everything is laid out for that. A code becomes a float16 number exactly
// (cvt.rn.f16x2.e4m3x2), and mma.m16n8k16 takes float16 operands; queries are float16 numbers of 11 bits after their row is
// brought to [1, 2) by a power of two, softmax weights float16 of 11 bits (bfloat16 ones of 8 would cost as much error as the
// output's own rounding). Sums, maxima and the output are float32.
//
// A warp has 16 keys at a time to itself: it copies them (16 rows of D codes, keys and values, contiguous in the page)
// with cp.async into a ring of its own, so that no warp waits for another before the end. Which key and which entry an index of the
// matrix instruction stands for is free as long as both operands agree: a thread's share of a key's row is 16 codes in a row (a
// 16-byte load gives four k-steps of B fragments), and its share of a value's row likewise (columns of the output are
// named accordingly, pairs of keys are put together with byte permutes). Nothing is transposed. Rows lie in the ring
// under an exclusive-or of their number, so that both ways of reading are free of bank conflicts.
//
// Pages have exponents of their own: keys' go into the factor of a page's scores; values' are the unit of the float32
// output, which is multiplied by a power of two (exactly) where the unit changes. The unit stays within 2^60 of the largest exponent
// seen, so that the output cannot overflow in small units; smaller pages' weights are scaled instead, which no number notices.
// The running maximum moves only when a score exceeds it by 2^8 (one vote a tile instead of shuffles for each row).
#include "mma_common.cuh"
#include "q8.cuh"

namespace {

constexpr int TILE = 16;              // keys of a step of a warp
constexpr float MOVE_LOG2 = 8.f;      // float16 weights go up to 2^8 then
constexpr int UNIT_RANGE = 60;

struct AttnQ8 {
  const __nv_bfloat16* rows;           // FUSED: the projection; else queries [tokens, heads, dim]
  uint8_t *k_pool, *v_pool;
  int8_t *k_exp, *v_exp;
  __nv_bfloat16* out;
  const float *rope_cos, *rope_sin, *slopes;
  const int *tile_seq, *tile_q0;       // not FUSED
  int tile_tokens;
  int heads, kv_heads, dim, pool_pages, rot_pairs, interleaved, write_cache, window, n_splits;
  int row_groups, key_groups;          // warps = row_groups * key_groups
  float scale;
  float* parts;                        // [grid x][grid y][n_splits][rows][dim + 2] where n_splits > 1
  int* error_flag;
};

template <int DP> struct Q8Shape {
  static constexpr int STAGES = DP == 256 ? 2 : 4;      // 256: beside 68 KB of queries in 128 rows
  static constexpr int STAGE_BYTES = 2 * TILE * DP;      // keys, then values
  static constexpr int Q_PITCH = DP * 2 + 16;
  static constexpr int PITCH = DP + 4;                   // floats of a row of the join
};

// where the 16-byte chunk `c` of the tile's row `key` lies: see the head of the file
template <int DP> __device__ __forceinline__ int place(int key, int c) {
  if (DP == 64) {
    const int row = key ^ ((key >> 2) & 1);
    return row * 64 + ((c ^ (((row >> 1) & 1) << 1)) << 4);
  }
  return key * DP + ((c ^ ((key & 6) ^ ((key & 1) << 2))) << 4);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  uint32_t h;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(h) : "f"(hi), "f"(lo));
  return h;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

// One token's key (or value) into its page, by one warp: the rule of store_q8_kernel for a page that gets one row.
__device__ void append_row(const __nv_bfloat16* row, const float* rc, const float* rs, int P, int interleaved, uint8_t* codes, int8_t* exps,
                           int at, int dim) {
  const int lane = threadIdx.x & 31;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, most = 0.f;
  if (lane * 8 < dim) {
    load_rotated8(row, lane, rc, rs, P, interleaved, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, finite_abs(x[e]));
  }
  int e = q8_exponent(warp_max(most));
  if (at > 0) {
    const int old = __ldcg(reinterpret_cast<const signed char*>(exps));
    e = max(e, old);
    if (e > old) {
      const float down = power_of_two(max(old - e, -126));
      for (int i = lane; i < at * dim / 16; i += 32) {
        uint4 w = __ldcg(reinterpret_cast<const uint4*>(codes) + i);
        uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float f[4];
          q8_unpack4(u[k], f);
          u[k] = q8_pack4(f[0] * down, f[1] * down, f[2] * down, f[3] * down);
        }
        reinterpret_cast<uint4*>(codes)[i] = w;
      }
    }
  }
  __syncwarp();
  const float by = power_of_two(-e);
  if (lane * 8 < dim)
    *reinterpret_cast<uint2*>(codes + size_t(at) * dim + lane * 8) =
        make_uint2(q8_pack4(x[0] * by, x[1] * by, x[2] * by, x[3] * by), q8_pack4(x[4] * by, x[5] * by, x[6] * by, x[7] * by));
  if (lane == 0) *exps = int8_t(e);
}

// MT: tiles of 16 rows that a warp holds; a code is unpacked once for all of them.
template <int DP, int MT, bool FUSED>
__global__ void __launch_bounds__(256, DP == 64 ? 2 : 1) attention_q8_kernel(StepBatch sb, AttnQ8 p) {
  using Shape = Q8Shape<DP>;
  constexpr int STAGES = Shape::STAGES, KS = DP / 16, NT = DP / 8;       // k-steps of a score, 8-column tiles of the output
  constexpr bool Q_REGS = MT * DP <= 128;
  pdl_entry();
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthreads = blockDim.x;
  const int g4 = lane >> 2, t4 = lane & 3;
  const int rg = warp % p.row_groups, kg = warp / p.row_groups;
  const int rows_pad = p.row_groups * 16 * MT;
  unsigned char* q_s = smem;
  int* row_exp = reinterpret_cast<int*>(q_s + size_t(rows_pad) * Shape::Q_PITCH);
  unsigned char* rings = reinterpret_cast<unsigned char*>(row_exp + rows_pad);
  unsigned char* ring = rings + size_t(warp) * STAGES * Shape::STAGE_BYTES;
  const int D = p.dim, qpk = p.heads / p.kv_heads;

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
  if (n_rows <= 0) return;
  const int past = sb.seq_past[seq], start = sb.seq_start[seq];
  const int first_pos = past + q0 + row0 / qpk, last_pos = past + q0 + (row0 + n_rows - 1) / qpk;
  const int low = p.window > 0 ? max(0, first_pos - p.window + 1) : 0;      // the first key that a row sees
  const int* pages = sb.pages + size_t(seq) * sb.pages_stride;
  const int split = blockIdx.z;
  // pages of this block (whole ones: the page that a step appends to has one reader), and of them this warp's tiles
  const int pg0 = low / PTB_PAGE, n_pages = last_pos / PTB_PAGE + 1 - pg0;
  const int pg_begin = pg0 + int((long long)split * n_pages / p.n_splits), pg_end = pg0 + int((long long)(split + 1) * n_pages / p.n_splits);
  const int t_begin = max(pg_begin * (PTB_PAGE / TILE), low / TILE), t_end = min(pg_end * (PTB_PAGE / TILE), last_pos / TILE + 1);

  const int fused_width = p.kv_heads * (qpk + 2) * D;
  if (FUSED && p.write_cache && pg_end == pg0 + n_pages && pg_begin < pg_end) {
    const int page = pages[pg_end - 1];
    const __nv_bfloat16* frow = p.rows + size_t(start) * fused_width + size_t(g) * (qpk + 2) * D;
    if (page >= 0 && page < p.pool_pages) {
      const size_t block = size_t(page) * p.kv_heads + g;
      for (int which = warp; which < 2; which += nthreads >> 5) {
        append_row(frow + size_t(qpk + which) * D, p.rope_cos + size_t(start) * p.rot_pairs, p.rope_sin + size_t(start) * p.rot_pairs,
                   which == 0 ? p.rot_pairs : 0, p.interleaved, (which == 0 ? p.k_pool : p.v_pool) + block * PTB_PAGE * D,
                   (which == 0 ? p.k_exp : p.v_exp) + block, past % PTB_PAGE, D);
        __threadfence();
      }
    }
    __syncthreads();
  }

  // what a lane knows of the warp's tile `lane` of a stretch of 32: its page and the page's exponents
  const int n_mine = t_begin + kg < t_end && rg * 16 * MT < n_rows ? (t_end - t_begin - kg + p.key_groups - 1) / p.key_groups : 0;
  auto look_up = [&](int stretch, int& page, int& exps) {
    const int i = stretch * 32 + lane;
    page = 0;
    exps = 0;
    if (i < n_mine) {
      page = pages[(t_begin + kg + i * p.key_groups) / (PTB_PAGE / TILE)];
      if (page < 0 || page >= p.pool_pages) {
        atomicExch(p.error_flag, 21);
        page = 0;
      }
      const size_t block = size_t(page) * p.kv_heads + g;
      exps = int(__ldcg(reinterpret_cast<const signed char*>(p.k_exp) + block)) * 256 +
             (int(__ldcg(reinterpret_cast<const signed char*>(p.v_exp) + block)) & 255);
    }
  };
  int spot[DP / 32];      // where this lane's 16-byte pieces of a tile go
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) {
    const int piece = lane + 32 * i, per_row = D / 16;
    spot[i] = piece < D ? place<DP>(piece / per_row, piece % per_row) : -1;
  }
  int page_now, exps_now, page_next = 0, exps_next = 0, exps_used;
  look_up(0, page_now, exps_now);
  exps_used = exps_now;
  auto issue = [&](int i) {
    if (i < n_mine) {
      if ((i & 31) == 0 && i > 0) {
        page_now = page_next;
        exps_now = exps_next;
      }
      if ((i & 31) == 16 && i + 16 < n_mine) look_up((i >> 5) + 1, page_next, exps_next);
      const int page = __shfl_sync(0xffffffffu, page_now, i & 31);
      const int t = t_begin + kg + i * p.key_groups;
      const size_t from = ((size_t(page) * p.kv_heads + g) * PTB_PAGE + (t & 3) * TILE) * D + lane * 16;
      const uint32_t to = smem_u32(ring + (i % STAGES) * Shape::STAGE_BYTES);
#pragma unroll
      for (int k = 0; k < DP / 32; ++k)
        if (spot[k] >= 0) {
          cp_async16(to + spot[k], p.k_pool + from + k * 512);
          cp_async16(to + TILE * DP + spot[k], p.v_pool + from + k * 512);
        }
    }
    copy_commit();
  };
  if (D < DP) {      // entries past the head size stay zero: no copy goes there
    for (int i = lane; i < STAGES * Shape::STAGE_BYTES / 16; i += 32) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  for (int i = 0; i < STAGES - 1; ++i) issue(i);      // on their way while the queries are made

  // queries: rotated (FUSED), brought to [1, 2) by a power of two, float16. A group of lanes holds a row, eight entries each.
  {
    constexpr int GL = DP / 8, PER = 32 / GL;
    const int c = lane % GL;
    for (int r = warp * PER + lane / GL; r < rows_pad;      // rows_pad is a multiple of 16: a warp leaves as one
         r += (nthreads >> 5) * PER) {
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (r < n_rows && c * 8 < D) {
        if (FUSED) {
          const __nv_bfloat16* row = p.rows + size_t(start) * fused_width + (size_t(g) * (qpk + 2) + r) * D;
          load_rotated8(row, c, p.rope_cos + size_t(start) * p.rot_pairs, p.rope_sin + size_t(start) * p.rot_pairs, p.rot_pairs,
                        p.interleaved, x);
        } else {
          const size_t t = start + q0 + (row0 + r) / qpk;
          unpack_bf16x8(*reinterpret_cast<const uint4*>(p.rows + (t * p.heads + g * qpk + (row0 + r) % qpk) * D + c * 8), x);
        }
      }
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
      *reinterpret_cast<uint4*>(q_s + size_t(r) * Shape::Q_PITCH + c * 16) = w;
      if (c == 0) row_exp[r] = e;
    }
  }
  __syncthreads();

  const float sl2 = p.scale * 1.4426950408889634f;
  int row_pos[MT][2];
  float row_fac[MT][2], slope[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (rg * MT + mt) * 16 + g4 + 8 * i;
      const bool ok = r < n_rows;
      row_pos[mt][i] = ok ? past + q0 + (row0 + r) / qpk : -1;
      row_fac[mt][i] = power_of_two(row_exp[r]);
      slope[mt][i] = ok && p.slopes ? p.slopes[g * qpk + (row0 + r) % qpk] : 0.f;
      if (!p.slopes) row_fac[mt][i] *= sl2;
    }
  // A fragments of two k-steps from one 16-byte read a row
  auto q_frags = [&](int mt, int step, uint32_t (&a)[4], uint32_t (&b)[4]) {      // steps `step` and step + 1
    const unsigned char* at = q_s + size_t((rg * MT + mt) * 16 + g4) * Shape::Q_PITCH + ((step >> 2) * 64 + t4 * 16 + (step & 3) * 4) * 2;
    const uint4 u = *reinterpret_cast<const uint4*>(at), d = *reinterpret_cast<const uint4*>(at + 8 * Shape::Q_PITCH);
    a[0] = u.x; a[2] = u.y; b[0] = u.z; b[2] = u.w;
    a[1] = d.x; a[3] = d.y; b[1] = d.z; b[3] = d.w;
  };
  uint32_t qa[Q_REGS ? MT : 1][Q_REGS ? KS : 1][4];
  if (Q_REGS) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int s = 0; s < KS; s += 2) q_frags(mt, s, qa[Q_REGS ? mt : 0][Q_REGS ? s : 0], qa[Q_REGS ? mt : 0][Q_REGS ? s + 1 : 0]);
  }

  float o[MT][NT][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int j = 0; j < NT; ++j) o[mt][j][0] = o[mt][j][1] = o[mt][j][2] = o[mt][j][3] = 0.f;
  float m_run[MT][2], l_run[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) m_run[mt][0] = m_run[mt][1] = -INFINITY, l_run[mt][0] = l_run[mt][1] = 0.f;
  int unit = Q8_EXP_MIN, largest = Q8_EXP_MIN;      // of the output; of the values' exponents so far

  for (int i = 0; i < n_mine; ++i) {
    copy_wait<STAGES - 2>();
    __syncwarp();
    issue(i + STAGES - 1);
    if ((i & 31) == 0) exps_used = exps_now;      // the copies are fewer than 32 tiles ahead
    const unsigned char* kt = ring + (i % STAGES) * Shape::STAGE_BYTES;
    const unsigned char* vt = kt + TILE * DP;
    const int key0 = (t_begin + kg + i * p.key_groups) * TILE;
    const int both = __shfl_sync(0xffffffffu, exps_used, i & 31);
    const int ev = int(int8_t(both & 255)), ek = (both - (both & 255)) >> 8;

    // scores
    float s[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < 2; ++j) s[mt][j][0] = s[mt][j][1] = s[mt][j][2] = s[mt][j][3] = 0.f;
#pragma unroll
    for (int r = 0; r < DP / 64; ++r) {
      const uint4 k0 = *reinterpret_cast<const uint4*>(kt + place<DP>(g4, t4 + 4 * r));
      const uint4 k1 = *reinterpret_cast<const uint4*>(kt + place<DP>(8 + g4, t4 + 4 * r));
      const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
      for (int kk = 0; kk < 4; kk += 2) {
        uint32_t b[2][2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          b[u][0][0] = q8_half2(w0[kk + u] & 0xffffu);
          b[u][0][1] = q8_half2(w0[kk + u] >> 16);
          b[u][1][0] = q8_half2(w1[kk + u] & 0xffffu);
          b[u][1][1] = q8_half2(w1[kk + u] >> 16);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t fa[4], fb[4];
          if (!Q_REGS) q_frags(mt, r * 4 + kk, fa, fb);
          const uint32_t(&a0)[4] = Q_REGS ? qa[Q_REGS ? mt : 0][Q_REGS ? r * 4 + kk : 0] : fa;
          const uint32_t(&a1)[4] = Q_REGS ? qa[Q_REGS ? mt : 0][Q_REGS ? r * 4 + kk + 1 : 0] : fb;
          mma_f16(s[mt][0], a0, b[0][0][0], b[0][0][1]);
          mma_f16(s[mt][1], a0, b[0][1][0], b[0][1][1]);
          mma_f16(s[mt][0], a1, b[1][0][0], b[1][0][1]);
          mma_f16(s[mt][1], a1, b[1][1][0], b[1][1][1]);
        }
      }
    }
    // scale, bias and mask; a tile that all rows see whole needs no mask
    const float fk = power_of_two(ek);
    const bool whole = key0 + TILE - 1 <= first_pos && (p.window == 0 || key0 > last_pos - p.window);
    bool moves = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = e >> 1;
          float v = s[mt][j][e] * (row_fac[mt][h] * fk);
          const int key = key0 + j * 8 + t4 * 2 + (e & 1);
          if (p.slopes) v = (v + alibi_bias(slope[mt][h], key)) * sl2;
          if (!whole && (key > row_pos[mt][h] || (p.window > 0 && key <= row_pos[mt][h] - p.window))) v = -INFINITY;
          s[mt][j][e] = v;
          moves = moves || v > m_run[mt][h] + MOVE_LOG2;
        }
    // the unit of the output, and the maxima where one has to move
    largest = max(largest, ev);
    const int unit_new = max(ev, largest - UNIT_RANGE);
    if (__any_sync(0xffffffffu, moves) || unit_new != unit) {
      const float change = power_of_two(min(max(unit - unit_new, -126), 126));
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float m = fmaxf(fmaxf(s[mt][0][2 * h], s[mt][0][2 * h + 1]), fmaxf(s[mt][1][2 * h], s[mt][1][2 * h + 1]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          m = fmaxf(m, m_run[mt][h]);
          const float corr = m_run[mt][h] == -INFINITY ? 0.f : exp2f(m_run[mt][h] - m);
          m_run[mt][h] = m;
          l_run[mt][h] *= corr;
          const float f = corr * change;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            o[mt][j][2 * h] *= f;
            o[mt][j][2 * h + 1] *= f;
          }
        }
      unit = unit_new;
    }
    const float small = power_of_two(max(ev - unit, -126));      // 1 but for pages 2^60 below the largest
    uint32_t pa[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float w[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float m = m_run[mt][h] == -INFINITY ? 0.f : m_run[mt][h];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = fast_exp2(s[mt][j][2 * h + e] - m);
            l_run[mt][h] += x;
            w[j][2 * h + e] = x * small;
          }
      }
      pa[mt][0] = pack_half(w[0][0], w[0][1]);
      pa[mt][1] = pack_half(w[0][2], w[0][3]);
      pa[mt][2] = pack_half(w[1][0], w[1][1]);
      pa[mt][3] = pack_half(w[1][2], w[1][3]);
    }
    // output. Keys that no row of the block sees are taken as zero: their codes may be anything.
    const bool edge = key0 + TILE - 1 > last_pos || key0 < low;
    constexpr int VW = DP == 64 ? 2 : 4;      // words of a key's row a thread takes at a time
#pragma unroll
    for (int rr = 0; rr < (DP + 127) / 128; ++rr) {
      uint32_t v[4][VW];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int key = (u >> 1) * 8 + t4 * 2 + (u & 1);
        if (DP == 64) {
          const uint2 x = *reinterpret_cast<const uint2*>(vt + place<DP>(key, g4 >> 1) + (g4 & 1) * 8);
          v[u][0] = x.x; v[u][1] = x.y;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(vt + place<DP>(key, g4 + 8 * rr));
          v[u][0] = x.x; v[u][1] = x.y; v[u][VW - 2] = x.z; v[u][VW - 1] = x.w;
        }
        if (edge && (key0 + key > last_pos || key0 + key < low)) {
#pragma unroll
          for (int q = 0; q < VW; ++q) v[u][q] = 0u;
        }
      }
#pragma unroll
      for (int q = 0; q < VW; ++q) {
        const uint32_t a01 = __byte_perm(v[0][q], v[1][q], 0x5140), a23 = __byte_perm(v[0][q], v[1][q], 0x7362);
        const uint32_t c01 = __byte_perm(v[2][q], v[3][q], 0x5140), c23 = __byte_perm(v[2][q], v[3][q], 0x7362);
        const uint32_t b0[4] = {q8_half2(a01 & 0xffffu), q8_half2(a01 >> 16), q8_half2(a23 & 0xffffu), q8_half2(a23 >> 16)};
        const uint32_t b1[4] = {q8_half2(c01 & 0xffffu), q8_half2(c01 >> 16), q8_half2(c23 & 0xffffu), q8_half2(c23 >> 16)};
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) mma_f16(o[mt][rr * 16 + q * 4 + e], pa[mt], b0[e], b1[e]);
      }
    }
  }
  copy_wait<0>();
  __syncthreads();      // the rings are done with: the parts of the rows take their place

  // this warp's share of its rows: the mean of the values under its weights, in their own units, then maximum and sum
  float* join = reinterpret_cast<float*>(rings);                                            // [key group][row][PITCH]
  float* join_ml = join + size_t(p.key_groups) * rows_pad * Shape::PITCH;                   // [key group][row][2]
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float l = l_run[mt][h];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const int r = kg * rows_pad + (rg * MT + mt) * 16 + g4 + 8 * h;
      const float inv = l == 0.f ? 0.f : power_of_two(unit) / l;
      if (t4 == 0) {
        join_ml[2 * r] = m_run[mt][h];
        join_ml[2 * r + 1] = l;
      }
      constexpr int COLS = DP == 64 ? 8 : 16;      // entries of the output in a row that a thread holds: [2 t4 + b][COLS]
      float* to = join + size_t(r) * Shape::PITCH;
#pragma unroll
      for (int rr = 0; rr < (DP + 127) / 128; ++rr)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int c = 0; c < COLS; c += 4)
            *reinterpret_cast<float4*>(to + rr * 128 + (2 * t4 + b) * COLS + c) =
                make_float4(o[mt][rr * 16 + c][2 * h + b] * inv, o[mt][rr * 16 + c + 1][2 * h + b] * inv,
                            o[mt][rr * 16 + c + 2][2 * h + b] * inv, o[mt][rr * 16 + c + 3][2 * h + b] * inv);
    }
  __syncthreads();
  const int quads = D / 4;
  float* parts = p.n_splits > 1 ? p.parts + ((size_t(blockIdx.x) * gridDim.y + blockIdx.y) * p.n_splits + split) * size_t(rows_pad) * (D + 2) : nullptr;
  for (int i = tid; i < n_rows * quads; i += nthreads) {
    const int r = i / quads, d = (i - r * quads) * 4;
    float m = -INFINITY;
    for (int k = 0; k < p.key_groups; ++k) m = fmaxf(m, join_ml[2 * (k * rows_pad + r)]);
    float l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    auto weight = [&](int k) {
      const float mk = join_ml[2 * (k * rows_pad + r)], lk = join_ml[2 * (k * rows_pad + r) + 1];
      return mk == -INFINITY && lk == 0.f ? 0.f : lk * exp2f(mk - m);
    };
    for (int k = 0; k < p.key_groups; ++k) l += weight(k);      // always in this order
    const float inv = l == 0.f ? 0.f : 1.f / l;      // before the values: they may be as large as float32 holds
    for (int k = 0; k < p.key_groups; ++k) {
      const float w = weight(k) * inv;
      const float4 v = *reinterpret_cast<const float4*>(join + size_t(k * rows_pad + r) * Shape::PITCH + d);
      if (w != 0.f) { acc[0] += v.x * w; acc[1] += v.y * w; acc[2] += v.z * w; acc[3] += v.w * w; }
    }
    if (p.n_splits > 1) {
      float* to = parts + size_t(r) * (D + 2);
      *reinterpret_cast<float2*>(to + d) = make_float2(acc[0], acc[1]);
      *reinterpret_cast<float2*>(to + d + 2) = make_float2(acc[2], acc[3]);
      if (d == 0) *reinterpret_cast<float2*>(to + D) = make_float2(m, l);
    } else {
      const size_t t = start + q0 + (row0 + r) / qpk;
      *reinterpret_cast<uint2*>(p.out + (t * p.heads + g * qpk + (row0 + r) % qpk) * D + d) =
          make_uint2(pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3]));
    }
  }
}

// The splits' parts of a row into its output, always in the order of the splits.
template <bool FUSED>
__global__ void __launch_bounds__(256) join_q8_kernel(StepBatch sb, AttnQ8 p, int rows_pad, int grid_y) {
  pdl_entry();
  const int x = blockIdx.x, y = blockIdx.y, D = p.dim, qpk = p.heads / p.kv_heads;
  const int g = FUSED ? y : y % p.kv_heads, row0 = FUSED ? 0 : y / p.kv_heads * rows_pad;
  const int seq = FUSED ? x : p.tile_seq[x], q0 = FUSED ? 0 : p.tile_q0[x];
  const int tokens = FUSED ? 1 : min(p.tile_tokens, sb.seq_new[seq] - q0);
  const int n_rows = min(rows_pad, tokens * qpk - row0), quads = D / 4;
  const float* parts = p.parts + (size_t(x) * grid_y + y) * p.n_splits * size_t(rows_pad) * (D + 2);
  const size_t pitch = size_t(rows_pad) * (D + 2);
  for (int i = blockIdx.z * blockDim.x + threadIdx.x; i < n_rows * quads; i += gridDim.z * blockDim.x) {
    const int r = i / quads, d = (i - r * quads) * 4;
    const float* at = parts + size_t(r) * (D + 2);
    float m = -INFINITY;
    for (int s = 0; s < p.n_splits; ++s) m = fmaxf(m, at[s * pitch + D]);
    float l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    auto weight = [&](int s) {
      const float2 ml = *reinterpret_cast<const float2*>(at + s * pitch + D);
      return ml.x == -INFINITY && ml.y == 0.f ? 0.f : ml.y * exp2f(ml.x - m);
    };
    for (int s = 0; s < p.n_splits; ++s) l += weight(s);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int s = 0; s < p.n_splits; ++s) {
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
  int dp, mt, row_groups, key_groups, rows_pad;
};
// rows: of a block's tile at most (more are divided among blocks)
Plan plan_of(int dim, int rows) {
  Plan q;
  q.dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  q.mt = rows > 16 && q.dp <= 128 ? 2 : 1;
  const int groups = (rows + 16 * q.mt - 1) / (16 * q.mt), most = 8 / q.mt;
  q.row_groups = groups < most ? groups : most;
  q.key_groups = 8 / q.row_groups;
  q.rows_pad = q.row_groups * 16 * q.mt;
  return q;
}

template <int DP, int MT, bool FUSED>
int launch_attn(const StepBatch& sb, const AttnQ8& p, const Plan& q, dim3 grid, cudaStream_t stream) {
  using Shape = Q8Shape<DP>;
  const int warps = q.row_groups * q.key_groups;
  const size_t ring = size_t(warps) * Shape::STAGES * Shape::STAGE_BYTES;
  const size_t join = size_t(q.key_groups) * q.rows_pad * (Shape::PITCH + 2) * sizeof(float);
  const size_t smem = size_t(q.rows_pad) * (Shape::Q_PITCH + sizeof(int)) + (ring > join ? ring : join);
  static SharedLimit limit;
  if (!limit.allows(attention_q8_kernel<DP, MT, FUSED>, smem)) return PTB_ERR_LAUNCH;
  launch_pdl(attention_q8_kernel<DP, MT, FUSED>, grid, dim3(warps * 32), smem, stream, sb, p);
  int status = launch_status();
  if (status == PTB_OK && p.n_splits > 1) {
    const int z = max(1, min(8, q.rows_pad * (p.dim / 4) / 512));
    launch_pdl(join_q8_kernel<FUSED>, dim3(grid.x, grid.y, z), dim3(256), 0, stream, sb, p, q.rows_pad, int(grid.y));
    status = launch_status();
  }
  return status;
}
template <bool FUSED>
int launch_any(const StepBatch& sb, const AttnQ8& p, const Plan& q, dim3 grid, cudaStream_t stream) {
  if (q.dp == 64) return q.mt == 1 ? launch_attn<64, 1, FUSED>(sb, p, q, grid, stream) : launch_attn<64, 2, FUSED>(sb, p, q, grid, stream);
  if (q.dp == 128) return q.mt == 1 ? launch_attn<128, 1, FUSED>(sb, p, q, grid, stream) : launch_attn<128, 2, FUSED>(sb, p, q, grid, stream);
  return launch_attn<256, 1, FUSED>(sb, p, q, grid, stream);
}
bool known(int heads, int kv_heads, int dim, int pool_pages) {
  return heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && kv_heads <= 65535 && dim >= 16 && dim <= 256 && dim % 16 == 0 && pool_pages > 0;
}
// Blocks that share a row's pages: about two on every SM in all (one where a block's rings take its shared memory), each with four pages.
int splits_of(long long blocks, int pages, int dp) {
  const long long want = (dp == 64 ? 2ll : 1ll) * sm_count() / (blocks > 0 ? blocks : 1);
  const long long most = pages / 4 < 64 ? pages / 4 : 64;
  return int(want < 1 || most < 1 ? 1 : want < most ? want : most);
}
}  // namespace

// How many blocks share a row's pages (n_splits below) and the floats of workspace that they need: rows = query heads of a K/V head times
// tokens of a tile; tiles = sequences of a step of single tokens, or tiles of a prompt; pages: that a row may see, at most.
PTB_API int ptb_attention_q8_splits(int tiles, int kv_heads, int rows, int dim, int pages) {
  const Plan q = plan_of(dim, rows);
  const long long chunks = (rows + q.rows_pad - 1) / q.rows_pad;
  return splits_of((long long)tiles * kv_heads * chunks, pages, q.dp);
}
PTB_API long long ptb_attention_q8_floats(int tiles, int kv_heads, int rows, int dim, int n_splits) {
  const Plan q = plan_of(dim, rows);
  const long long chunks = (rows + q.rows_pad - 1) / q.rows_pad;
  return n_splits > 1 ? (long long)tiles * kv_heads * chunks * n_splits * q.rows_pad * (dim + 2) : 0;
}

// A step of single tokens. fused [n_seqs, kv_heads * (heads / kv_heads + 2) * dim] bfloat16, out [n_seqs, heads * dim]; pools and exponents as
// in cache_q8.cu. At most 128 query heads a K/V head.
PTB_API int ptb_attention_decode_q8(const void* fused, void* k_pool, void* k_exp, void* v_pool, void* v_exp, int pool_pages, void* out,
                                    const StepBatch* sb, const float* rope_cos, const float* rope_sin, int rot_pairs, int interleaved,
                                    const float* slopes, int heads, int kv_heads, int dim, float scale, int window, int write_cache,
                                    int n_splits, float* parts, long long part_floats, int* error_flag, cudaStream_t stream) {
  if (sb->n_seqs <= 0) return PTB_OK;
  if (!known(heads, kv_heads, dim, pool_pages) || heads / kv_heads > 128 || sb->n_tokens != sb->n_seqs || rot_pairs < 0 || 2 * rot_pairs > dim ||
      window < 0 || n_splits < 1 || n_splits > 65535 || error_flag == nullptr || (rot_pairs > 0 && (rope_cos == nullptr || rope_sin == nullptr)))
    return PTB_ERR_SIZE;
  if (!aligned16(fused) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out) || (reinterpret_cast<uintptr_t>(parts) & 15)) return PTB_ERR_ALIGN;
  if (ptb_attention_q8_floats(sb->n_seqs, kv_heads, heads / kv_heads, dim, n_splits) > part_floats) return PTB_ERR_SIZE;
  AttnQ8 p = {};
  p.rows = (const __nv_bfloat16*)fused; p.k_pool = (uint8_t*)k_pool; p.v_pool = (uint8_t*)v_pool; p.k_exp = (int8_t*)k_exp;
  p.v_exp = (int8_t*)v_exp; p.out = (__nv_bfloat16*)out; p.rope_cos = rope_cos; p.rope_sin = rope_sin; p.slopes = slopes;
  p.heads = heads; p.kv_heads = kv_heads; p.dim = dim; p.pool_pages = pool_pages; p.rot_pairs = rot_pairs; p.interleaved = interleaved;
  p.write_cache = write_cache; p.window = window; p.n_splits = n_splits; p.scale = scale; p.parts = parts; p.error_flag = error_flag;
  const Plan q = plan_of(dim, heads / kv_heads);
  p.row_groups = q.row_groups; p.key_groups = q.key_groups;
  return launch_any<true>(*sb, p, q, dim3(sb->n_seqs, kv_heads, n_splits), stream);
}

// Prompts and chunks whose keys and values are in the pages already: q [tokens, heads, dim] bfloat16, out [tokens, heads * dim]; tiles of at most
// tile_tokens consecutive new tokens of one sequence.
PTB_API int ptb_attention_q8(const void* q_rows, const void* k_pool, const void* k_exp, const void* v_pool, const void* v_exp, int pool_pages,
                             void* out, const StepBatch* sb, const int* tile_seq, const int* tile_q0, int n_tiles, int tile_tokens,
                             const float* slopes, int heads, int kv_heads, int dim, float scale, int window, int n_splits, float* parts,
                             long long part_floats, int* error_flag, cudaStream_t stream) {
  if (n_tiles <= 0) return PTB_OK;
  if (!known(heads, kv_heads, dim, pool_pages) || window < 0 || n_splits < 1 || n_splits > 65535 || error_flag == nullptr || tile_tokens < 1 ||
      (long long)tile_tokens * (heads / kv_heads) > (1 << 24))
    return PTB_ERR_SIZE;
  if (!aligned16(q_rows) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out) || (reinterpret_cast<uintptr_t>(parts) & 15)) return PTB_ERR_ALIGN;
  const int rows = tile_tokens * (heads / kv_heads);
  if (ptb_attention_q8_floats(n_tiles, kv_heads, rows, dim, n_splits) > part_floats) return PTB_ERR_SIZE;
  const Plan q = plan_of(dim, rows);
  const long long chunks = (rows + q.rows_pad - 1) / q.rows_pad;
  if (chunks * kv_heads > 65535) return PTB_ERR_SIZE;
  AttnQ8 p = {};
  p.rows = (const __nv_bfloat16*)q_rows; p.k_pool = (uint8_t*)k_pool; p.v_pool = (uint8_t*)v_pool; p.k_exp = (int8_t*)k_exp;
  p.v_exp = (int8_t*)v_exp; p.out = (__nv_bfloat16*)out; p.slopes = slopes; p.tile_seq = tile_seq; p.tile_q0 = tile_q0;
  p.tile_tokens = tile_tokens; p.heads = heads; p.kv_heads = kv_heads; p.dim = dim; p.pool_pages = pool_pages; p.window = window;
  p.n_splits = n_splits; p.scale = scale; p.parts = parts; p.error_flag = error_flag;
  p.row_groups = q.row_groups; p.key_groups = q.key_groups;
  return launch_any<false>(*sb, p, q, dim3(n_tiles, unsigned(chunks * kv_heads), n_splits), stream);
}
