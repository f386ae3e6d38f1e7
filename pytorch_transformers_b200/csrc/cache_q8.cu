// Writing to, reading from and copying the pages of a cache in 8 bits (q8.cuh).
#include <new>

#include "q8.cuh"

namespace {

constexpr int STORE_THREADS = 256, Q_HEADS = 4;

// ------------------------------------------------------------------------------------------------ append
// Projection rows into rotated queries, and keys (rotated) and values into the pages.
//
// The first blocks take a page each: (page that the step writes to) x (K/V head) x (keys or values). A page's new rows, 64 at most,
// stay in registers between the reduction that gives its exponent and the rounding: one pass over the projection. One block
// has the page to itself, so no order among blocks can change what a page holds. The other blocks rotate queries: a thread has an eighth of a
// head (with pairs (i, i + n) that eighth and its pairs' other halves) of up to four heads of a token, whose angles are the same.
struct StoreParams {
  const __nv_bfloat16* fused;
  __nv_bfloat16* q_out;
  uint8_t *k_pool, *v_pool;
  int8_t *k_exp, *v_exp;
  const float *rope_cos, *rope_sin;
  int rot_pairs, interleaved, kv_heads, q_per_kv, dim, pool_pages;
  int page_blocks;             // blocks of pages; the others are queries'
  int halves, q_units;         // pairs (i, i + n) in whole eighths; threads for a head
  int* error_flag;
};

// MOST: eighths of a page's rows that a thread holds (4 for heads up to 128, 8 up to 256)
template <int MOST> __global__ void __launch_bounds__(STORE_THREADS) store_q8_kernel(StepBatch sb, StoreParams p) {
  pdl_entry();
  __shared__ float scratch[32];
  const int tid = threadIdx.x, eighths = p.dim / 8, rows = p.q_per_kv + 2;
  const size_t width = size_t(p.kv_heads) * rows * p.dim;
  if (int(blockIdx.x) >= p.page_blocks) {
    const int heads = p.kv_heads * p.q_per_kv, groups = (heads + Q_HEADS - 1) / Q_HEADS;
    const long long i = (long long)(blockIdx.x - p.page_blocks) * STORE_THREADS + tid;
    if (i >= (long long)sb.n_tokens * groups * p.q_units) return;
    const int at = int(i / p.q_units), unit = int(i - (long long)at * p.q_units), t = at / groups, h0 = (at - t * groups) * Q_HEADS;
    const float *rc = p.rope_cos + size_t(t) * p.rot_pairs, *rs = p.rope_sin + size_t(t) * p.rot_pairs;
    const uint4* row = reinterpret_cast<const uint4*>(p.fused + size_t(t) * width);
    uint4* out = reinterpret_cast<uint4*>(p.q_out + size_t(t) * heads * p.dim);
    const int half = p.rot_pairs / 8;
    const bool both = p.halves && unit < half;      // eighth `unit` and the one of its pairs' other halves
    const int c = p.halves && !both ? unit + half : unit;
    uint4 own[Q_HEADS], other[Q_HEADS];
#pragma unroll
    for (int k = 0; k < Q_HEADS; ++k) {
      const int h = min(h0 + k, heads - 1), g = h / p.q_per_kv;
      const uint4* head = row + (g * rows + h - g * p.q_per_kv) * eighths;
      own[k] = head[c];
      other[k] = both ? head[c + half] : own[k];
    }
    if (both) {
      float cs[8], sn[8];
      load_angles(rc, rs, 8 * unit, cs, sn);
#pragma unroll
      for (int k = 0; k < Q_HEADS; ++k) {
        if (h0 + k >= heads) break;
        float x[8], y[8];
        rotate_halves(cs, sn, own[k], other[k], x, y);
        out[(h0 + k) * eighths + c] = pack_bf16x8(x);
        out[(h0 + k) * eighths + c + half] = pack_bf16x8(y);
      }
      return;
    }
    const Angles angles = angles_of(c, rc, rs, p.halves ? 0 : p.rot_pairs, p.interleaved);      // past the rotated entries, or other kinds of pairs
#pragma unroll
    for (int k = 0; k < Q_HEADS; ++k) {
      if (h0 + k >= heads) break;
      const int h = h0 + k, g = h / p.q_per_kv;
      float x[8];
      if (angles.mode == 3) load_rotated8(reinterpret_cast<const __nv_bfloat16*>(row + (g * rows + h - g * p.q_per_kv) * eighths), c, rc, rs, p.rot_pairs, 0, x);
      else rotate8(angles, own[k], own[k], x);
      out[h * eighths + c] = pack_bf16x8(x);
    }
    return;
  }
  if (sb.n_tokens == sb.n_seqs) {      // single tokens: a warp for a row (64 sequences, 8 K/V heads: 3.1 us; a block for each 8.5)
    const int at = blockIdx.x * (STORE_THREADS / 32) + tid / 32, seq = at / (2 * p.kv_heads), g = at % (2 * p.kv_heads) >> 1;
    if (seq >= sb.n_seqs) return;
    const bool keys = (at & 1) == 0;
    const int past = sb.seq_past[seq], index = past / PTB_PAGE;
    const int page = index < sb.pages_stride ? sb.pages[size_t(seq) * sb.pages_stride + index] : -1;
    if (page < 0 || page >= p.pool_pages || sb.seq_new[seq] != 1) {      // 54: as many tokens as sequences, but not one each
      if ((tid & 31) == 0) atomicExch(p.error_flag, sb.seq_new[seq] != 1 ? 54 : 51);
      return;
    }
    const size_t block = size_t(page) * p.kv_heads + g, t = sb.seq_start[seq];
    bool rose;
    append_row(p.fused + t * width + size_t(g * rows + p.q_per_kv + (keys ? 0 : 1)) * p.dim, p.rope_cos + t * p.rot_pairs, p.rope_sin + t * p.rot_pairs,
               keys ? p.rot_pairs : 0, p.interleaved, (keys ? p.k_pool : p.v_pool) + block * PTB_PAGE * p.dim, (keys ? p.k_exp : p.v_exp) + block,
               past % PTB_PAGE, p.dim, nullptr, rose);
    return;
  }
  const int job = blockIdx.x / (2 * p.kv_heads), rest = blockIdx.x % (2 * p.kv_heads);
  const int g = rest >> 1;
  const bool keys = (rest & 1) == 0;
  int local = job;
  const int seq = find_job(sb.n_seqs, local, [&](int s) {
    const int past = sb.seq_past[s], n = sb.seq_new[s];
    return n > 0 ? (past + n - 1) / PTB_PAGE - past / PTB_PAGE + 1 : 0;
  });
  if (seq < 0) return;
  const int past = sb.seq_past[seq], n_new = sb.seq_new[seq], start = sb.seq_start[seq];
  const int index = past / PTB_PAGE + local;
  const int page = index < sb.pages_stride ? sb.pages[size_t(seq) * sb.pages_stride + index] : -1;
  if (page < 0 || page >= p.pool_pages) {      // a table that names no page: said, and nothing is written
    if (tid == 0) atomicExch(p.error_flag, 51);
    return;
  }
  const int first = max(past - index * PTB_PAGE, 0), last = min(past + n_new - index * PTB_PAGE, PTB_PAGE);   // the new rows of the page
  const int t0 = start + index * PTB_PAGE + first - past;
  const size_t block = size_t(page) * p.kv_heads + g;
  uint8_t* codes = (keys ? p.k_pool : p.v_pool) + block * PTB_PAGE * p.dim;
  int8_t* exps = (keys ? p.k_exp : p.v_exp) + block;
  const int old = *exps;
  const __nv_bfloat16* src = p.fused + size_t(g * rows + p.q_per_kv + (keys ? 0 : 1)) * p.dim;
  // keys whose every entry is rotated, in halves: a thread takes an eighth and that of its pairs' other halves, x[k] and x[k + MOST / 2]
  const bool both = keys && p.halves && 2 * p.rot_pairs == p.dim;
  const int half = p.rot_pairs / 8, total = (last - first) * (both ? half : eighths);
  float x[MOST][8];
  float most = 0.f;
  if (both) {
#pragma unroll
    for (int k = 0; k < MOST / 2; ++k) {
      const int i = tid + k * STORE_THREADS;
      if (i < total) {
        const int r = i / half, c = i - r * half;
        const size_t t = t0 + r;
        const uint4* row = reinterpret_cast<const uint4*>(src + t * width);
        float cs[8], sn[8];
        load_angles(p.rope_cos + t * p.rot_pairs, p.rope_sin + t * p.rot_pairs, 8 * c, cs, sn);
        rotate_halves(cs, sn, row[c], row[c + half], x[k], x[k + MOST / 2]);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fmaxf(finite_abs(x[k][e]), finite_abs(x[k + MOST / 2][e])));
      }
    }
  } else
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    const int i = tid + k * STORE_THREADS;
    if (i < total) {
      const int r = i / eighths, c = i - r * eighths;
      const size_t t = t0 + r;
      load_rotated8(src + t * width, c, p.rope_cos + t * p.rot_pairs, p.rope_sin + t * p.rot_pairs, keys ? p.rot_pairs : 0, p.interleaved, x[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, finite_abs(x[k][e]));
    }
  }
  int e = q8_exponent(block_max(most, scratch));
  if (first > 0) {
    e = max(e, old);
    if (e > old) {      // the page's earlier codes, rounded again
      const float down = power_of_two(max(old - e, -126));
      for (int i = tid; i < first * p.dim / 16; i += STORE_THREADS) {
        uint4 w = reinterpret_cast<uint4*>(codes)[i];
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
  const float by = power_of_two(-e);
  auto codes8 = [&](const float (&v)[8]) {
    return make_uint2(q8_pack4(v[0] * by, v[1] * by, v[2] * by, v[3] * by), q8_pack4(v[4] * by, v[5] * by, v[6] * by, v[7] * by));
  };
  if (both) {
#pragma unroll
    for (int k = 0; k < MOST / 2; ++k) {
      const int i = tid + k * STORE_THREADS;
      if (i < total) {
        const int r = i / half, c = i - r * half;
        uint2* to = reinterpret_cast<uint2*>(codes + size_t(first + r) * p.dim) + c;
        to[0] = codes8(x[k]);
        to[half] = codes8(x[k + MOST / 2]);
      }
    }
  } else
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    const int i = tid + k * STORE_THREADS;
    if (i < total) {
      *reinterpret_cast<uint2*>(codes + size_t(first) * p.dim + size_t(i) * 8) = codes8(x[k]);      // rows of a page lie one after another
    }
  }
  if (tid == 0) *exps = int8_t(e);      // every thread has read the old one: the reduction lies between
}

// ------------------------------------------------------------------------------------------------ read back
// Pages as bfloat16 values (exact, but for what lies below bfloat16's normal numbers): those that `ids` names, or with ids null all that
// the step's sequences span from `window` on, one after another, whose places go into `table` (as wide as the step's own) and whose rows behind a
// sequence's last token are zero. Rows of `dim` codes become rows of `out_dim` values, zero beyond dim. A block takes a page of one
// K/V head, keys and values.
struct UnpackParams {
  const uint8_t *k_pool, *v_pool;
  const int8_t *k_exp, *v_exp;
  __nv_bfloat16 *k_out, *v_out;
  const int* ids;
  int* table;
  int kv_heads, dim, out_dim, pool_pages, window;
  int* error_flag;
};
__global__ void __launch_bounds__(256) unpack_q8_kernel(StepBatch sb, UnpackParams p) {
  pdl_entry();
  const int job = blockIdx.x, g = blockIdx.y, tid = threadIdx.x;
  int page, valid = PTB_PAGE;
  if (p.ids) {
    page = p.ids[job];
  } else {
    int local = job;
    auto low = [&](int s) { return p.window > 0 ? max(0, sb.seq_past[s] - p.window + 1) / PTB_PAGE : 0; };
    auto count = [&](int s) { return sb.seq_new[s] > 0 ? (sb.seq_past[s] + sb.seq_new[s] + PTB_PAGE - 1) / PTB_PAGE - low(s) : 0; };
    if (g == 0 && job + 1 == int(gridDim.x)) {      // 55: the step spans more pages than the workspace has
      int more = job + 1;
      if (find_job(sb.n_seqs, more, count) >= 0) {
        if (tid == 0) atomicExch(p.error_flag, 55);
        for (int s = 0, before = 0; s < sb.n_seqs; before += count(s++))      // the places without one name a page that there is
          for (int i = tid; i < count(s); i += 256)
            if (before + i > job && (low(s) + i < sb.pages_stride || (i == 0 && sb.pages_stride > 0)))
              p.table[size_t(s) * sb.pages_stride + min(low(s) + i, sb.pages_stride - 1)] = 0;
      }
    }
    const int seq = find_job(sb.n_seqs, local, count);
    if (seq < 0) return;
    const int index = low(seq) + local;
    const bool listed = index < sb.pages_stride;      // a table too narrow for its sequence is neither read nor written past a row's end
    page = listed ? sb.pages[size_t(seq) * sb.pages_stride + index] : -1;
    valid = min(PTB_PAGE, sb.seq_past[seq] + sb.seq_new[seq] - index * PTB_PAGE);
    if (g == 0 && tid == 0) {
      int* row = p.table + size_t(seq) * sb.pages_stride;
      if (listed) row[index] = job;
      else if (local == 0 && sb.pages_stride > 0) row[sb.pages_stride - 1] = job;      // no place of the row is the sequence's: what stands for all
    }
  }
  const bool known = page >= 0 && page < p.pool_pages;
  if (!known) {
    if (g == 0 && tid == 0) atomicExch(p.error_flag, 51);
    valid = 0;
    page = 0;
  }
  const size_t block = size_t(page) * p.kv_heads + g, to = (size_t(job) * p.kv_heads + g) * PTB_PAGE * p.out_dim;
  const float fk = power_of_two(p.k_exp[block]), fv = power_of_two(p.v_exp[block]);
  const int words = p.out_dim / 16, total = PTB_PAGE * words;
  for (int i = tid; i < 2 * total; i += 256) {
    const bool keys = i < total;
    const int j = keys ? i : i - total, r = j / words, c = j - r * words;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r < valid && c * 16 < p.dim)
      w = *reinterpret_cast<const uint4*>((keys ? p.k_pool : p.v_pool) + (block * PTB_PAGE + r) * p.dim + c * 16);
    const float f = keys ? fk : fv;
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    uint4* out = reinterpret_cast<uint4*>((keys ? p.k_out : p.v_out) + to + size_t(j) * 16);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float a[4], b[4];
      q8_unpack4(u[2 * k], a);
      q8_unpack4(u[2 * k + 1], b);
      const float v[8] = {a[0] * f, a[1] * f, a[2] * f, a[3] * f, b[0] * f, b[1] * f, b[2] * f, b[3] * f};
      out[k] = pack_bf16x8(v);
    }
  }
}

// ------------------------------------------------------------------------------------------------ heads of other sizes
// Rows of `from` entries as rows of `to` entries, zero past `from`, or cut to `to`: heads that the tcgen05 prompt kernel does not take go through it as
// heads of 64 or 128. A thread moves 16 bytes.
__global__ void __launch_bounds__(256) pitch_rows_kernel(const uint4* __restrict__ src, uint4* __restrict__ dst, long long rows, int from, int to) {
  pdl_entry();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long r = i / to;
  const int c = int(i - r * to);
  if (r < rows) dst[i] = c < from ? src[r * from + c] : make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------------------------------------------ copies
// Pages of several tensors [entries][pages][page bytes] in one launch. The pairs travel as the kernel's parameters: no copy of
// them to the device, none of their memory to keep until the kernel has run.
constexpr int COPY_TENSORS = 8, COPY_PAIRS = 960, COPY_THREADS = 256, COPY_ILP = 8;
struct CopyTensor {
  const unsigned char* src;
  unsigned char* dst;
  long long src_entry, dst_entry;      // bytes from one entry's pages to the next's
  long long page_bytes;
  int entries, unit;                   // unit: bytes of a load and store, a power of two up to 16
  long long first_block;               // blocks before this tensor's
  long long units;                     // of all of its pages to copy
};
struct CopyParams {
  CopyTensor t[COPY_TENSORS];
  int n_tensors, n_pairs;
  int src[COPY_PAIRS], dst[COPY_PAIRS];
};
static_assert(sizeof(CopyParams) <= 16384, "kernel parameters");

template <typename W>
__device__ __forceinline__ void copy_units(const CopyParams& p, const CopyTensor& t, long long block) {
  const long long per_page = t.page_bytes / sizeof(W);
  const long long base = block * (COPY_THREADS * COPY_ILP) + threadIdx.x;
  W w[COPY_ILP];
  W* to[COPY_ILP];
  // One division for the first unit (in 32 bits where they do): its 64-bit form for each unit was most of the kernel's time. The
  // others lie COPY_THREADS apart, in the same page or a next one.
  const bool narrow = t.units < (1ll << 32);
  long long page = narrow ? (long long)(unsigned(base) / unsigned(per_page)) : base / per_page;
  long long in = base - page * per_page;
  const W* from = nullptr;
  W* into = nullptr;
#pragma unroll
  for (int k = 0; k < COPY_ILP; ++k) {
    const long long u = base + k * COPY_THREADS;
    if (k > 0) {
      in += COPY_THREADS;
      if (in >= per_page) {
        const long long on = per_page >= COPY_THREADS ? 1 : narrow ? (long long)(unsigned(in) / unsigned(per_page)) : in / per_page;
        page += on;
        in -= on * per_page;
        from = nullptr;
      }
    }
    to[k] = nullptr;
    if (u < t.units) {
      if (from == nullptr) {
        const unsigned entry = unsigned(page) / unsigned(p.n_pairs);      // pages: pairs * entries, below 2^31
        const int pair = int(unsigned(page) - entry * unsigned(p.n_pairs));
        from = reinterpret_cast<const W*>(t.src + (long long)entry * t.src_entry + p.src[pair] * t.page_bytes);
        into = reinterpret_cast<W*>(t.dst + (long long)entry * t.dst_entry + p.dst[pair] * t.page_bytes);
      }
      w[k] = from[in];
      to[k] = into + in;
    }
  }
#pragma unroll
  for (int k = 0; k < COPY_ILP; ++k)
    if (to[k]) *to[k] = w[k];
}

__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(const __grid_constant__ CopyParams p) {
  int i = 0;
  while (i + 1 < p.n_tensors && (long long)blockIdx.x >= p.t[i + 1].first_block) ++i;
  const CopyTensor& t = p.t[i];
  const long long block = blockIdx.x - t.first_block;
  switch (t.unit) {
    case 16: copy_units<uint4>(p, t, block); break;
    case 8: copy_units<uint2>(p, t, block); break;
    case 4: copy_units<uint32_t>(p, t, block); break;
    case 2: copy_units<uint16_t>(p, t, block); break;
    default: copy_units<uint8_t>(p, t, block);
  }
}

bool q8_sizes(int kv_heads, int q_per_kv, int dim) {
  return kv_heads > 0 && q_per_kv > 0 && dim >= 16 && dim <= 256 && dim % 16 == 0 && kv_heads <= 65535;
}
}  // namespace

// fused [n_tokens, kv_heads * (q_per_kv + 2) * dim] bfloat16; q_out [n_tokens, heads, dim] bfloat16; pools [pool_pages, kv_heads, 64, dim]
// e4m3 and exponents [pool_pages, kv_heads] int8, or null to rotate queries only. rope_cos / rope_sin [n_tokens, rot_pairs] float32
// where rot_pairs > 0.
PTB_API int ptb_store_q8(const void* fused, void* q_out, void* k_pool, void* k_exp, void* v_pool, void* v_exp, int pool_pages,
                         const StepBatch* sb, const float* rope_cos, const float* rope_sin, int rot_pairs, int interleaved, int kv_heads,
                         int q_per_kv, int dim, int* error_flag, cudaStream_t stream) {
  if (sb->n_tokens <= 0) return PTB_OK;
  if (!q8_sizes(kv_heads, q_per_kv, dim) || rot_pairs < 0 || 2 * rot_pairs > dim || error_flag == nullptr ||
      (rot_pairs > 0 && (rope_cos == nullptr || rope_sin == nullptr)))
    return PTB_ERR_SIZE;
  if (!aligned16(fused) || !aligned16(q_out) || !aligned16(k_pool) || !aligned16(v_pool)) return PTB_ERR_ALIGN;
  // pages that the step writes to: one for each single token, else at most this
  const long long jobs = k_pool == nullptr ? 0 : sb->n_tokens == sb->n_seqs ? sb->n_seqs : sb->n_tokens / PTB_PAGE + 2ll * sb->n_seqs;
  const long long page_blocks = sb->n_tokens == sb->n_seqs ? (jobs * 2 * kv_heads + STORE_THREADS / 32 - 1) / (STORE_THREADS / 32) : jobs * 2 * kv_heads;
  const int halves = rot_pairs > 0 && !interleaved && rot_pairs % 8 == 0, q_units = dim / 8 - (halves ? rot_pairs / 8 : 0);
  const long long q_groups = ((long long)kv_heads * q_per_kv + Q_HEADS - 1) / Q_HEADS;
  if ((long long)sb->n_tokens * q_groups > 0x7fffffffll) return PTB_ERR_SIZE;
  const long long q_blocks = ((long long)sb->n_tokens * q_groups * q_units + STORE_THREADS - 1) / STORE_THREADS;
  if (page_blocks + q_blocks > 0x7fffffffll) return PTB_ERR_SIZE;
  StoreParams p;
  p.fused = (const __nv_bfloat16*)fused; p.q_out = (__nv_bfloat16*)q_out;
  p.k_pool = (uint8_t*)k_pool; p.v_pool = (uint8_t*)v_pool; p.k_exp = (int8_t*)k_exp; p.v_exp = (int8_t*)v_exp;
  p.rope_cos = rope_cos; p.rope_sin = rope_sin; p.rot_pairs = rot_pairs; p.interleaved = interleaved;
  p.kv_heads = kv_heads; p.q_per_kv = q_per_kv; p.dim = dim; p.pool_pages = pool_pages; p.page_blocks = int(page_blocks);
  p.halves = halves; p.q_units = q_units;
  p.error_flag = error_flag;
  const dim3 grid(unsigned(page_blocks + q_blocks)), block(STORE_THREADS);
  if (dim <= 128) launch_pdl(store_q8_kernel<4>, grid, block, 0, stream, *sb, p);
  else launch_pdl(store_q8_kernel<8>, grid, block, 0, stream, *sb, p);
  return launch_status();
}

// n_pages pages as bfloat16 values [n_pages, kv_heads, 64, out_dim]: those in `ids` (sb and table null), or all that the step spans (ids null; n_pages
// at least as many as there are).
PTB_API int ptb_unpack_q8(const void* k_pool, const void* k_exp, const void* v_pool, const void* v_exp, int pool_pages, const int* ids,
                          const StepBatch* sb, int* table, int n_pages, int window, void* k_out, void* v_out, int kv_heads, int dim,
                          int out_dim, int* error_flag, cudaStream_t stream) {
  if (n_pages <= 0) return PTB_OK;
  if (!q8_sizes(kv_heads, 1, dim) || out_dim < dim || out_dim > 256 || out_dim % 16 != 0 || error_flag == nullptr || pool_pages <= 0 ||
      (ids == nullptr) != (sb != nullptr) || (sb != nullptr && table == nullptr))
    return PTB_ERR_SIZE;
  if (!aligned16(k_pool) || !aligned16(v_pool) || !aligned16(k_out) || !aligned16(v_out)) return PTB_ERR_ALIGN;
  UnpackParams p;
  p.k_pool = (const uint8_t*)k_pool; p.v_pool = (const uint8_t*)v_pool; p.k_exp = (const int8_t*)k_exp; p.v_exp = (const int8_t*)v_exp;
  p.k_out = (__nv_bfloat16*)k_out; p.v_out = (__nv_bfloat16*)v_out; p.ids = ids; p.table = table;
  p.kv_heads = kv_heads; p.dim = dim; p.out_dim = out_dim; p.pool_pages = pool_pages; p.window = window; p.error_flag = error_flag;
  StepBatch none = {};
  launch_pdl(unpack_q8_kernel, dim3(n_pages, kv_heads), dim3(256), 0, stream, sb ? *sb : none, p);
  return launch_status();
}

// `rows` rows of from_dim bfloat16 entries into rows of to_dim (multiples of 8), padded with zeros or cut.
PTB_API int ptb_pitch_rows(const void* src, void* dst, long long rows, int from_dim, int to_dim, cudaStream_t stream) {
  if (rows <= 0) return PTB_OK;
  if (from_dim <= 0 || to_dim <= 0 || from_dim % 8 != 0 || to_dim % 8 != 0 || rows * (to_dim / 8) > (1ll << 38)) return PTB_ERR_SIZE;
  if (!aligned16(src) || !aligned16(dst)) return PTB_ERR_ALIGN;
  launch_pdl(pitch_rows_kernel, dim3(unsigned((rows * (to_dim / 8) + 255) / 256)), dim3(256), 0, stream, (const uint4*)src, (uint4*)dst, rows,
             from_dim / 8, to_dim / 8);
  return launch_status();
}

// src[i] -> dst[i] (host arrays) in each of n_tensors tensors, of which `tensors` has six numbers each: source and target, bytes from an
// entry's pages to the next's in both, bytes of a page, entries. Pages out of range, a target named twice, and a page that is source and
// target at once (where a tensor is copied within itself) are refused before anything is launched: then every order of the
// copies gives the same bytes.
PTB_API int ptb_copy_pages(const long long* tensors, int n_tensors, const int* src, const int* dst, long long n_pairs, int src_pages,
                           int dst_pages, cudaStream_t stream) {
  if (n_pairs <= 0 || n_tensors <= 0) return PTB_OK;
  if (n_tensors > COPY_TENSORS || src_pages < 0 || dst_pages < 0) return PTB_ERR_SIZE;
  bool within = false;
  for (int k = 0; k < n_tensors; ++k) within = within || tensors[6 * k] == tensors[6 * k + 1];
  const size_t marks = size_t(src_pages) + size_t(dst_pages);
  unsigned char* seen = new (std::nothrow) unsigned char[marks + 1]();
  if (seen == nullptr) return PTB_ERR_SIZE;
  int status = PTB_OK;
  for (long long i = 0; i < n_pairs && status == PTB_OK; ++i) {
    if (src[i] < 0 || src[i] >= src_pages || dst[i] < 0 || dst[i] >= dst_pages || seen[size_t(src_pages) + dst[i]]) status = PTB_ERR_PAGES;
    else {
      seen[src[i]] = 1;
      seen[size_t(src_pages) + dst[i]] = 1;
    }
  }
  if (within)
    for (int i = 0; i < src_pages && i < dst_pages && status == PTB_OK; ++i)
      if (seen[i] && seen[size_t(src_pages) + i]) status = PTB_ERR_PAGES;
  delete[] seen;
  if (status != PTB_OK) return status;
  CopyParams p = {};
  for (long long at = 0; at < n_pairs; at += COPY_PAIRS) {
    p.n_pairs = int(n_pairs - at < COPY_PAIRS ? n_pairs - at : COPY_PAIRS);
    p.n_tensors = 0;
    long long blocks = 0;
    for (int k = 0; k < n_tensors; ++k) {
      const long long* v = tensors + 6 * k;
      if (v[4] <= 0 || v[5] <= 0) continue;
      CopyTensor& t = p.t[p.n_tensors++];
      t.src = reinterpret_cast<const unsigned char*>(v[0]); t.dst = reinterpret_cast<unsigned char*>(v[1]);
      t.src_entry = v[2]; t.dst_entry = v[3]; t.page_bytes = v[4]; t.entries = int(v[5]);
      const unsigned long long bits = 16 | reinterpret_cast<uintptr_t>(t.src) | reinterpret_cast<uintptr_t>(t.dst) |
                                      (unsigned long long)t.page_bytes | (unsigned long long)t.src_entry | (unsigned long long)t.dst_entry;
      t.unit = int(bits & (~bits + 1));
      if ((long long)p.n_pairs * t.entries > 0x7fffffffll) return PTB_ERR_SIZE;
      t.units = (long long)p.n_pairs * t.entries * (t.page_bytes / t.unit);
      t.first_block = blocks;
      blocks += (t.units + COPY_THREADS * COPY_ILP - 1) / (COPY_THREADS * COPY_ILP);
    }
    if (blocks == 0) continue;
    if (blocks > 0x7fffffffll) return PTB_ERR_SIZE;
    for (int i = 0; i < p.n_pairs; ++i) {
      p.src[i] = src[at + i];
      p.dst[i] = dst[at + i];
    }
    copy_pages_kernel<<<unsigned(blocks), COPY_THREADS, 0, stream>>>(p);
    status = launch_status();
    if (status != PTB_OK) return status;
  }
  return PTB_OK;
}
