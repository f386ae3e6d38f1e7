// Writing to, reading from and copying the pages of a cache in 8 bits (q8.cuh).
#include <new>

#include "q8.cuh"

namespace {

constexpr int STORE_THREADS = 256;

// ------------------------------------------------------------------------------------------------ append
// Projection rows into rotated queries, and keys (rotated) and values into the pages.
//
// The first blocks take a page each: (page that the step writes to) x (K/V head) x (keys or values). A page's new rows, 64 at most,
// stay in registers between the reduction that gives its exponent and the rounding: one pass over the projection. One block
// has the page to itself, so no order among blocks can change what a page holds. The other blocks rotate queries, a
// thread eight entries at a time.
struct StoreParams {
  const __nv_bfloat16* fused;
  __nv_bfloat16* q_out;
  uint8_t *k_pool, *v_pool;
  int8_t *k_exp, *v_exp;
  const float *rope_cos, *rope_sin;
  int rot_pairs, interleaved, kv_heads, q_per_kv, dim, pool_pages;
  int page_blocks;             // blocks of pages; the others are queries'
  int* error_flag;
};

// MOST: eighths of a page's rows that a thread holds (4 for heads up to 128, 8 up to 256)
template <int MOST> __global__ void __launch_bounds__(STORE_THREADS) store_q8_kernel(StepBatch sb, StoreParams p) {
  pdl_entry();
  __shared__ float scratch[32];
  const int tid = threadIdx.x, eighths = p.dim / 8, rows = p.q_per_kv + 2;
  const size_t width = size_t(p.kv_heads) * rows * p.dim;
  if (int(blockIdx.x) >= p.page_blocks) {
    const int heads = p.kv_heads * p.q_per_kv;
    const long long total = (long long)sb.n_tokens * heads * eighths;
    const long long i = (long long)(blockIdx.x - p.page_blocks) * STORE_THREADS + tid;
    if (i >= total) return;
    const int c = int(i % eighths);
    const long long th = i / eighths;
    const int h = int(th % heads), t = int(th / heads);
    const int g = h / p.q_per_kv;
    const __nv_bfloat16* row = p.fused + size_t(t) * width + size_t(g * rows + h - g * p.q_per_kv) * p.dim;
    float x[8];
    load_rotated8(row, c, p.rope_cos + size_t(t) * p.rot_pairs, p.rope_sin + size_t(t) * p.rot_pairs, p.rot_pairs, p.interleaved, x);
    *reinterpret_cast<uint4*>(p.q_out + (size_t(th) * eighths + c) * 8) = pack_bf16x8(x);
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
  const int page = sb.pages[size_t(seq) * sb.pages_stride + index];
  if (page < 0 || page >= p.pool_pages) {      // a table that names no page: said, and nothing is written
    if (tid == 0) atomicExch(p.error_flag, 21);
    return;
  }
  const int first = max(past - index * PTB_PAGE, 0), last = min(past + n_new - index * PTB_PAGE, PTB_PAGE);   // the new rows of the page
  const int t0 = start + index * PTB_PAGE + first - past;
  const size_t block = size_t(page) * p.kv_heads + g;
  uint8_t* codes = (keys ? p.k_pool : p.v_pool) + block * PTB_PAGE * p.dim;
  int8_t* exps = (keys ? p.k_exp : p.v_exp) + block;
  const int old = *exps;
  const __nv_bfloat16* src = p.fused + size_t(g * rows + p.q_per_kv + (keys ? 0 : 1)) * p.dim;
  const int total = (last - first) * eighths;
  float x[MOST][8];
  float most = 0.f;
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
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    const int i = tid + k * STORE_THREADS;
    if (i < total) {
      const uint2 w = make_uint2(q8_pack4(x[k][0] * by, x[k][1] * by, x[k][2] * by, x[k][3] * by),
                                 q8_pack4(x[k][4] * by, x[k][5] * by, x[k][6] * by, x[k][7] * by));
      *reinterpret_cast<uint2*>(codes + size_t(first) * p.dim + size_t(i) * 8) = w;      // rows of a page lie one after another
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
    const int seq = find_job(sb.n_seqs, local, [&](int s) {
      return sb.seq_new[s] > 0 ? (sb.seq_past[s] + sb.seq_new[s] + PTB_PAGE - 1) / PTB_PAGE - low(s) : 0;
    });
    if (seq < 0) return;
    const int index = low(seq) + local;
    page = sb.pages[size_t(seq) * sb.pages_stride + index];
    valid = min(PTB_PAGE, sb.seq_past[seq] + sb.seq_new[seq] - index * PTB_PAGE);
    if (g == 0 && tid == 0) p.table[size_t(seq) * sb.pages_stride + index] = job;
  }
  const bool known = page >= 0 && page < p.pool_pages;
  if (!known) {
    if (g == 0 && tid == 0) atomicExch(p.error_flag, 21);
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
#pragma unroll
  for (int k = 0; k < COPY_ILP; ++k) {
    const long long u = base + k * COPY_THREADS;
    to[k] = nullptr;
    if (u < t.units) {
      const long long page = u / per_page, in = u - page * per_page;
      const int pair = int(page % p.n_pairs);
      const long long entry = page / p.n_pairs;
      w[k] = *(reinterpret_cast<const W*>(t.src + entry * t.src_entry + p.src[pair] * t.page_bytes) + in);
      to[k] = reinterpret_cast<W*>(t.dst + entry * t.dst_entry + p.dst[pair] * t.page_bytes) + in;
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
  const long long page_blocks = jobs * 2 * kv_heads;
  const long long q_blocks = ((long long)sb->n_tokens * kv_heads * q_per_kv * (dim / 8) + STORE_THREADS - 1) / STORE_THREADS;
  if (page_blocks + q_blocks > 0x7fffffffll) return PTB_ERR_SIZE;
  StoreParams p;
  p.fused = (const __nv_bfloat16*)fused; p.q_out = (__nv_bfloat16*)q_out;
  p.k_pool = (uint8_t*)k_pool; p.v_pool = (uint8_t*)v_pool; p.k_exp = (int8_t*)k_exp; p.v_exp = (int8_t*)v_exp;
  p.rope_cos = rope_cos; p.rope_sin = rope_sin; p.rot_pairs = rot_pairs; p.interleaved = interleaved;
  p.kv_heads = kv_heads; p.q_per_kv = q_per_kv; p.dim = dim; p.pool_pages = pool_pages; p.page_blocks = int(page_blocks);
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

// src[i] -> dst[i] (host arrays) in each of n_tensors tensors: pages of page_bytes[k] bytes, entries of src_entry[k] and dst_entry[k] bytes.
// Pages out of range, a target named twice, and a page that is source and target at once (where a tensor is copied within itself) are
// refused before anything is launched: then every order of the copies gives the same bytes.
PTB_API int ptb_copy_pages(const void* const* src_base, void* const* dst_base, const long long* src_entry, const long long* dst_entry,
                           const long long* page_bytes, const int* entries, int n_tensors, const int* src, const int* dst, long long n_pairs,
                           int src_pages, int dst_pages, cudaStream_t stream) {
  if (n_pairs <= 0 || n_tensors <= 0) return PTB_OK;
  if (n_tensors > COPY_TENSORS || src_pages < 0 || dst_pages < 0) return PTB_ERR_SIZE;
  bool within = false;
  for (int k = 0; k < n_tensors; ++k) within = within || src_base[k] == dst_base[k];
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
      if (page_bytes[k] <= 0 || entries[k] <= 0) continue;
      CopyTensor& t = p.t[p.n_tensors++];
      t.src = (const unsigned char*)src_base[k]; t.dst = (unsigned char*)dst_base[k];
      t.src_entry = src_entry[k]; t.dst_entry = dst_entry[k]; t.page_bytes = page_bytes[k]; t.entries = entries[k];
      const unsigned long long bits = 16 | reinterpret_cast<uintptr_t>(t.src) | reinterpret_cast<uintptr_t>(t.dst) |
                                      (unsigned long long)t.page_bytes | (unsigned long long)t.src_entry | (unsigned long long)t.dst_entry;
      t.unit = int(bits & (~bits + 1));
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
