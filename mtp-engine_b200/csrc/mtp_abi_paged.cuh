// mtp_abi_paged.cuh -- C entry points of the operators that serve from a paged
// cache: query/key norm with rotation and cache write, prompt and decode
// attention with a window, eviction.  Included by mtp_abi.cu (argument checks,
// plans and launches only; the kernels are in the headers named below).
#pragma once

#include "mtp_kvevict.cuh"
#include "mtp_promptattn_tc.cuh"
#include "mtp_qknorm_rope.cuh"
#include "mtp_splitattn.cuh"

namespace {

// Launch of a kernel that reads what the one before it on the stream wrote
// (griddepcontrol.wait): its blocks are set up while that one runs out.
template <typename Kern, typename... A>
int launch_dependent(Kern kern, unsigned grid_x, unsigned grid_y, int threads, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid_x, grid_y, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MTP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
  MTP_LAUNCH_CHECK();
  return MTP_OK;
}

// a dtype code from an 8-byte member, out of range where it is none
int code(int64_t dtype) { return dtype >= 0 && dtype <= MTP_DTYPE_E4M3 ? (int)dtype : -1; }

bool pool_fits(int64_t P, int64_t B, int64_t H, int64_t ps) {
  // rows of the pool are numbered in 32 bits (a row is D elements)
  return (double)P * B * H * ps < 2147483647.0;
}

// ---------------------------------------------------------------- norm + rotation
template <typename T>
int launch_rope_vec(const rope::Args& a, int lph, unsigned gx, unsigned gy, cudaStream_t s) {
#define MTP_ROPE(L)                                                                              \
  (a.interleaved ? rope::qk_norm_rope_kernel<T, L, true><<<dim3(gx, gy), rope::kThreads, 0, s>>>(a) \
                 : rope::qk_norm_rope_kernel<T, L, false><<<dim3(gx, gy), rope::kThreads, 0, s>>>(a))
  if (lph == 4) MTP_ROPE(4);
  else if (lph == 8) MTP_ROPE(8);
  else MTP_ROPE(16);
#undef MTP_ROPE
  MTP_LAUNCH_CHECK();
  return MTP_OK;
}

// ---------------------------------------------------------------- window attention
enum WindowPath { kPathTensor, kPathSplit, kPathAny };
constexpr int kNoWindow = 1 << 30;  // positions stay below it, so differences of positions fit 32 bits

struct WindowPlan {
  WindowPath path = kPathAny;
  int dp = 0;  // head size of the tiles
  int row_tiles = 1, max_warps = 1, min_blocks = 1;
  int tpt = 0, pairs = 0, splits = 1;  // tensor-core tiles
  int window = kNoWindow, sinks = 0;   // as the kernels take them
  int64_t score_ld = 0;
  size_t part_o = 0, part_ml = 0, scores = 0, row_ml = 0;  // bytes
  size_t total() const { return part_o + part_ml + scores + row_ml + 256; }
};

// Blocks of 16 keys that a warp takes at least before another warp joins in
// (one sequence of 4096: 2 blocks 18.4 us, 4 16.4, 8 18.5).
constexpr int kSplitMinBlocks = 4;

// Which kernel, from types, sizes and alignment alone:
//   16-bit, head sizes 64 .. 128 in steps of 8, more than 16 rows per key head: tcgen05 tiles;
//   other 16-bit calls with head sizes up to 256 in steps of 8: warp-level tiles of 16 rows;
//   everything else: one block per row, fp32.
WindowPlan window_plan(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_keys, int64_t window,
                       int64_t sinks, int dtype, bool aligned, bool weights) {
  WindowPlan p;
  // The caller's window and sinks may be anything up to 2^63 - 1 ("everything").
  // Brought below 2^30 here, before any sum with them: the sizes below and the
  // kernels go by the same values.
  if (window > 0 && window <= kNoWindow) {
    p.window = (int)window;
    p.sinks = (int)(sinks < 0 ? 0 : (sinks < kNoWindow ? sinks : kNoWindow));
  }
  const int64_t reach = (int64_t)p.window + p.sinks;  // the most keys that one row sees
  const int64_t G = Hq / Hkv;
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = sm_count(dev >= 0 && dev < kMaxDevices ? dev : 0);
  const bool wide = is16bit(dtype) && aligned && D % 8 == 0 && D <= 256;
  if (wide && D >= 64 && D <= 128 && S > 1 && S * G > split::kRows && G <= 128) {
    p.path = kPathTensor;
    p.dp = D <= 64 ? 64 : 128;
    p.tpt = (int)(128 / G);
    p.pairs = (int)((S + 2 * p.tpt - 1) / (2 * p.tpt));
    const double items = (double)B * Hkv * p.pairs;
    int64_t most = max_keys;
    if (reach + 2 * p.tpt < most) most = reach + 2 * p.tpt;
    const int64_t chunks = most / attn::kChunk + 1;
    // Fewer items than SMs, or a last round that leaves most of them idle: cut
    // the chunk lists.  Cost in chunks: a round is one piece and about 1.5
    // chunks of set-up and output; joining the pieces costs a launch and writing
    // and reading them (256 rows of D fp32 each; a chunk takes about 2 us).  The
    // constants fit one case, 512 rows behind 32000 keys (363 us without the
    // joining's cost, 354 with it).
    // The lengths are on the device, so the plan goes by the table's width: in a
    // table far wider than its sequences, short prompts are cut for nothing
    // (Hq 32, Hkv 8, D 128, one prompt in a table of its own length and in one
    // of 32768: 512 tokens 25 and 44 us, 1024 33 and 85, 2048 55 and 142, with
    // 77-136 MB of scratch; 8192 524 and 528).
    double best = 0;
    for (int n = 1; n <= 32 && n * 2 <= chunks + 1; ++n) {
      if (n > 1 && items * n > 8.0 * sms) break;
      const double rounds = (double)(int64_t)((items * n + sms - 1) / sms);
      const double cost = rounds * ((double)chunks / n + 1.5) + (n > 1 ? 2.0 + items * n * D * 1.6e-4 : 0.0);
      if (n == 1 || cost < best) {
        best = cost;
        p.splits = n;
      }
    }
    if (p.splits > 1) {
      const size_t slots = (size_t)B * Hkv * p.pairs * p.splits * 256;
      p.part_o = align256(slots * D * 4);
      p.part_ml = align256(slots * 2 * 4);
    }
    return p;
  }
  if (wide) {
    int64_t most = max_keys;  // keys that one tile of rows sees
    if (reach + split::kRows < most) most = reach + split::kRows;
    p.path = kPathSplit;
    p.dp = D <= 64 ? 64 : (D <= 128 ? 128 : 256);
    p.row_tiles = (int)((S * G + split::kRows - 1) / split::kRows);
    const int per_sm = p.dp == 64 ? 4 : (p.dp == 128 ? 2 : 1);  // by shared memory: 48, 96, 192 KB a block
    const double blocks = (double)B * p.row_tiles * Hkv * ((most + split::kKeys - 1) / split::kKeys);
    p.min_blocks = kSplitMinBlocks;
    const int64_t all = (int64_t)sms * per_sm * split::kWarps;
    const double want = blocks / p.min_blocks;
    p.max_warps = (int)(want < 1 ? 1 : (want > (double)all ? all : (int64_t)want));
    p.part_o = align256((size_t)p.max_warps * 2 * split::kRows * D * 4);
    p.part_ml = align256((size_t)p.max_warps * 2 * split::kRows * 2 * 4);
  }
  if (weights) {
    p.score_ld = (max_keys + split::kKeys - 1) / split::kKeys * split::kKeys;
    if (reach + split::kKeys < p.score_ld) p.score_ld = (reach + split::kKeys) / split::kKeys * split::kKeys;
    p.scores = align256((size_t)B * Hq * p.score_ld * 4);
    p.row_ml = align256((size_t)B * Hq * 2 * 4);
  }
  return p;
}

template <int AB_FMT, int DP>
int launch_prompt_inst(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const prompt::Params& p,
                       int sms, int dev, cudaStream_t s) {
  static bool attr[kMaxDevices] = {};
  constexpr int smem = prompt::smem_bytes(DP);
  if (int st = set_smem_once(prompt::prompt_attention_tc_kernel<AB_FMT, DP>, smem, attr, dev)) return st;
  const unsigned grid = (unsigned)(p.items < sms ? p.items : sms);
  prompt::prompt_attention_tc_kernel<AB_FMT, DP><<<grid, prompt::kThreads, smem, s>>>(tq, tk, tv, p);
  MTP_LAUNCH_CHECK();
  if (p.splits == 1) return MTP_OK;
  const int64_t warps = (int64_t)p.B * p.S * p.Hq;
  return launch_dependent(prompt::prompt_merge_kernel<typename std::conditional<AB_FMT == 1, __nv_bfloat16, __half>::type>,
                          (unsigned)((warps + 7) / 8), 1, 256, s, p);
}

int launch_prompt(const split::Args& a, const WindowPlan& pl, cudaStream_t s) {
  const int ps = (int)a.page_size;
  prompt::Params p{};
  p.slab = ps % attn::kChunk == 0 ? attn::kChunk
                                  : (ps >= 8 && attn::kChunk % ps == 0 ? ps : 0);
  const uint64_t D = a.D, E = 2;
  CUtensorMap tq, tk, tv;
  {
    const uint64_t dims[4] = {D, (uint64_t)a.Hq, (uint64_t)a.S, (uint64_t)a.B};
    const uint64_t str[3] = {D * E, (uint64_t)a.Hq * D * E, (uint64_t)a.S * a.Hq * D * E};
    const uint32_t box[4] = {64, (uint32_t)a.G, (uint32_t)pl.tpt, 1};
    if (int st = make_map(&tq, a.q, a.dtype, 4, dims, str, box)) return st;
  }
  {
    // pools as [P * B * Hkv * page_size, D]: one (page, b, h) slab = page_size consecutive rows
    const uint64_t rows = (uint64_t)a.num_pages * a.B * a.Hkv * ps;
    const uint64_t dims[2] = {D, rows > 0 ? rows : 1};
    const uint64_t str[1] = {D * E};
    const uint32_t box[2] = {64, (uint32_t)(p.slab > 0 ? p.slab : 8)};
    const void* k = rows > 0 ? a.k_pages : a.q;  // an empty pool is never read
    const void* v = rows > 0 ? a.v_pages : a.q;
    if (int st = make_map(&tk, k, a.dtype, 2, dims, str, box)) return st;
    if (int st = make_map(&tv, v, a.dtype, 2, dims, str, box)) return st;
  }
  p.page_table = a.page_table;
  p.table_stride = a.table_stride;
  p.k_pool = static_cast<const uint8_t*>(a.k_pages);
  p.v_pool = static_cast<const uint8_t*>(a.v_pages);
  p.seq_lens = a.seq_lens;
  p.q_lens = a.q_lens;
  p.out = a.out;
  p.part_o = a.part_o;
  p.part_ml = a.part_ml;
  p.B = a.B;
  p.S = a.S;
  p.Hq = a.Hq;
  p.Hkv = a.Hkv;
  p.G = a.G;
  p.D = a.D;
  p.ps = ps;
  p.num_pages = (int)a.num_pages;
  p.window = a.window;
  p.sinks = a.sinks;
  p.tpt = pl.tpt;
  p.pairs = pl.pairs;
  p.splits = pl.splits;
  p.items = a.B * a.Hkv * pl.pairs * pl.splits;
  p.table_vec = aligned16(a.page_table) && a.table_stride % 4 == 0;
  p.scale_log2 = a.scale_log2;
  int dev;
  if (int st = current_device(&dev)) return st;
  const int sms = sm_count(dev);
  if (a.dtype == MTP_DTYPE_BF16)
    return pl.dp == 64 ? launch_prompt_inst<1, 64>(tq, tk, tv, p, sms, dev, s)
                       : launch_prompt_inst<1, 128>(tq, tk, tv, p, sms, dev, s);
  return pl.dp == 64 ? launch_prompt_inst<0, 64>(tq, tk, tv, p, sms, dev, s)
                     : launch_prompt_inst<0, 128>(tq, tk, tv, p, sms, dev, s);
}

template <typename T, int DP, bool MANY>
int launch_split_inst(const split::Args& a, cudaStream_t s) {
  static bool attr[kMaxDevices] = {};
  int dev;
  if (int st = current_device(&dev)) return st;
  constexpr int smem = split::smem_bytes(DP);
  if (int st = set_smem_once(split::split_attention_kernel<T, DP, MANY>, smem, attr, dev)) return st;
  const unsigned grid = (unsigned)((a.max_warps + split::kWarps - 1) / split::kWarps);
  split::split_attention_kernel<T, DP, MANY><<<grid, split::kThreads, smem, s>>>(a);
  MTP_LAUNCH_CHECK();
  const int64_t per_unit = (int64_t)a.S * a.G < split::kRows ? (int64_t)a.S * a.G : split::kRows;
  const unsigned rows = (unsigned)((int64_t)a.B * a.row_tiles * a.Hkv * per_unit);
  return launch_dependent(split::split_merge_kernel<T>, rows, 1, split::kMergeWarps * 32, s, a);
}

template <typename T>
int launch_split_t(const split::Args& a, int dp, cudaStream_t s) {
  const bool many = a.S > 1;
  if (dp == 64) return many ? launch_split_inst<T, 64, true>(a, s) : launch_split_inst<T, 64, false>(a, s);
  if (dp == 128) return many ? launch_split_inst<T, 128, true>(a, s) : launch_split_inst<T, 128, false>(a, s);
  return many ? launch_split_inst<T, 256, true>(a, s) : launch_split_inst<T, 256, false>(a, s);
}

// ---------------------------------------------------------------- eviction
template <typename V>
int launch_move(const evict::Args& a, int words, int lanes, cudaStream_t s) {
  const unsigned grid = (unsigned)((int64_t)a.B * a.H * 2 * (words / lanes));
  return launch_dependent(evict::evict_move_kernel<V>, grid, 1, evict::kMoveThreads, s, a, words, lanes);
}

}  // namespace

extern "C" {

int mtp_qk_norm_rope(const mtp_qk_norm_rope_args* args) {
  MTP_NVTX("mtp_qk_norm_rope");
  if (!args) return fail(MTP_ERR_ARG, "null arguments");
  const mtp_qk_norm_rope_args& g = *args;
  const int64_t B = g.B, S = g.S, Hq = g.Hq, Hkv = g.Hkv, D = g.D, rot_dim = g.rot_dim, max_pos = g.max_pos;
  const int64_t table_stride = g.table_stride, num_pages = g.num_pages, page_size = g.page_size;
  const int dtype = code(g.dtype), q_weight_dtype = code(g.q_weight_dtype), k_weight_dtype = code(g.k_weight_dtype);
  const void *q = g.q, *k = g.k, *v = g.v, *q_weight = g.q_weight, *k_weight = g.k_weight;
  void *q_out = g.q_out, *k_out = g.k_out, *k_pages = g.k_pages, *v_pages = g.v_pages;
  const int32_t *positions = g.positions, *page_table = g.page_table, *start = g.start;
  const float *cos = g.cos, *sin = g.sin;
  const bool paged = page_table != nullptr;
  if (B < 0 || S < 0 || Hq < 0 || Hkv < 0 || D <= 0 || max_pos < 0 || rot_dim < 0)
    return fail(MTP_ERR_SHAPE, "bad norm/rotation sizes");
  if (rot_dim % 2 != 0 || rot_dim > D)
    return fail(MTP_ERR_SHAPE, "rotated size %lld is odd or above the head size %lld", (long long)rot_dim,
                (long long)D);
  if (paged && (page_size <= 0 || num_pages < 0 || table_stride < 0 || page_size > INT32_MAX ||
                table_stride > INT32_MAX))
    return fail(MTP_ERR_SHAPE, "bad page sizes");
  if (!valid_dtype(dtype) || dtype == MTP_DTYPE_E4M3) return fail(MTP_ERR_DTYPE, "unsupported dtype %d", dtype);
  if ((q_weight && (!valid_dtype(q_weight_dtype) || q_weight_dtype == MTP_DTYPE_E4M3)) ||
      (k_weight && (!valid_dtype(k_weight_dtype) || k_weight_dtype == MTP_DTYPE_E4M3)))
    return fail(MTP_ERR_DTYPE, "unsupported norm weight dtypes %d, %d", q_weight_dtype, k_weight_dtype);
  // sizes before any sum or product of them, which would wrap
  if (B > INT32_MAX / 2 || S > INT32_MAX / 2 || Hq > INT32_MAX / 2 || Hkv > INT32_MAX / 2 || D > INT32_MAX / 2)
    return fail(MTP_ERR_SHAPE, "too many rows");
  if (B * S == 0 || Hq + Hkv == 0) return MTP_OK;
  if ((Hq > 0 && (!q || !q_out)) || (Hkv > 0 && !k) || (rot_dim > 0 && (!cos || !sin)))
    return fail(MTP_ERR_ARG, "null tensor pointer");
  if (!paged && ((Hkv > 0 && !k_out) || !positions)) return fail(MTP_ERR_ARG, "null tensor pointer");
  if (paged && (!k_pages || !v_pages || !start || (Hkv > 0 && !v))) return fail(MTP_ERR_ARG, "null tensor pointer");
  const int64_t heads = Hq + (paged ? 2 : 1) * Hkv;
  if (heads > INT32_MAX / 2 || (double)B * S * heads > 8e9) return fail(MTP_ERR_SHAPE, "too many rows");
  rope::Args a{};
  const void* x[3] = {q, k, v};
  const int64_t* st[3] = {g.q_stride, g.k_stride, g.v_stride};
  for (int i = 0; i < 3; ++i) {
    a.x[i] = x[i];
    a.sb[i] = st[i][0];
    a.ss[i] = st[i][1];
    a.sh[i] = st[i][2];
  }
  a.positions = positions;
  a.cos = cos;
  a.sin = sin;
  a.max_pos = max_pos;
  a.half = (int)(rot_dim / 2);
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.w_dtype[0] = q_weight_dtype;
  a.w_dtype[1] = k_weight_dtype;
  a.eps = (float)g.eps;
  a.normalise = g.normalise != 0;
  a.interleaved = g.interleaved != 0;
  a.q_out = q_out;
  a.k_out = paged ? nullptr : k_out;
  a.pages[0] = k_pages;
  a.pages[1] = v_pages;
  a.page_table = page_table;
  a.table_stride = table_stride;
  a.num_pages = num_pages;
  a.page_size = (int)page_size;
  a.start = paged ? start : nullptr;
  a.count = g.count;
  a.B = (int)B;
  a.S = (int)S;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.D = (int)D;
  a.dtype = dtype;
  const int e16 = 16 / dtype_bytes(dtype);  // elements in 16 bytes
  bool vec = D % 8 == 0 && D <= 256 && (a.interleaved ? a.half % 4 == 0 : a.half % 8 == 0) && aligned16(cos) &&
             aligned16(sin) && aligned16(q_out) && aligned16(a.k_out);
  for (int i = 0; i < (paged ? 3 : 2); ++i) {
    vec &= aligned16(x[i]);
    for (int d = 0; d < 3; ++d) vec &= st[i][d] % e16 == 0;
  }
  if (paged) vec &= aligned16(k_pages) && aligned16(v_pages);
  int dev;
  if (int r = current_device(&dev)) return r;
  const cudaStream_t s = as_stream(g.stream);
  if (!vec) {
    const int64_t rows = B * S * heads, blocks = (rows + rope::kThreads / 32 - 1) / (rope::kThreads / 32);
    if (blocks > INT32_MAX) return fail(MTP_ERR_SHAPE, "too many rows");
    rope::qk_norm_rope_any_kernel<<<(unsigned)blocks, rope::kThreads, 0, s>>>(a);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
  }
  for (int i = 0; i < 2; ++i) a.w_vec[i] = a.w[i] && a.w_dtype[i] == dtype && aligned16(a.w[i]);
  const int lph = D <= 64 ? 4 : (D <= 128 ? 8 : 16);
  const int groups = rope::kThreads / lph, sms = sm_count(dev);
  // As many tokens to a block as bring the call down to one round of two blocks
  // per SM (a group's set-up then serves more heads), 16 at most: calls of up to
  // 32 tokens per SM take one round, prompts several; where one token each leaves
  // SMs without a block, its heads go over several blocks.
  a.tokens = 1;
  while (a.tokens < 16 && (B * S + a.tokens - 1) / a.tokens > 2 * sms) a.tokens *= 2;
  const int64_t gx = (B * S + a.tokens - 1) / a.tokens;
  const int64_t most = (heads + groups / a.tokens - 1) / (groups / a.tokens);
  int64_t gy = (2 * sms + gx - 1) / gx;
  gy = gy < 1 ? 1 : (gy > most ? most : gy);
  if (gx > INT32_MAX || gy > 65535) return fail(MTP_ERR_SHAPE, "too many rows");
  if (dtype == MTP_DTYPE_F32) return launch_rope_vec<float>(a, lph, (unsigned)gx, (unsigned)gy, s);
  if (dtype == MTP_DTYPE_BF16) return launch_rope_vec<__nv_bfloat16>(a, lph, (unsigned)gx, (unsigned)gy, s);
  return launch_rope_vec<__half>(a, lph, (unsigned)gx, (unsigned)gy, s);
}

size_t mtp_paged_window_attention_workspace(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                                            int64_t max_keys, int64_t window, int64_t sinks, int dtype,
                                            int with_weights) {
  if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_keys < 0 || Hq % Hkv != 0) return 256;
  return window_plan(B, S, Hq, Hkv, D, max_keys, window, sinks, dtype, true, with_weights != 0).total();
}

int mtp_paged_window_attention(const mtp_paged_window_attention_args* args) {
  MTP_NVTX("mtp_paged_window_attention");
  if (!args) return fail(MTP_ERR_ARG, "null arguments");
  const mtp_paged_window_attention_args& g = *args;
  const int64_t B = g.B, S = g.S, Hq = g.Hq, Hkv = g.Hkv, D = g.D, num_pages = g.num_pages, page_size = g.page_size;
  const int64_t table_stride = g.table_stride, window = g.window, sinks = g.sinks, weight_ld = g.weight_ld;
  const int dtype = code(g.dtype);
  const void *q = g.q, *k_pages = g.k_pages, *v_pages = g.v_pages;
  void *out = g.out, *workspace = g.workspace;
  const int32_t *page_table = g.page_table, *seq_lens = g.seq_lens, *q_lens = g.q_lens;
  float* key_weights = g.key_weights;
  const float scale = (float)g.scale;
  const size_t workspace_bytes = g.workspace_bytes > 0 ? (size_t)g.workspace_bytes : 0;
  const cudaStream_t s = as_stream(g.stream);
  if (B < 0 || S < 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || page_size <= 0 || num_pages < 0 || table_stride < 0 ||
      window < 0 || sinks < 0)
    return fail(MTP_ERR_SHAPE, "bad window attention sizes");
  if (Hq % Hkv != 0) return fail(MTP_ERR_SHAPE, "Hq=%lld not a multiple of Hkv=%lld", (long long)Hq, (long long)Hkv);
  if (D > 256) return fail(MTP_ERR_SHAPE, "head_dim %lld > 256", (long long)D);
  if (key_weights && (S != 1 || weight_ld < table_stride))
    return fail(MTP_ERR_SHAPE, "key weights need one query row per sequence and rows of the page table's width");
  if (!valid_dtype(dtype) || dtype == MTP_DTYPE_E4M3) return fail(MTP_ERR_DTYPE, "unsupported dtype %d", dtype);
  if (B == 0 || S == 0) return MTP_OK;
  if (!q || !out || !seq_lens || (table_stride > 0 && (!page_table || !k_pages || !v_pages)))
    return fail(MTP_ERR_ARG, "null tensor pointer");
  if (!pool_fits(num_pages, B, Hkv, page_size)) return fail(MTP_ERR_SHAPE, "the pool has 2^31 rows or more");
  if ((double)B * S * (Hq + 16.0 * Hkv) > 2147483647.0 || table_stride > kNoWindow || num_pages > INT32_MAX ||
      page_size > INT32_MAX)
    return fail(MTP_ERR_SHAPE, "too many query rows or positions");
  // the tiles fold a positive scale into the exponent
  const bool aligned = aligned16(q) && aligned16(out) && aligned16(k_pages) && aligned16(v_pages) && scale > 0.f;
  const WindowPlan p =
      window_plan(B, S, Hq, Hkv, D, table_stride, window, sinks, dtype, aligned, key_weights != nullptr);
  if (!workspace || workspace_bytes < p.total() || !aligned16(workspace))
    return fail(MTP_ERR_WORKSPACE, "workspace of %zu bytes, 16-byte aligned, needed", p.total());
  split::Args a{};
  a.q = q;
  a.out = out;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.page_table = page_table;
  a.table_stride = table_stride;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.seq_lens = seq_lens;
  a.q_lens = q_lens;
  a.B = (int)B;
  a.S = (int)S;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.D = (int)D;
  a.dtype = dtype;
  a.window = p.window;
  a.sinks = p.sinks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.row_tiles = p.row_tiles;
  a.max_warps = p.max_warps;
  a.min_blocks = p.min_blocks;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float*>(ws + p.part_o);
  if (key_weights) {
    a.scores = reinterpret_cast<float*>(ws + p.part_o + p.part_ml);
    a.score_ld = p.score_ld;
    a.row_ml = reinterpret_cast<float*>(ws + p.part_o + p.part_ml + p.scores);
    a.key_weights = key_weights;
    a.weight_ld = weight_ld;
  }
  if (p.path == kPathTensor) return launch_prompt(a, p, s);
  if (p.path == kPathSplit) {
    if (int st = dtype == MTP_DTYPE_BF16 ? launch_split_t<__nv_bfloat16>(a, p.dp, s)
                                         : launch_split_t<__half>(a, p.dp, s))
      return st;
  } else {
    split::split_any_kernel<<<(unsigned)(B * S * Hq), split::kAnyWarps * 32, 0, s>>>(a);
    MTP_LAUNCH_CHECK();
  }
  if (key_weights && p.score_ld > 0) {
    const int64_t per_unit = (p.score_ld + 255) / 256;
    return launch_dependent(split::split_key_weights_kernel, (unsigned)(B * Hkv),
                            (unsigned)(per_unit < 65535 ? per_unit : 65535), 256, s, a);
  }
  return MTP_OK;
}

size_t mtp_paged_kv_evict_workspace(int64_t B, int64_t H, int64_t budget) {
  if (B <= 0 || H <= 0 || budget <= 0) return 256;
  return align256((size_t)B * H * budget * 8) + 256;
}

int mtp_paged_kv_evict(const mtp_paged_kv_evict_args* args) {
  MTP_NVTX("mtp_paged_kv_evict");
  if (!args) return fail(MTP_ERR_ARG, "null arguments");
  const mtp_paged_kv_evict_args& g = *args;
  const int64_t B = g.B, H = g.H, D = g.D, budget = g.budget, sinks = g.sinks, recent = g.recent;
  const int64_t table_stride = g.table_stride, num_pages = g.num_pages, page_size = g.page_size;
  const int64_t weight_ld = g.weight_ld;
  const int dtype = code(g.dtype);
  void *k_pages = g.k_pages, *v_pages = g.v_pages, *workspace = g.workspace;
  const int32_t *page_table = g.page_table, *seq_lens = g.seq_lens;
  float* key_weights = g.key_weights;
  int32_t *kept = g.kept, *new_lens = g.new_lens;
  const size_t workspace_bytes = g.workspace_bytes > 0 ? (size_t)g.workspace_bytes : 0;
  const cudaStream_t s = as_stream(g.stream);
  if (B < 0 || H <= 0 || D <= 0 || page_size <= 0 || num_pages < 0 || table_stride < 0 || weight_ld < 0 ||
      budget < 0 || sinks < 0 || recent < 0)
    return fail(MTP_ERR_SHAPE, "bad eviction sizes");
  if (sinks > budget || recent > budget - sinks)
    return fail(MTP_ERR_SHAPE, "sinks %lld and recent %lld do not fit the budget of %lld", (long long)sinks,
                (long long)recent, (long long)budget);
  if (!valid_dtype(dtype) || dtype == MTP_DTYPE_E4M3) return fail(MTP_ERR_DTYPE, "unsupported dtype %d", dtype);
  if (B == 0) return MTP_OK;
  if (!seq_lens || !new_lens || (budget > 0 && !kept) ||
      (table_stride > 0 && weight_ld > 0 && (!k_pages || !v_pages || !page_table || !key_weights)))
    return fail(MTP_ERR_ARG, "null tensor pointer");
  if (!pool_fits(num_pages, B, H, page_size)) return fail(MTP_ERR_SHAPE, "the pool has 2^31 rows or more");
  if (table_stride > INT32_MAX || budget > INT32_MAX / 2 || (double)B * H * D * 2 > 2147483647.0)
    return fail(MTP_ERR_SHAPE, "too many positions or heads");
  if (!workspace || workspace_bytes < mtp_paged_kv_evict_workspace(B, H, budget) || !aligned16(workspace))
    return fail(MTP_ERR_WORKSPACE, "workspace of %zu bytes, 16-byte aligned, needed",
                mtp_paged_kv_evict_workspace(B, H, budget));
  evict::Args a{};
  a.pages[0] = k_pages;
  a.pages[1] = v_pages;
  a.page_table = page_table;
  a.table_stride = table_stride;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.seq_lens = seq_lens;
  a.weights = key_weights;
  a.weight_ld = weight_ld;
  a.kept = kept;
  a.new_lens = new_lens;
  a.rows = static_cast<int2*>(workspace);
  a.B = (int)B;
  a.H = (int)H;
  a.D = (int)D;
  a.budget = (int)budget;
  a.sinks = (int)sinks;
  a.recent = (int)recent;
  int dev;
  if (int st = current_device(&dev)) return st;
  evict::evict_select_kernel<<<(unsigned)(B * H), evict::kThreads, 0, s>>>(a);
  MTP_LAUNCH_CHECK();
  if (budget == 0 || table_stride <= budget || weight_ld <= budget) return MTP_OK;  // no sequence is longer
  const int row_bytes = (int)D * dtype_bytes(dtype);
  const bool wide = row_bytes % 16 == 0 && aligned16(k_pages) && aligned16(v_pages);
  const int word = wide ? 16 : dtype_bytes(dtype);
  const int words = row_bytes / word;
  // 128 bytes of a row to a block, or 32 where that leaves SMs without one
  int lanes = 8;
  while (words % lanes != 0) lanes >>= 1;
  if (wide)
    while (lanes > 2 && B * H * 2 * (words / lanes) < 2 * sm_count(dev)) lanes >>= 1;
  if (word == 16) return launch_move<uint4>(a, words, lanes, s);
  if (word == 4) return launch_move<uint32_t>(a, words, lanes, s);
  return launch_move<uint16_t>(a, words, lanes, s);
}

}  // extern "C"
