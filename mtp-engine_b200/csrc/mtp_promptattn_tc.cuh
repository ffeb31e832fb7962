// mtp_promptattn_tc.cuh -- causal attention of many new tokens over a paged
// cache (prompts, pieces of prompts) on the sm_100a tensor cores, with
// grouped-query heads, ragged lengths, a sliding window and first tokens that
// stay visible ("sinks").  The row and key sets are those of mtp_splitattn.cuh,
// which serves calls with few rows.
//
// An item is one (sequence, key head, pair of query tiles): a tile holds
// tpt = 128 / G positions x G heads (row r = position * G + head), so a
// 128-key chunk of K and V is read once for 256 rows.  Persistent: one block
// of 640 threads per SM walks over the items, the ones with the most keys
// first and every other round in reverse, which evens out causal lengths
// without a counter in memory.  Roles:
//   warps 0-15  softmax, eight warps to a tile: four for the first 64 keys of a
//               chunk and four for the last 64, one thread per row each.  Scores
//               from tensor memory, the row's maximum exchanged between the two
//               threads, lazy rescaling, P (16-bit) back over the scores, half of
//               the output each.  With one thread per row (128 scores in its
//               registers, two warps per SM sub-partition) the exponentials ran
//               at half the rate of the exp2 unit.
//   warps 16, 18  producers of Q and K, and of V: whole page slabs by TMA, or
//               token by token where a chunk's table is not page-granular or
//               where the chunk holds keys that no row of the call may see
//               (those are zero-filled: their slots may hold anything, and
//               0 * NaN is NaN).  Two warps because a page load takes one of
//               them 100 cycles and more, 32 loads a chunk with 16-token pages
//   warp 17     tcgen05.mma issuer
//   warp 19     of the first block: records lengths outside their range, once per launch
// All rings and barrier phases run on from item to item: the next item's keys
// are already on their way, and its first scores are computed, while the
// softmax warps write the last item's output.
//
// Chunks of an item: those that hold sinks, then those from the first row's
// window to the last row's position; a tile stops at its own last chunk.
//
// Bound: the two products of a chunk take 2 x 512 tensor cycles per tile
// (D = 128) and its 16384 exponentials 1024 cycles of the SM's exp2 units, so
// 2048 cycles per chunk for both tiles is the floor of either pipe.  Measured
// (B200, Hq 32, Hkv 8, D 128, bf16, 16-token pages, calls back to back): one
// causal prompt of 8192 tokens 577-583 us (950 TFLOP/s; tensor pipe 51 % and exp2
// unit 52 % of active cycles); two prompts of 2750 and 5501 tokens with a window
// of 1024 211-213 us; 512 tokens behind 32000 356 us, 26 of them the joining of
// pieces.  Page sizes below 8, or that neither divide 128 nor are multiples of it
// (24, 48), and tables that are not page-granular are gathered token by token, by
// one warp that waits for its copies before the next chunk: 2048 tokens 131 us
// instead of 55.
#pragma once

#include "mtp_attention_tc.cuh"
#include "mtp_splitattn.cuh"

namespace mtp {
namespace prompt {

using attn::kChunk;
constexpr int kThreads = 640;  // 96 registers each
constexpr int kSoftmaxWarps = 16;
constexpr int kWarpK = 16, kWarpMma = 17, kWarpV = 18, kWarpCheck = 19;
constexpr int kHalfBytes = 128 * 128;  // 128 rows x 64 dims
constexpr int tile_bytes(int dp) { return dp / 64 * kHalfBytes; }
constexpr int num_buf(int dp) { return dp == 128 ? 4 : 8; }  // 128 KB of K and V in flight
constexpr int kExchangeBytes = 2 * 2 * 2 * 128 * 4;           // [turn][tile][half of the keys][row]
constexpr int smem_bytes(int dp) {
  return 2 * tile_bytes(dp) + num_buf(dp) * tile_bytes(dp) + kExchangeBytes + 256 + 1024;
}
static_assert(smem_bytes(128) <= 227 * 1024 && smem_bytes(64) <= 227 * 1024, "shared memory per CTA");

struct Params {
  const int32_t* page_table;
  int64_t table_stride;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const int32_t* seq_lens;
  const int32_t* q_lens;
  void* out;      // [B, S, Hq, D]
  float* part_o;  // [items][256][D] (splits > 1)
  float* part_ml; // [items][256][2]
  int B, S, Hq, Hkv, G, D, ps, num_pages;
  int window, sinks;
  int slab;      // rows of a TMA page load (0: always token by token)
  int tpt;       // positions per tile
  int pairs;     // tile pairs per sequence
  int splits;    // pieces of a pair's chunk list
  int items;     // B * Hkv * pairs * splits
  int table_vec; // page-table rows 16-byte aligned
  float scale_log2;
};

// One item: its rows and the chunks it goes over.
struct Item {
  int b, kvh, s0;  // first position (row of the call) of the pair
  int len, n;      // the sequence
  int call_lo;     // first key that some row's window reaches
  int ns, c_lo;    // chunks 0 .. ns-1 (sinks), then c_lo, c_lo + 1, ...
  int i0;          // this item's part of the list: [i0, i0 + max(n_it))
  int n_it[2];     // chunks of tile 0 and 1
  __device__ __forceinline__ int chunk(int i) const { return i0 + i < ns ? i0 + i : c_lo + (i0 + i - ns); }
  __device__ __forceinline__ int count() const { return max(n_it[0], n_it[1]); }
  // whether key j may be seen by some row of the call
  __device__ __forceinline__ bool used(const Params& p, int j) const {
    return j < len && (j >= call_lo || j < p.sinks);
  }
  // whether all keys of chunk c are used
  __device__ __forceinline__ bool whole(const Params& p, int c) const {
    const int first = c * kChunk;
    return first + kChunk <= len && (first >= call_lo || first + kChunk <= p.sinks);
  }
};

__device__ __forceinline__ Item item_of(const Params& p, int index) {
  Item it;
  const int split = index % p.splits;
  int u = index / p.splits;
  it.kvh = u % p.Hkv;
  u /= p.Hkv;
  it.b = u % p.B;
  it.s0 = (p.pairs - 1 - u / p.B) * 2 * p.tpt;  // the last positions first
  const split::Seq seq = split::lengths(p.seq_lens, p.q_lens, p.table_stride, p.S, it.b);
  it.len = seq.len;
  it.n = seq.n;
  it.ns = it.c_lo = it.i0 = it.n_it[0] = it.n_it[1] = 0;
  it.call_lo = max(0, it.len - it.n - p.window + 1);
  if (it.s0 >= it.n) return it;
  const int past = it.len - it.n;
  const int lo = max(0, past + it.s0 - p.window + 1);
  it.ns = (min(p.sinks, lo) + kChunk - 1) / kChunk;
  it.c_lo = max(it.ns, lo / kChunk);
  const int last0 = past + min(it.s0 + p.tpt, it.n) - 1;
  const int e0 = it.ns + max(0, last0 / kChunk - it.c_lo + 1);
  int e1 = 0;
  if (it.s0 + p.tpt < it.n) {
    const int last1 = past + min(it.s0 + 2 * p.tpt, it.n) - 1;
    e1 = it.ns + max(0, last1 / kChunk - it.c_lo + 1);
  }
  const int total = max(e0, e1);
  it.i0 = (int)((int64_t)total * split / p.splits);
  const int i1 = (int)((int64_t)total * (split + 1) / p.splits);
  it.n_it[0] = max(0, min(i1, e0) - it.i0);
  it.n_it[1] = max(0, min(i1, e1) - it.i0);
  return it;
}

// Item of round r for this block; -1: none, and `more` says whether a later
// round may have one.
__device__ __forceinline__ int item_index(const Params& p, int r, bool* more) {
  const int64_t base = (int64_t)r * gridDim.x;
  *more = base < p.items;
  const int64_t i = base + ((r & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
  return i < p.items ? (int)i : -1;
}

// Visible keys [32 w, 32 w + 32) of chunk c for a row at position pos, as bits.
__device__ __forceinline__ uint32_t mask_word(int base, int pos, int lo, int sinks) {
  const int hi = pos - base, lw = lo - base, sb = sinks - base;
  const uint32_t below = hi < 0 ? 0u : (hi >= 31 ? 0xffffffffu : (2u << hi) - 1u);
  const uint32_t above = lw <= 0 ? 0xffffffffu : (lw >= 32 ? 0u : ~((1u << lw) - 1u));
  const uint32_t sink = sb <= 0 ? 0u : (sb >= 32 ? 0xffffffffu : (1u << sb) - 1u);
  return below & (above | sink);
}

// Pool rows of tokens tok0 + lane + 32 i (-1: not used, or a page id outside
// the pool, recorded): see attn::token_rows.
__device__ __forceinline__ void token_rows(const Params& p, const Item& it, int tok0, int lane, int (&rows)[4]) {
  const int32_t* table = p.page_table + (int64_t)it.b * p.table_stride;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int tok = tok0 + lane + 32 * i;
    rows[i] = -1;
    if (it.used(p, tok)) {
      const int64_t pg = resolve_page(__ldg(table + tok), p.num_pages);
      if (pg >= 0) rows[i] = (int)(((pg * p.B + it.b) * p.Hkv + it.kvh) * p.ps + tok % p.ps);
      else record_error(MTP_ERR_DEVICE);
    }
  }
}

// Starts the copies of 128 rows into one K or V buffer (layout as TMA's
// 128-byte swizzle leaves it); rows of -1 and dimensions past D are zero-filled.
template <int DP>
__device__ __forceinline__ void fill_tokens(uint8_t* dst, const uint8_t* pool, const int (&rows)[4], int lane, int D) {
  constexpr int kPieces = DP / 8, kPerCopy = 32 / kPieces;
  const int j = lane % kPieces, half = j >> 3, jj = j & 7, sub = lane / kPieces;
  const uint32_t base = smem_u32(dst) + half * kHalfBytes;
  const bool in = j * 8 < D;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
#pragma unroll
    for (int u = 0; u < 32 / kPerCopy; ++u) {
      const int i = 32 * q + kPerCopy * u + sub;
      const int row = __shfl_sync(0xffffffffu, rows[q], i & 31);
      const bool go = row >= 0 && in;
      const uint8_t* src = go ? pool + (int64_t)row * (D * 2) + j * 16 : pool;
      attn::cp_async16(base + i * 128 + ((jj ^ (i & 7)) << 4), src, go ? 16u : 0u);
    }
  }
}

// mbar_wait with its limit in clock cycles: reading the nanosecond timer on the
// way into a wait costs hundreds of cycles, which here sit between one tile's P
// and its next product.
constexpr long long kWaitLimitCycles = 4000000000ll;  // about 2 s

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*abort) return false;
    if (clock64() - t0 > kWaitLimitCycles) {
      *abort = 1;
      record_error(MTP_ERR_TIMEOUT);
      return false;
    }
  }
}

// In place of an exchanged value: a signalling NaN, which no arithmetic gives.
constexpr uint32_t kGone = 0x7fa5a5a5u;

// P of 16 scores: 2^(s * mul - m) packed as 16-bit pairs, with the running sums
// (of the unrounded values) in (ls0, ls1).  16 bits because the second product
// has V's type on both sides; its error is bounded as in mtp_splitattn.cuh.
template <int AB_FMT>
__device__ __forceinline__ void exp_pack16(const uint32_t (&s)[16], float mul, float m_use, float& ls0, float& ls1,
                                           uint32_t (&out)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float x0, x1;
    attn::ffma2(x0, x1, __uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1]), mul, mul, -m_use, -m_use);
    const float e0 = attn::ex2(x0), e1 = attn::ex2(x1);
    attn::add2(ls0, ls1, e0, e1);
    out[j] = attn::pack_bf16(e0, e1, AB_FMT == 1 ? MTP_DTYPE_BF16 : MTP_DTYPE_F16);
  }
}

// 32 lanes x 8 consecutive 32-bit columns <- 8 registers per thread
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// True in one lane of a converged warp.  Products, commits and page loads are
// issued as `if (elect_one()) { ... } __syncwarp();`: the branch tells the
// compiler that one lane is active, so operands go through uniform registers,
// and the other lanes wait behind it -- those registers belong to the whole
// warp, and a lane that ran ahead to the next load's address would change them
// under the instruction still to be issued.
__device__ __forceinline__ bool elect_one() {
  uint32_t lead;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(lead)
      :
      : "memory");
  return lead != 0;
}

// AB_FMT: 1 = bf16, 0 = f16; DP: 64 or 128, the head size of the tiles (64 <=
// D <= DP; the dimensions past D arrive as zeros)
template <int AB_FMT, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_attention_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                               const __grid_constant__ CUtensorMap tmV, Params p) {
  constexpr int kTileBytes = tile_bytes(DP), kNumBuf = num_buf(DP), kHalves = DP / 64;
  constexpr uint32_t IDESC_S = make_idesc(AB_FMT, 128, kChunk);        // Q (K-major) x K (K-major)
  constexpr uint32_t IDESC_PV = make_idesc(AB_FMT, 128, DP, 0u, 1u);  // P (K-major) x V (MN-major)

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sBuf = sQ + 2 * kTileBytes;
  float* sExchange = reinterpret_cast<float*>(sBuf + kNumBuf * kTileBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sExchange) + kExchangeBytes);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* buf_full = bars + 2;
  uint64_t* buf_empty = buf_full + kNumBuf;
  uint64_t* s_full = buf_empty + kNumBuf;  // [2]
  uint64_t* p_full = s_full + 2;           // [2 tiles][first 48 keys of each half, last 16]
  uint64_t* pv_done = p_full + 4;          // [2]
  uint64_t* drain = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 + 2 * kNumBuf + 2 + 4 + 2 + 1) * 8 + 8 <= 256, "barrier area");

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < kNumBuf; ++i) {
      mbar_init(&buf_full[i], 1);
      mbar_init(&buf_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[2 * t], 8);  // one arrival per softmax warp of the tile
      mbar_init(&p_full[2 * t + 1], 8);
      mbar_init(&pv_done[t], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kWarpMma) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const int ppc = p.slab > 0 ? kChunk / p.slab : 0;  // page slabs per chunk

  if (warp >= kSoftmaxWarps) {  // producer, MMA
    bool ok = true, more = true;
    if (warp == kWarpK || warp == kWarpV) {
      // -------------------------------------------------------------- producers (whole warps)
      const int kv = warp == kWarpV;
      const CUtensorMap* const map = kv ? &tmV : &tmK;
      const uint8_t* const pool = kv ? p.v_pool : p.k_pool;
      if (lane == 0) {
        if (kv == 0) tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(map);
      }
      int chunks = 0, queries = 0;  // chunks and Q loads so far
      // Lane l reads the page ids of tokens 4 l .. 4 l + 3 of a chunk, one chunk
      // ahead.  A chunk is page-granular if all tokens of every slab lie in the
      // page of the slab's first one.
      const int per_slab = p.slab > 0 ? p.slab / 4 : 1;  // lanes of a slab
      int id[4];
      auto read_ids = [&](const Item& it, int c) {
        id[0] = id[1] = id[2] = id[3] = INT32_MIN;
        if (p.slab > 0 && it.whole(p, c)) {  // then all 128 columns are inside the table
          const int32_t* src = p.page_table + (int64_t)it.b * p.table_stride + c * kChunk + lane * 4;
          if (p.table_vec) {
            const int4 e = __ldg(reinterpret_cast<const int4*>(src));
            id[0] = e.x, id[1] = e.y, id[2] = e.z, id[3] = e.w;
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) id[k] = __ldg(src + k);
          }
        }
      };
      for (int r = 0; ok; ++r) {
        const int index = item_index(p, r, &more);
        if (!more) break;
        if (index < 0) continue;
        const Item it = item_of(p, index);
        const int n_it = it.count();
        if (n_it == 0) continue;
        read_ids(it, it.chunk(0));
        if (kv == 0) {
          bool got = true;
          if (lane == 0) {
            got = mbar_wait(q_empty, (queries & 1) ^ 1u, abort_flag);
            if (got) {
              const int tiles = it.s0 + p.tpt < it.n ? 2 : 1;
              mbar_expect_tx(q_full, tiles * kHalves * p.tpt * p.G * 128);
              for (int t = 0; t < tiles; ++t)
                for (int h = 0; h < kHalves; ++h)
                  tma_load_4d(sQ + t * kTileBytes + h * kHalfBytes, &tmQ, h * 64, it.kvh * p.G, it.s0 + t * p.tpt,
                              it.b, q_full);
            }
          }
          if (!__shfl_sync(0xffffffffu, got, 0)) break;
          ++queries;
        }
        for (int i = 0; i < n_it && ok; ++i, ++chunks) {
          const int c = it.chunk(i);
          const int page = (int)resolve_page(id[0], p.num_pages);  // -1 where nothing was read
          bool gran = page >= 0;
#pragma unroll
          for (int k = 1; k < 4; ++k) gran &= (int)resolve_page(id[k], p.num_pages) == page;
          const int head = __shfl_sync(0xffffffffu, page, lane / per_slab * per_slab);
          const bool per_token = !__all_sync(0xffffffffu, gran && head == page);
          const int pg = __shfl_sync(0xffffffffu, page, (lane * per_slab) & 31);  // page of this lane's slab
          if (i + 1 < n_it) read_ids(it, it.chunk(i + 1));
          bool got = true;
          const int buf = 2 * (chunks % (kNumBuf / 2)) + kv;
          if (lane == 0) {
            got = mbar_wait(&buf_empty[buf], ((chunks / (kNumBuf / 2)) & 1) ^ 1u, abort_flag);
            if (got && !per_token) mbar_expect_tx(&buf_full[buf], kTileBytes);
          }
          if (!__shfl_sync(0xffffffffu, got, 0)) {
            ok = false;
            break;
          }
          __syncwarp();
          uint8_t* dst = sBuf + buf * kTileBytes;
          if (per_token) {
            int rows[4];
            token_rows(p, it, c * kChunk, lane, rows);
            fill_tokens<DP>(dst, pool, rows, lane, p.D);
            attn::cp_async_wait_all();  // each lane waits for its copies, fences them for the tensor cores
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&buf_full[buf]);
          } else {
            // one load after the other from a converged warp: coordinates and
            // addresses in uniform registers, as for the products below
            const int mine = ((pg * p.B + it.b) * p.Hkv + it.kvh) * p.ps + (c * kChunk + lane * p.slab) % p.ps;
#pragma unroll 1
            for (int u = 0; u < ppc; ++u) {
              const int row = __shfl_sync(0xffffffffu, mine, u);
              if (elect_one()) {
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
                  tma_load_2d(dst + h * kHalfBytes + u * p.slab * 128, map, h * 64, row, &buf_full[buf]);
              }
              __syncwarp();
            }
          }
        }
      }
      // After an abort too: no copy of this warp may land after the block's end.
      // Page loads whose chunk nobody waits for any more are among the last
      // kNumBuf / 2; each wait has its own limit and goes on although others gave up.
      attn::cp_async_wait_all();
      if (lane == 0) {
        constexpr int kRing = kNumBuf / 2;
        for (int j = max(0, chunks - kRing); j < chunks; ++j)
          mbar_wait(&buf_full[2 * (j % kRing) + kv], (j / kRing) & 1, abort_flag, /*honour_abort=*/false);
        if (queries > 0) mbar_wait(q_full, (queries - 1) & 1, abort_flag, /*honour_abort=*/false);
      }
      __syncwarp();
    } else if (warp == kWarpMma) {
      // -------------------------------------------------------------- MMA issuer
      // The whole warp walks the loop and an elected lane issues: with every
      // value the same in all lanes, descriptors and addresses stay in uniform
      // registers (issued from a one-lane branch a product took ~90 cycles of
      // this warp, above the 64 it takes the tensor pipe).
      const uint64_t q_desc = sw128_kmajor_desc(smem_u32(sQ));
      const uint64_t k_desc = sw128_kmajor_desc(smem_u32(sBuf));
      const uint64_t v_desc = sw128_mnmajor_desc(smem_u32(sBuf), kHalfBytes);
      int buf = 0;                    // ring buffer of the current K
      uint32_t phase = 0;             // and its parity
      uint32_t q_phase = 0;
      uint32_t p_phase[2] = {0, 0};  // parity of each tile's next P
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        const bool got = __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag));
        tc_fence_after();
        return got;
      };
      auto after = [&](int k, int n) { return k + n >= kNumBuf ? k + n - kNumBuf : k + n; };
      // S of tile t; free: whether K's buffer and q: whether Q's are released behind it
      auto issue_s = [&](int t, int k, bool free, bool q_free) {
        const uint32_t d = tmem_base + (uint32_t)(t * 128);
        const uint64_t qa = q_desc + (uint64_t)(t * (kTileBytes >> 4)), ka = k_desc + (uint64_t)(k * (kTileBytes >> 4));
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < DP / 16; ++x) {
            const uint32_t off = ((x >> 2) * kHalfBytes + (x & 3) * 32) >> 4;
            umma_f16(d, qa + off, ka + off, IDESC_S, x > 0);
          }
          umma_commit(&s_full[t]);
          if (free) umma_commit(&buf_empty[k]);
          if (q_free) umma_commit(q_empty);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) umma_commit(bar);
        __syncwarp();
      };
      // O_t += P_t V for the first 48 keys of each half of the chunk (part 0), or their last 16
      auto issue_pv = [&](int t, int k, int part, bool acc, bool last, bool free) {
        const uint32_t d = tmem_base + (uint32_t)(256 + t * 128);
        const uint32_t pa = tmem_base + (uint32_t)(t * 128);
        const uint64_t va = v_desc + (uint64_t)(k * (kTileBytes >> 4));
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (((x & 3) == 3) == (part == 1))
              umma_f16_ts(d, pa + (x >> 2) * 64 + (x & 3) * 8, va + (uint64_t)((x * 16 * 128) >> 4), IDESC_PV,
                          (acc || x > 0) ? 1u : 0u);
          if (last) umma_commit(&pv_done[t]);
          if (free) umma_commit(&buf_empty[k]);
        }
        __syncwarp();
      };
      for (int r = 0; ok; ++r) {
        const int index = item_index(p, r, &more);
        if (!more) break;
        if (index < 0) continue;
        const Item it = item_of(p, index);
        const int n0 = __shfl_sync(0xffffffffu, it.n_it[0], 0), n1 = __shfl_sync(0xffffffffu, it.n_it[1], 0);
        const int n_it = max(n0, n1);
        if (n_it == 0) continue;
        if (!(ok = wait(q_full, q_phase))) break;
        q_phase ^= 1u;
        if (!(ok = wait(&buf_full[buf], phase))) break;
        if (n0 > 0) issue_s(0, buf, n1 == 0, n1 == 0 && n_it == 1);
        if (n1 > 0) issue_s(1, buf, true, n_it == 1);
#pragma unroll 1
        for (int i = 0; i < n_it; ++i) {
          const int v = after(buf, 1), next = after(buf, 2);
          const uint32_t v_phase = phase ^ (v < buf ? 1u : 0u), next_phase = phase ^ (next < buf ? 1u : 0u);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int n_t = t == 0 ? n0 : n1;
            if (i < n_t) {
              if (!(ok = wait(&p_full[2 * t], p_phase[t]))) break;
              if (t == 0 || i >= n0) {  // the first tile of the chunk
                if (!(ok = wait(&buf_full[v], v_phase))) break;
              }
              issue_pv(t, v, 0, i > 0, false, false);
              if (!(ok = wait(&p_full[2 * t + 1], p_phase[t]))) break;
              issue_pv(t, v, 1, true, i + 1 == n_t, t == 1 || i >= n1);  // V is free behind the chunk's last tile
              p_phase[t] ^= 1u;
              if (i + 1 < n_t) {
                if (t == 0 || i + 1 >= n0) {
                  if (!(ok = wait(&buf_full[next], next_phase))) break;
                }
                const bool last_tile = t == 1 || i + 1 >= n1;
                issue_s(t, next, last_tile, last_tile && i + 2 == n_it);
              }
            }
          }
          if (!ok) break;
          buf = next;
          phase = next_phase;
        }
      }
      commit(drain);
      if (lane == 0) mbar_wait(drain, 0, abort_flag, /*honour_abort=*/false);
      __syncwarp();
    } else if (warp == kWarpCheck && blockIdx.x == 0) {
      for (int b = lane; b < p.B; b += 32) split::lengths(p.seq_lens, p.q_lens, p.table_stride, p.S, b, true);
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const int t = warp / 8, half = warp / 4 % 2;  // tile, half of the chunk's keys
    const int q = warp & 3;
    const int row = q * 32 + lane;  // row within the tile == TMEM lane
    const int row_s = row / p.G, g = row % p.G;
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_off + (uint32_t)(t * 128 + half * 64);  // this half's scores
    const uint32_t p_addr = s_addr;  // and its P, over the first 32 of its 64 columns
    const uint32_t o_addr = tmem_base + lane_off + (uint32_t)(256 + t * 128 + half * (DP / 2));  // half of the output
    // The two warps that share 32 rows tell each other a value per row.  They
    // meet at a named barrier, which knows no limit, so they go through the same
    // number of exchanges whatever their waits come to: a warp whose wait ran
    // out still meets its partner once, with kGone in place of a value, and both
    // leave behind that exchange.
    float* const ex_mine = sExchange + (t * 2 + half) * 128 + row;
    float* const ex_other = sExchange + (t * 2 + (half ^ 1)) * 128 + row;
    int turn = 0;
    auto exchange = [&](float v) -> float {
      ex_mine[turn] = v;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + t * 4 + q) : "memory");
      const float o = ex_other[turn];
      turn ^= 2 * 2 * 128;  // the other set of slots next time: this one may still be being read
      return o;
    };
    int done = 0, finished = 0;  // chunks and items of this tile so far
    bool ok = true, more = true;
    for (int r = 0; ok; ++r) {
      const int index = item_index(p, r, &more);
      if (!more) break;
      if (index < 0) continue;
      const Item it = item_of(p, index);
      const int s = it.s0 + t * p.tpt + row_s;  // row of the call
      const bool in_tile = row_s < p.tpt && s < p.S;
      const bool row_ok = in_tile && s < it.n;
      const int pos = row_ok ? it.len - it.n + s : -1;
      const int lo = pos - p.window + 1;
      const int n_it = t == 0 ? it.n_it[0] : it.n_it[1];
      float m_run = -INFINITY, l_run = 0.f;
      for (int i = 0; i < n_it; ++i) {
        const int first = it.chunk(i) * kChunk + half * 64;
        if (!__all_sync(0xffffffffu, wait_bar(&s_full[t], (done + i) & 1, abort_flag))) {
          exchange(__uint_as_float(kGone));
          ok = false;
          break;
        }
        tc_fence_after();
        const bool no_masked = first + 63 <= pos && (first >= lo || first + 64 <= p.sinks);
        // four blocks of 16 scores and, later, of 8 registers of P: larger
        // blocks of consecutive registers cost spills
        uint32_t sc[4][16];
#pragma unroll
        for (int k = 0; k < 4; ++k) tmem_ld16(s_addr + 16 * k, sc[k]);
        tmem_wait_ld();
        if (!no_masked) {
          const uint32_t mw[2] = {mask_word(first, pos, lo, p.sinks), mask_word(first + 32, pos, lo, p.sinks)};
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (!((mw[j >> 5] >> (j & 31)) & 1u)) sc[j >> 4][j & 15] = 0xff800000u;  // -inf
        }
        float m4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) m4[k] = fmaxf(__uint_as_float(sc[k][0]), __uint_as_float(sc[k][1]));
#pragma unroll
        for (int j = 2; j < 16; j += 2)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            m4[k] = attn::fmax3(m4[k], __uint_as_float(sc[k][j]), __uint_as_float(sc[k][j + 1]));
        const float mx = p.scale_log2 * fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        const float other = exchange(mx);
        if (__any_sync(0xffffffffu, __float_as_uint(other) == kGone)) {
          ok = false;
          break;
        }
        // both halves go by the greater maximum
        const float m_new = attn::fmax3(m_run, mx, other);
        if (i > 0) {
          // The scores of this chunk were issued after the last chunk's P V, so
          // O and P's columns are free here without another wait.
          const bool need = m_new > m_run + attn::kRescaleThreshold;
          if (__any_sync(0xffffffffu, need)) {
            const float alpha = need ? attn::ex2(m_run - m_new) : 1.0f;
#pragma unroll 1
            for (int j = 0; j < DP / 32; ++j) {
              uint32_t o[16];
              tmem_ld16(o_addr + j * 16, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st16(o_addr + j * 16, o);
            }
            tmem_wait_st();
            if (need) {
              l_run *= alpha;
              m_run = m_new;
            }
          }
        } else {
          m_run = m_new;
        }
        const float m_use = (m_run == -INFINITY) ? 0.f : m_run;
        // P in two parts, 48 keys and 16: only a quarter of P V is left to do
        // once the last part is there
        float ls0 = 0.f, ls1 = 0.f;
        {
          uint32_t pk[8];
          exp_pack16<AB_FMT>(sc[0], p.scale_log2, m_use, ls0, ls1, pk);
          tmem_st8(p_addr, pk);
        }
        {
          uint32_t pk[8];
          exp_pack16<AB_FMT>(sc[1], p.scale_log2, m_use, ls0, ls1, pk);
          tmem_st8(p_addr + 8, pk);
        }
        {
          uint32_t pk[8];
          exp_pack16<AB_FMT>(sc[2], p.scale_log2, m_use, ls0, ls1, pk);
          tmem_st8(p_addr + 16, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t]);
        {
          uint32_t pk[8];
          exp_pack16<AB_FMT>(sc[3], p.scale_log2, m_use, ls0, ls1, pk);
          tmem_st8(p_addr + 24, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + 1]);
        l_run += ls0 + ls1;
      }
      if (!ok) break;
      done += n_it;
      if (n_it > 0) {
        l_run += exchange(l_run);
        const bool got = __all_sync(0xffffffffu, wait_bar(&pv_done[t], finished & 1, abort_flag));
        ++finished;
        tc_fence_after();
        if (!got) continue;  // no output; on to the next item's first exchange
      }
      constexpr int kCols = DP / 2;  // this half's columns of the output
      const int col0 = half * kCols;
      if (p.splits == 1) {
        const float inv = l_run > 0.f ? 1.0f / l_run : 0.f;
        uint8_t* orow = static_cast<uint8_t*>(p.out) +
                        ((((int64_t)it.b * p.S + s) * p.Hq + (int64_t)it.kvh * p.G + g) * p.D + col0) * 2;
#pragma unroll 1
        for (int j = 0; j < kCols / 32; ++j) {
          uint32_t o[32];
          if (n_it > 0) {
            tmem_ld32(o_addr + j * 32, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0u;
          }
          if (in_tile) {
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k)
              w[k] = row_ok ? attn::pack_bf16(__uint_as_float(o[2 * k]) * inv, __uint_as_float(o[2 * k + 1]) * inv,
                                              AB_FMT == 1 ? MTP_DTYPE_BF16 : MTP_DTYPE_F16)
                            : 0u;  // rows behind q_lens
            uint4* dst = reinterpret_cast<uint4*>(orow + j * 64);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (col0 + j * 32 + k * 8 < p.D)
                dst[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
          }
        }
      } else if (n_it > 0 || row_ok) {
        const int64_t slot = (int64_t)index * 256 + t * 128 + row;
        float* po = p.part_o + slot * p.D + col0;
#pragma unroll 1
        for (int j = 0; j < (n_it > 0 ? kCols / 32 : 0); ++j) {
          uint32_t o[32];
          tmem_ld32(o_addr + j * 32, o);
          tmem_wait_ld();
          if (row_ok) {
            float4* dst = reinterpret_cast<float4*>(po + j * 32);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (col0 + j * 32 + k * 4 < p.D)
                dst[k] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                     __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
          }
        }
        if (row_ok && half == 0) {
          p.part_ml[slot * 2] = m_run;
          p.part_ml[slot * 2 + 1] = l_run;  // 0: no key of this piece is visible, and its output is not read
        }
      }
      // the next item's products overwrite O only after this warp's next arrival at p_full
      tc_fence_before();
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Joins the pieces of each row (splits > 1), in their order; zero for rows
// behind q_lens.  One warp per row of the call.
template <typename T>
__global__ void __launch_bounds__(256) prompt_merge_kernel(Params p) {
  const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (row >= (int64_t)p.B * p.S * p.Hq) return;
  const int h = (int)(row % p.Hq), s = (int)(row / p.Hq % p.S), b = (int)(row / p.Hq / p.S);
  const int kvh = h / p.G, g = h % p.G;
  const int pair = s / (2 * p.tpt), t = s / p.tpt % 2, r = (s % p.tpt) * p.G + g;
  const int64_t base = (((int64_t)(p.pairs - 1 - pair) * p.B + b) * p.Hkv + kvh) * p.splits;
  const int n = split::lengths(p.seq_lens, p.q_lens, p.table_stride, p.S, b).n;
  T* out = static_cast<T*>(p.out) + row * p.D;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, L = 0.f;
  const bool mine = lane * 4 < p.D;
  if (s < n) {
    float M = -INFINITY;
    for (int i = 0; i < p.splits; ++i) M = fmaxf(M, p.part_ml[((base + i) * 256 + t * 128 + r) * 2]);
#pragma unroll 4
    for (int i = 0; i < p.splits; ++i) {
      const int64_t slot = (base + i) * 256 + t * 128 + r;
      const float m = p.part_ml[slot * 2], l = p.part_ml[slot * 2 + 1];
      if (l == 0.f) continue;  // no key of this piece is visible to the row: its output may not be written
      // -inf with a sum is a NaN query's (a maximum passes NaN over, the sum holds it): 0 * NaN stays NaN
      const float w = m == -INFINITY ? 0.f : attn::ex2(m - M);
      L += w * l;
      if (mine) {
        const float4 v = *reinterpret_cast<const float4*>(p.part_o + slot * p.D + lane * 4);
        acc[0] += w * v.x;
        acc[1] += w * v.y;
        acc[2] += w * v.z;
        acc[3] += w * v.w;
      }
    }
  }
  const float inv = L > 0.f ? 1.0f / L : 0.f;
  if (mine)
    *reinterpret_cast<uint2*>(out + lane * 4) = make_uint2(split::Mma<T>::pack(acc[0] * inv, acc[1] * inv),
                                                           split::Mma<T>::pack(acc[2] * inv, acc[3] * inv));
}

}  // namespace prompt
}  // namespace mtp
