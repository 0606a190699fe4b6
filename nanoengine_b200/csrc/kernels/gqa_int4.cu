// Grouped-query paged attention over a key / value cache held in 4 bits (kv4.cuh): decode steps and short portions.
//
//   softmax(q k^T scale) v with k = (c - 8) s of 4-bit codes, a scale per 32 dims; causal, optionally the last `window` keys only
//
// Least traffic: D/2 + D/32 bytes a key row, 17/64 of bf16.  A unit of work is a tile of 64 keys (32 for heads of 256) for up to 16 (token, head of the
// group) rows of one sequence and KV head.  The units of the whole batch, laid end to end, are cut into equal shares, one per warp that fits the GPU:
// ragged contexts keep no SM waiting, whatever their number, and no warp waits for another.  A warp walks its share with a ring of bulk copies of its own.
// Where a share cuts a row tile, the pieces are written as 32-bit partial results, two places per warp, and a second kernel joins the pieces of every
// tile that a cut runs through.
//
// A key is unpacked once, in registers, straight into the fragments of mma.m16n8k16: a lane owns a contiguous quarter of a key row and an eighth of a value
// row; the dims of a step of the first product and the keys of a step of the second are permuted to match (query rows and probabilities follow).  Up to 16
// rows of queries are the 16 rows of a product.  Where a sequence has no more than 8, the products are transposed (S^T = K Q^T, O^T = V^T P^T): keys and value
// dims are the 16 rows, the same unpacked registers make half as many products, and the results take half the registers, so that a third CTA fits an SM.
// Portions with many rows per key run on the tensor-core prompt kernel over expanded pages instead.
//
// A masked nibble is a bf16 pair of subnormals c 2^-133 (16 c 2^-133 for the upper nibble of a byte), so that one fused multiply-add per pair gives
// (c - 8) s 2^-24, exactly; the 2^24 goes into the softmax scale and the last division.  Scores, maxima, sums and results are 32-bit.  Probabilities enter
// the second product as over bf16 pages: heads of 128 without a window as bf16 (2^-8), all others as two bf16 terms (2^-17, a second product on the same unpacked
// values); their sum is a column (row) of ones of the same products.  One term would be faster where two are taken (us of one / two: 60 x 3000 keys, 16 / 2 heads of
// 256: 39 / 41, four tokens: 85 / 98; 128 x 4096, 32 / 8 heads of 64: 74 / 83, 64 / 4: 54 / 65; 64 / 4 of 128, window 1000: 34 / 38), but a layer would lose
// bits with its cache, and its decode steps against its prompts.  Every byte stands for a finite value, so a masked key
// (probability 0) adds nothing whatever its page holds.
//
// Bound by the chain unpack, product, softmax of two (three) warps a scheduler, not by HBM: cycles of a warp for a tile of 64 keys and 16 rows: waiting for copies 290,
// scores 1460, maximum 290, values 1770, next copy 580; a product and the two pairs that feed it take 9.7 cycles of their pipes, of which none is full (matrix
// 32 %, integer 31 %, issue slots 41 %).  Measured (B200, calls in a graph, us, GB/s of 6530): 128 x 4096 keys, 64 / 4 heads of 128 (16 rows): 86, 3320;
// 32 / 8 heads (4 rows): 115, 4960; 2 x 131072 keys, 64 / 4: 50; 60 x 3000, 16 / 2 heads of 256: 41; 33 x 2504, four tokens, 32 / 8: 37; 1 x 1001: 10.  Slower: queries in shared memory, tiles of 32 keys, copies by cp.async, three CTAs per SM with 16 rows (they spill).  tcgen05 with the keys
// unpacked into tensor memory and the values into shared memory, three CTAs per SM, a warp of its own for copies and products: 116 where this one takes 89; the
// unpacked values cross shared memory twice, and barriers between unpacking, products and softmax leave the pipes idle.
#include "kv4.cuh"

namespace ne {

constexpr int kKernelI4 = 31;
constexpr int kI4Warps = 4, kI4Threads = 32 * kI4Warps, kI4Slots = 2;

struct I4Args {
  const __nv_bfloat16* q; long long q_ld;              // [T, Hq, D], rows q_ld apart
  const uint8_t* k; const uint8_t* v; int num_blocks, block_size;
  const int* block_tables; long long bt_ld; int bt_width;
  const int* cu_seqlens_q; const int* context_lens; int num_seqs;
  int T, Hq, Hkv, g, rows, tq, head_tiles, window, shares;   // rows of a row tile: tq tokens x min(g, rows) heads; head_tiles = ceil(g / rows)
  int max_tiles;                                       // places in cuts
  float scale_log2;
  __nv_bfloat16* out;                                  // [T, Hq, D]
  float* part; float* lse2;                            // [shares, 2, rows, D], [shares, 2, rows]
  int4* cuts;                                          // [1 + row tiles]: how many row tiles there are; what the join needs of each
};

template <int D, int R> struct I4Geo {                                  // R: rows of a row tile, 8 or 16
  static constexpr int keys = D == 256 ? 32 : 64;                       // of a tile
  static constexpr int slots = kI4Slots;                                // of a warp's ring (three: 43 us where two take 40 for 33 x 2504 keys, four tokens)
  static constexpr int ctas = D == 64 || (D == 128 && R == 8) ? 3 : 2;  // resident per SM
  static constexpr int row = D / 2, srow = D / 32;                      // bytes of a row's codes and scales
  static constexpr int codes = keys * row, half = codes + keys * srow, stage = 2 * half;
  static constexpr int words = D / 32;                                  // words of a key row a lane owns (a quarter of the row)
  static constexpr int vwords = D / 64;                                 // words of a value row a lane owns (an eighth)
  static constexpr int ks = D / 16;                                     // k steps of the first product
  static constexpr int nt = D / 8;                                      // column tiles of the second one
  static constexpr bool q_regs = D <= 128 || R == 8;                            // query fragments in registers, else in shared memory
  static constexpr int warp_bytes = slots * stage + (q_regs ? 0 : ks * 512);
  static constexpr int smem = kI4Warps * warp_bytes;
};

// ---- shares: the units of all sequences end to end ----
struct I4Seq { int q_beg, q_len, ctx, first, per_tile, tiles; };        // first: first tile of keys; per_tile: units of a (row tile, head)

template <int KEYS> __device__ __forceinline__ I4Seq i4_seq(const I4Args& a, int q_beg, int q_end, int ctx) {
  I4Seq s;
  s.q_beg = q_beg;
  s.q_len = max(0, q_end - q_beg);                                       // (as claimed: it says where the rows stand, also where some lie behind the last one of q)
  s.ctx = (int)max(0ll, min((long long)ctx, (long long)a.bt_width * a.block_size));
  const int first_key = a.window > 0 ? max(0, s.ctx - s.q_len - a.window + 1) : 0;
  s.first = first_key / KEYS;
  s.per_tile = max(1, (s.ctx + KEYS - 1) / KEYS - s.first);              // a tile that sees no key still writes its zeros
  s.tiles = (min(s.q_len, max(0, a.T - max(q_beg, 0))) + a.tq - 1) / a.tq;
  return s;
}
template <int KEYS> __device__ __forceinline__ I4Seq i4_load(const I4Args& a, int i) {
  return i4_seq<KEYS>(a, a.cu_seqlens_q[i], a.cu_seqlens_q[i + 1], a.context_lens[i]);
}

// Units of a share: equal ones, but no less than two
__device__ __forceinline__ int i4_share(long long total, int shares) { return (int)max((total + shares - 1) / shares, 2ll); }

struct I4Shared {
  uint64_t bar[kI4Warps * kI4Slots];                                  // a slot's tile has landed
  uint32_t bad[kI4Warps * kI4Slots];                                  // pieces of it whose page lies outside the cache
  int abort, tiles[kI4Warps];
  long long units[kI4Warps];
  int4 start[kI4Warps];                                                  // where a warp's share starts: sequence, (row tile, head) of it, unit of that; row tiles in front of the sequence
  int3 seq[kI4Warps];                                                    // begin, end and context of that sequence
  int beg[kI4Threads], end[kI4Threads], ctx[kI4Threads];                 // what the sequences from the first of these on are
};

// Totals (units, row tiles), and where the shares of this CTA's warps start.  All threads of the CTA, each with a run of sequences.  (Units are counted in 64
// bits: a prompt of 262144 tokens has 3 10^9 of them where three tokens make a row tile.)
struct I4Total { long long units; int tiles, share; };
template <int KEYS> __device__ __forceinline__ I4Total i4_plan(const I4Args& a, I4Shared& sh) {
  const int run = (a.num_seqs + kI4Threads - 1) / kI4Threads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s0 = threadIdx.x * run, s1 = min(a.num_seqs, s0 + run), heads = a.Hkv * a.head_tiles;
  long long mine = 0;
  int tiles = 0;
  for (int i = s0; i < s1; i++) {
    const I4Seq s = i4_load<KEYS>(a, i);
    tiles += s.tiles * heads;
    mine += (long long)s.tiles * heads * s.per_tile;
  }
  long long incl = mine;
  int incl_t = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    const int t = __shfl_up_sync(0xffffffffu, incl_t, o);
    if (lane >= o) { incl += v; incl_t += t; }
  }
  if (lane == 31) { sh.units[warp] = incl; sh.tiles[warp] = incl_t; }
  __syncthreads();
  long long before = incl - mine;
  int before_t = incl_t - tiles;
  I4Total total = {0, 0, 0};
#pragma unroll
  for (int w = 0; w < kI4Warps; w++) {
    if (w < warp) { before += sh.units[w]; before_t += sh.tiles[w]; }
    total.units += sh.units[w]; total.tiles += sh.tiles[w];
  }
  total.share = i4_share(total.units, a.shares);
#pragma unroll
  for (int w = 0; w < kI4Warps; w++) {                                   // the thread whose run a share starts in finds the sequence
    const long long u = ((long long)blockIdx.x * kI4Warps + w) * total.share;
    if (u < before || u >= before + mine) continue;
    long long base = before;
    int t = before_t;
    for (int i = s0;; i++) {
      const int3 x = make_int3(a.cu_seqlens_q[i], a.cu_seqlens_q[i + 1], a.context_lens[i]);
      const I4Seq s = i4_seq<KEYS>(a, x.x, x.y, x.z);
      const int n = s.tiles * heads;
      const long long end = base + (long long)n * s.per_tile;
      if (u < end || i + 1 >= s1) {
        const int th = (int)((u - base) / s.per_tile);
        sh.start[w] = make_int4(i, th, (int)(u - base - (long long)th * s.per_tile), t);
        sh.seq[w] = x;
        break;
      }
      base = end;
      t += n;
    }
  }
  __syncthreads();
  return total;
}

// A piece of work: units [unit, unit + units) of one (row tile, head)
struct I4Piece {
  I4Seq s; int seq, tile, hkv, ht, index, unit, units;                   // ht: tile of the group's heads; index: of this row tile among all
  int gh, head0, tok0, n_tok, base_limit, t_begin, t_end;                // t_begin .. t_end: its tiles of keys that any row sees
};
template <int KEYS> __device__ __forceinline__ void i4_fill(const I4Args& a, I4Piece& p, int left) {
  p.units = min(p.s.per_tile - p.unit, left);
  p.gh = min(a.g - p.ht * a.rows, a.rows);
  p.head0 = p.hkv * a.g + p.ht * a.rows;
  p.tok0 = p.s.q_beg + p.tile * a.tq;
  p.n_tok = p.tok0 < 0 ? 0 : min(min(a.tq, p.s.q_len - p.tile * a.tq), a.T - p.tok0);
  p.base_limit = p.s.ctx - p.s.q_len + p.tile * a.tq;                    // last key the tile's first token sees
  const int max_limit = p.base_limit + p.n_tok - 1;
  const int low = a.window > 0 ? max(0, p.base_limit - a.window + 1) / KEYS : 0;
  p.t_begin = max(p.s.first + p.unit, low);
  p.t_end = p.n_tok > 0 ? min(p.s.first + p.unit + p.units, max_limit >= 0 ? max_limit / KEYS + 1 : 0) : 0;
}
// the piece that a share starts with; `left` units the share has
template <int KEYS> __device__ __forceinline__ I4Piece i4_first(const I4Args& a, const int4& at, const int3& seq, int left) {
  I4Piece p;
  p.seq = at.x;
  p.s = i4_seq<KEYS>(a, seq.x, seq.y, seq.z);
  const int heads = a.Hkv * a.head_tiles, head = at.y % heads;
  p.unit = at.z;
  p.index = at.w + at.y;
  p.tile = at.y / heads;
  p.hkv = head / a.head_tiles;
  p.ht = head - p.hkv * a.head_tiles;
  i4_fill<KEYS>(a, p, left);
  return p;
}
// the piece behind p
template <int KEYS> __device__ __forceinline__ void i4_next(const I4Args& a, const I4Shared& sh, I4Piece& p, int left) {
  p.unit = 0;
  p.index++;
  if (++p.ht == a.head_tiles) {
    p.ht = 0;
    if (++p.hkv == a.Hkv) {
      p.hkv = 0;
      if (++p.tile == p.s.tiles) {
        p.tile = 0;
        do {
          const int i = ++p.seq - sh.start[0].x;
          p.s = i < kI4Threads ? i4_seq<KEYS>(a, sh.beg[i], sh.end[i], sh.ctx[i]) : i4_load<KEYS>(a, p.seq);
        } while (p.s.tiles == 0 && p.seq + 1 < a.num_seqs);
      }
    }
  }
  i4_fill<KEYS>(a, p, left);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Element pairs of an 8 x 8 matrix of 16-bit values, lane 4 i + j with (i, 2 j) and (i, 2 j + 1), to those of its transpose
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Multipliers of one scale (or of a pair of scales) as bf16 pairs, from (byte << 4) in both halves: s 2^109 for the lower nibble of a byte, s 2^105 for the
// upper one, -8 s 2^-24.  None leaves bf16's exponents.  (Two of them by exact products: the integer pipe is the busier one.)
struct I4Scale { uint32_t lo, hi, z; };
__device__ __forceinline__ I4Scale i4_scale(uint32_t b4) {
  const uint32_t lo = b4 + 0x6E006E00u;
  return {lo, hmul2_bf16(lo, 0x3D803D80u), hmul2_bf16(lo, 0x80088008u)};
}
__device__ __forceinline__ uint32_t i4_lower(uint32_t w, const I4Scale& s) { return hfma2_bf16(w & 0x000F000Fu, s.lo, s.z); }
__device__ __forceinline__ uint32_t i4_upper(uint32_t w, const I4Scale& s) { return hfma2_bf16(w & 0x00F000F0u, s.hi, s.z); }

// Two probabilities as bf16, and what that rounding leaves of them, as bf16 again: together 2^-17 of each
__device__ __forceinline__ uint32_t pair_rest(uint32_t p, float a, float b) { return pack_bf16x2(a - __uint_as_float(p << 16), b - __uint_as_float(p & 0xffff0000u)); }

template <int D, int R, bool kPlain, bool kSplitP>
__global__ void __launch_bounds__(kI4Threads, I4Geo<D, R>::ctas) gqa_int4_kernel(const I4Args a) {
  using G = I4Geo<D, R>;
  constexpr bool kNarrow = R == 8;                                       // the keys and the value dims are the 16 rows of a product, the query rows its 8 columns
  constexpr int ST = G::slots, JT = G::keys / 8;                         // JT: column tiles of the scores
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ I4Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = lane & 3, n = lane >> 2;                                 // fragment coordinates: column pair, row
  if (threadIdx.x == 0) {
    sh.abort = 0;
    for (int i = 0; i < kI4Warps * ST; i++) mbar_init(smem_u32(&sh.bar[i]), 1);
    mbar_fence_init();
  }
  pdl_wait();                                                            // (no early trigger: join CTAs that wait beside the last shares cost 41 us where 39.5 do, 60 x 3000, heads of 256)
  const I4Total total = i4_plan<G::keys>(a, sh);                         // (its barriers also publish the initialised mbarriers)
  if (blockIdx.x == 0 && threadIdx.x == 0) a.cuts[0] = make_int4(total.tiles, 0, 0, 0);
  const int share = total.share;
  if ((long long)blockIdx.x * kI4Warps * share >= total.units) return;
  const int mine = blockIdx.x * kI4Warps + warp;                         // this warp's share
  const long long u0 = (long long)mine * share;
  int left = (int)min((long long)share, max(0ll, total.units - u0));         // units of it still to do
  uint8_t* ring = smem + warp * G::warp_bytes;
  uint64_t* bars = sh.bar + warp * ST;
  const uint32_t page_bytes = (uint32_t)a.block_size * (G::row + G::srow), id_bytes = a.Hkv * page_bytes;      // of one head, of a page id
  const bool one_page = a.block_size == G::keys;                         // a tile of keys is a page (kPlain: lies in one)
  const float scale = a.scale_log2 * 16777216.f;

  // The copies of a tile of keys into a slot.  Pages outside the cache are marked; those behind the context stay masked, whatever the slot holds.
  auto fetch = [&](const I4Piece& p, int tile, int slot, int id) {
    const uint32_t bar = smem_u32(bars + slot), dst = smem_u32(ring) + slot * G::stage;
    if constexpr (kPlain) {
      if (lane == 0) {
        const bool there = id >= 0 && id < a.num_blocks && NE_INDEX_OK(id, BK_CACHE_PAGES, kKernelI4, __LINE__);
        sh.bad[warp * ST + slot] = !there;                               // seen by the others behind the barrier's phase
        if (!there) mbar_arrive(bar);
        else {
          const unsigned long long at = (unsigned long long)(uint32_t)id * id_bytes + (uint32_t)p.hkv * page_bytes;
          mbar_expect_tx(bar, G::stage);
          if (one_page) {
            bulk_load(dst, a.k + at, G::half, bar);
            bulk_load(dst + G::half, a.v + at, G::half, bar);
          } else {
            const int tok = tile * G::keys % a.block_size, c0 = tok * G::row, s0 = a.block_size * G::row + tok * G::srow;
            bulk_load(dst, a.k + at + c0, G::codes, bar);
            bulk_load(dst + G::codes, a.k + at + s0, G::half - G::codes, bar);
            bulk_load(dst + G::half, a.v + at + c0, G::codes, bar);
            bulk_load(dst + G::half + G::codes, a.v + at + s0, G::half - G::codes, bar);
          }
        }
      }
    } else {
    // pages smaller than a tile: a lane copies each
    const int bs = a.block_size, pg = tile * (G::keys / bs) + lane;
    const bool seen = lane < G::keys / bs && pg < (p.s.ctx + bs - 1) / bs;
    const int pid = seen ? a.block_tables[(long long)p.seq * a.bt_ld + pg] : -1;
    const bool there = pid >= 0 && pid < a.num_blocks && NE_INDEX_OK(pid, BK_CACHE_PAGES, kKernelI4, __LINE__);
    const unsigned all = __ballot_sync(0xffffffffu, there), bad = __ballot_sync(0xffffffffu, seen && !there);
    if (lane == 0) {
      sh.bad[warp * ST + slot] = bad;
      if (all) mbar_expect_tx(bar, __popc(all) * 2 * bs * (G::row + G::srow)); else mbar_arrive(bar);
    }
    __syncwarp();
    if (there) {
      const unsigned long long at = (unsigned long long)(uint32_t)pid * id_bytes + (uint32_t)p.hkv * page_bytes;
      const uint32_t c0 = dst + lane * bs * G::row, s0 = dst + G::codes + lane * bs * G::srow;
      bulk_load(c0, a.k + at, bs * G::row, bar);
      bulk_load(s0, a.k + at + bs * G::row, bs * G::srow, bar);
      bulk_load(c0 + G::half, a.v + at, bs * G::row, bar);
      bulk_load(s0 + G::half, a.v + at + bs * G::row, bs * G::srow, bar);
    }
    }
  };
  // page of a tile of keys (its id is read one tile ahead of the copies)
  auto page_of = [&](const I4Piece& p, int tile) {
    return kPlain && tile < p.t_end ? a.block_tables[(long long)p.seq * a.bt_ld + (one_page ? tile : tile * G::keys / a.block_size)] : -1;
  };

  I4Piece p;
  int slot = 0, phase = 0;                                               // of the next tile to read
  if (left > 0) {
    p = i4_first<G::keys>(a, sh.start[warp], sh.seq[warp], left);
    if (p.t_begin < p.t_end) fetch(p, p.t_begin, 0, page_of(p, p.t_begin));
  }
  if (const int i = sh.start[0].x + threadIdx.x; i < a.num_seqs) {
    sh.beg[threadIdx.x] = a.cu_seqlens_q[i]; sh.end[threadIdx.x] = a.cu_seqlens_q[i + 1]; sh.ctx[threadIdx.x] = a.context_lens[i];
  }
  __syncthreads();                                                       // the table of sequences
  if (left == 0) return;
  // The second tile is asked for when the first is there: all warps start at once, and the first tiles of some would come behind the second ones of others
  bool lead = p.t_begin + 1 < p.t_end;
  int id = page_of(p, p.t_begin + 1);

  while (true) {
    const int n_tok = p.n_tok, gh = p.gh, head0 = p.head0, tok0 = p.tok0, base_limit = p.base_limit, max_limit = p.base_limit + p.n_tok - 1;
    if (!lead) id = page_of(p, p.t_begin + ST);

    // this lane's two query rows (fragment rows n and n + 8): token and head
    // (narrow: it loads row n and has results of rows 2 c and 2 c + 1)
    const int r0 = kNarrow ? 2 * c : n, r1 = kNarrow ? 2 * c + 1 : n + 8;
    const int t0 = r0 / gh, t1 = r1 / gh, h0 = r0 - t0 * gh, h1 = r1 - t1 * gh;
    const bool ok0 = t0 < n_tok, ok1 = t1 < n_tok;
    const int lim0 = ok0 ? base_limit + t0 : -1, lim1 = ok1 ? base_limit + t1 : -1;
    constexpr int QF = kNarrow ? 2 : 4;                                  // registers of a query fragment
    uint32_t qa[G::q_regs ? G::ks : 1][QF];
    uint4* sq = reinterpret_cast<uint4*>(ring + ST * G::stage);
    {
      const int tq0 = kNarrow ? n / gh : t0, hq0 = kNarrow ? n - tq0 * gh : h0;
      const bool okq = kNarrow ? tq0 < n_tok : ok0;
      const uint2* p0 = reinterpret_cast<const uint2*>(a.q + (long long)(tok0 + (okq ? tq0 : 0)) * a.q_ld + (long long)(head0 + (okq ? hq0 : 0)) * D + c * (D / 4));
      const uint2* p1 = reinterpret_cast<const uint2*>(a.q + (long long)(tok0 + (ok1 ? t1 : 0)) * a.q_ld + (long long)(head0 + (ok1 ? h1 : 0)) * D + c * (D / 4));
      if constexpr (G::q_regs) {
        // the products want the words of a step in neighbouring registers, the loads pairs of them: without an operation in between, every product moves them
        const uint32_t nil = (uint32_t)a.shares >> 31;
#pragma unroll
        for (int ks = 0; ks < G::ks; ks++) {
          const uint2 x0 = okq ? p0[ks] : make_uint2(0, 0);
          if constexpr (kNarrow) { qa[ks][0] = x0.x ^ nil; qa[ks][1] = x0.y ^ nil; }
          else {
            const uint2 x1 = ok1 ? p1[ks] : make_uint2(0, 0);
            qa[ks][0] = x0.x ^ nil; qa[ks][1] = x1.x ^ nil; qa[ks][2] = x0.y ^ nil; qa[ks][3] = x1.y ^ nil;
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < G::ks; ks++) {
          const uint2 x0 = ok0 ? p0[ks] : make_uint2(0, 0), x1 = ok1 ? p1[ks] : make_uint2(0, 0);
          sq[ks * 32 + lane] = make_uint4(x0.x, x1.x, x0.y, x1.y);
        }
        __syncwarp();
      }
    }

    constexpr int NT = kNarrow ? G::nt / 2 : G::nt, SJ = kNarrow ? JT / 2 : JT;        // products' results: columns or (narrow) pairs of rows of D and of a tile of keys
    float o[NT][4], l[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY;

#pragma unroll 1
    for (int tile = p.t_begin; tile < p.t_end; tile++) {
      const uint8_t* kt = ring + slot * G::stage;
      const uint8_t* vt = kt + G::half;
      const bool landed = mbar_wait(smem_u32(bars + slot), phase, (volatile int*)&sh.abort, kKernelI4, 100 + slot, 1);
      if (!__all_sync(0xffffffffu, landed)) {                            // a copy has not come: let the others land before the block's memory goes
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
        return;
      }
      if (lead) {
        fetch(p, tile + 1, 1, id);
        id = page_of(p, tile + ST);
        lead = false;
      }
      if (const uint32_t bad = sh.bad[warp * ST + slot]) {               // pages outside the cache read as zeros: code 8
        const int piece = min(a.block_size, G::keys);
        for (int q = 0; q < G::keys / piece; q++)
          if (bad >> q & 1)
            for (int i = lane; i < piece * G::row / 4; i += 32) {
              reinterpret_cast<uint32_t*>(ring + slot * G::stage + q * piece * G::row)[i] = 0x88888888u;
              reinterpret_cast<uint32_t*>(ring + slot * G::stage + G::half + q * piece * G::row)[i] = 0x88888888u;
            }
        fence_proxy_async_smem();                                        // the slot's next copy comes behind these stores
        __syncwarp();
      }
        // scores: column tile j = (kk, t) holds in fragment column 2 c' + e the key 16 kk + 4 (2 t + e) + (c' ^ e): neighbouring lanes read neighbouring rows
        // (narrow: fragment row n of the pair (kk, 0), (kk, 1) is the key of column n)
        float s[SJ][4];
#pragma unroll
        for (int j = 0; j < SJ; j++) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int jb = 0; jb < JT; jb += 2) {
#pragma unroll
          for (int i0 = 0; i0 < G::words; i0 += (G::words < 4 ? G::words : 4)) {
            constexpr int NW = G::words < 4 ? G::words : 4;
            uint32_t w[2][NW];
            I4Scale sc[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const int key = 16 * ((jb + j) >> 1) + 4 * (2 * (j & 1) + (n & 1)) + ((n >> 1) ^ (n & 1));
              const uint8_t* src = kt + key * G::row + c * (G::row / 4) + 4 * i0;
              if constexpr (NW == 2) { const uint2 x = *reinterpret_cast<const uint2*>(src); w[j][0] = x.x; w[j][1] = x.y; }
              else { const uint4 x = *reinterpret_cast<const uint4*>(src); w[j][0] = x.x; w[j][1] = x.y; w[j][2] = x.z; w[j][3] = x.w; }
              sc[j] = i4_scale(kt[G::codes + key * G::srow + (D == 64 ? c >> 1 : D == 128 ? c : 2 * c + i0 / 4)] * 0x00100010u);
            }
#pragma unroll
            for (int i = 0; i < NW; i++) {
              if constexpr (kNarrow) {
                const uint32_t (&qe)[2] = qa[2 * (i0 + i)], (&qo)[2] = qa[2 * (i0 + i) + 1];
                const uint32_t ke[4] = {i4_lower(w[0][i], sc[0]), i4_lower(w[1][i], sc[1]), i4_upper(w[0][i], sc[0]), i4_upper(w[1][i], sc[1])};
                mma_16816(s[jb / 2], ke, qe[0], qe[1]);
                const uint32_t ko[4] = {i4_lower(w[0][i] >> 8, sc[0]), i4_lower(w[1][i] >> 8, sc[1]), i4_upper(w[0][i] >> 8, sc[0]), i4_upper(w[1][i] >> 8, sc[1])};
                mma_16816(s[jb / 2], ko, qo[0], qo[1]);
              } else {
              uint32_t qe[4], qo[4];
              if constexpr (G::q_regs) {
#pragma unroll
                for (int r = 0; r < 4; r++) { qe[r] = qa[2 * i][r]; qo[r] = qa[2 * i + 1][r]; }
              } else {
                const uint4 x = sq[(2 * (i0 + i)) * 32 + lane], y = sq[(2 * (i0 + i) + 1) * 32 + lane];
                qe[0] = x.x; qe[1] = x.y; qe[2] = x.z; qe[3] = x.w;
                qo[0] = y.x; qo[1] = y.y; qo[2] = y.z; qo[3] = y.w;
              }
#pragma unroll
              for (int j = 0; j < 2; j++) mma_16816(s[jb + j], qe, i4_lower(w[j][i], sc[j]), i4_upper(w[j][i], sc[j]));
#pragma unroll
              for (int j = 0; j < 2; j++) mma_16816(s[jb + j], qo, i4_lower(w[j][i] >> 8, sc[j]), i4_upper(w[j][i] >> 8, sc[j]));
              }
            }
          }
        }
        const int key0 = tile * G::keys;
        if (key0 + G::keys - 1 > base_limit || (a.window > 0 && key0 <= max_limit - a.window)) {
          const int low0 = a.window > 0 ? lim0 - a.window : -1, low1 = a.window > 0 ? lim1 - a.window : -1;
#pragma unroll
          for (int j = 0; j < JT; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              // narrow: tile j's half of the pair's results, one key for both rows
              const int key = key0 + 16 * (j >> 1) + (kNarrow ? 4 * (2 * (j & 1) + (n & 1)) + ((n >> 1) ^ (n & 1)) : 4 * (2 * (j & 1) + e) + (c ^ e));
              float& y0 = kNarrow ? s[j / 2][2 * (j & 1)] : s[kNarrow ? 0 : j][e];
              float& y1 = kNarrow ? s[j / 2][2 * (j & 1) + 1] : s[kNarrow ? 0 : j][2 + e];
              if (key > lim0 || key <= low0) y0 = -INFINITY;
              if (key > lim1 || key <= low1) y1 = -INFINITY;
            }
        }
        float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
        for (int j = 0; j < SJ; j++) {
          x0 = fmaxf(x0, fmaxf(s[j][0], s[j][kNarrow ? 2 : 1]));
          x1 = fmaxf(x1, fmaxf(s[j][kNarrow ? 1 : 2], s[j][3]));
        }
        x0 *= scale; x1 *= scale;
        // the reference maximum moves only when a score exceeds it by more than 2^8 (or is the first): rare, so that the rows' lanes compare notes only then
        if (__any_sync(0xffffffffu, x0 > m0 + 8.f || x1 > m1 + 8.f || (m0 == -INFINITY && x0 > m0) || (m1 == -INFINITY && x1 > m1))) {
#pragma unroll
          for (int d = kNarrow ? 4 : 1; d < (kNarrow ? 32 : 4); d <<= 1) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
          }
          const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
          const float f0 = n0 == -INFINITY ? 1.f : exp2f(m0 - n0), f1 = n1 == -INFINITY ? 1.f : exp2f(m1 - n1);
          m0 = n0; m1 = n1;
          // narrow: columns 2 c and 2 c + 1 alternate
          const float fa = kNarrow ? f1 : f0, fb = kNarrow ? f0 : f1;
          l[0] *= f0; l[1] *= fa; l[2] *= fb; l[3] *= f1;
#pragma unroll
          for (int i = 0; i < NT; i++) { o[i][0] *= f0; o[i][1] *= fa; o[i][2] *= fb; o[i][3] *= f1; }
        }
        const float z0 = m0 == -INFINITY ? 0.f : -m0, z1 = m1 == -INFINITY ? 0.f : -m1;
#pragma unroll
        for (int kk = 0; kk < G::keys / 16; kk++) {
          uint32_t pr[4], pl[4];                                         // probabilities; with kSplitP what their rounding leaves
          if constexpr (kNarrow) {
            // a lane has two rows of one key, the product wants two keys of one row
#pragma unroll
            for (int t = 0; t < 2; t++) {
              const float x = exp2f(fmaf(s[kk][2 * t], scale, z0)), y = exp2f(fmaf(s[kk][2 * t + 1], scale, z1));
              const uint32_t p2 = pack_bf16x2(x, y);
              pr[t] = transpose_8x8(p2);
              if constexpr (kSplitP) pl[t] = transpose_8x8(pair_rest(p2, x, y));
            }
            const uint32_t ones[4] = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
            mma_16816(l, ones, pr[0], pr[1]);                            // the sum of the probabilities as they are rounded
            if constexpr (kSplitP) mma_16816(l, ones, pl[0], pl[1]);
          } else {
#pragma unroll
          for (int t = 0; t < 2; t++) {
            const float (&v)[4] = s[2 * kk + t];
            const float x0 = exp2f(fmaf(v[0], scale, z0)), x1 = exp2f(fmaf(v[1], scale, z0)), y0 = exp2f(fmaf(v[2], scale, z1)), y1 = exp2f(fmaf(v[3], scale, z1));
            pr[2 * t] = pack_bf16x2(x0, x1);
            pr[2 * t + 1] = pack_bf16x2(y0, y1);
            if constexpr (kSplitP) { pl[2 * t] = pair_rest(pr[2 * t], x0, x1); pl[2 * t + 1] = pair_rest(pr[2 * t + 1], y0, y1); }
          }
          mma_16816(l, pr, 0x3F803F80u, 0x3F803F80u);
          if constexpr (kSplitP) mma_16816(l, pl, 0x3F803F80u, 0x3F803F80u);
          }
          // values: this lane's four keys of the step, an eighth of each row
          uint32_t w[4][G::vwords], sb[4];
#pragma unroll
          for (int x = 0; x < 4; x++) {
            const int key = 16 * kk + 4 * x + (c ^ (x & 1));
            const uint8_t* src = vt + key * G::row + n * (G::row / 8);
            if constexpr (D == 64) w[x][0] = *reinterpret_cast<const uint32_t*>(src);
            else if constexpr (D == 128) { const uint2 y = *reinterpret_cast<const uint2*>(src); w[x][0] = y.x; w[x][1] = y.y; }
            else { const uint4 y = *reinterpret_cast<const uint4*>(src); w[x][0] = y.x; w[x][1] = y.y; w[x][2] = y.z; w[x][3] = y.w; }
            sb[x] = vt[G::codes + key * G::srow + (D == 64 ? n >> 2 : D == 128 ? n >> 1 : n)];
          }
          const I4Scale sa = i4_scale(sb[0] * 16 + sb[1] * 0x100000u), sz = i4_scale(sb[2] * 16 + sb[3] * 0x100000u);
#pragma unroll
          for (int i = 0; i < G::vwords; i++) {
            // a word's low half: even dims 0 2 4 6, high half: odd dims; two keys side by side
            const uint32_t al = __byte_perm(w[0][i], w[1][i], 0x5410), ah = __byte_perm(w[0][i], w[1][i], 0x7632);
            const uint32_t bl = __byte_perm(w[2][i], w[3][i], 0x5410), bh = __byte_perm(w[2][i], w[3][i], 0x7632);
            auto both = [&](int j, uint32_t a0, uint32_t b0, uint32_t a1, uint32_t b1) {       // dims j and j + 1 of the lane's eight: first keys, second keys
              if constexpr (kNarrow) {
                const uint32_t x[4] = {a0, a1, b0, b1};
                mma_16816(o[4 * i + j / 2], x, pr[0], pr[1]);
                if constexpr (kSplitP) mma_16816(o[4 * i + j / 2], x, pl[0], pl[1]);
              } else {
                mma_16816(o[kNarrow ? 0 : 8 * i + j], pr, a0, b0);
                mma_16816(o[kNarrow ? 0 : 8 * i + j + 1], pr, a1, b1);
                if constexpr (kSplitP) { mma_16816(o[kNarrow ? 0 : 8 * i + j], pl, a0, b0); mma_16816(o[kNarrow ? 0 : 8 * i + j + 1], pl, a1, b1); }
              }
            };
            both(0, i4_lower(al, sa), i4_lower(bl, sz), i4_lower(ah, sa), i4_lower(bh, sz));
            both(2, i4_upper(al, sa), i4_upper(bl, sz), i4_upper(ah, sa), i4_upper(bh, sz));
            both(4, i4_lower(al >> 8, sa), i4_lower(bl >> 8, sz), i4_lower(ah >> 8, sa), i4_lower(bh >> 8, sz));
            both(6, i4_upper(al >> 8, sa), i4_upper(bl >> 8, sz), i4_upper(ah >> 8, sa), i4_upper(bh >> 8, sz));
          }
        }
        __syncwarp();                                                    // every lane has read the slot
      if (tile + ST < p.t_end) fetch(p, tile + ST, slot, id);
      id = page_of(p, tile + ST + 1);
      if (++slot == ST) { slot = 0; phase ^= 1; }
    }

    // what follows this piece, and its first copies
    const bool whole = p.units == p.s.per_tile, head = p.unit == 0;
    if (head && lane == 0 && p.index < a.max_tiles) {                                      // the row tile's entry for the join: rows, first share with a piece of it, pieces
      const int pieces = (int)((u0 + (min((long long)share, total.units - u0) - left) + p.s.per_tile - 1) / share) - mine + 1;
      a.cuts[1 + p.index] = make_int4(tok0, max(0, n_tok * gh) | gh << 8 | pieces << 16, head0, mine);
    }
    left -= p.units;
    if (left > 0) {
      i4_next<G::keys>(a, sh, p, left);
#pragma unroll 1
      for (int i = 0; i < ST; i++)
        if (p.t_begin + i < p.t_end) fetch(p, p.t_begin + i, slot + i < ST ? slot + i : slot + i - ST, page_of(p, p.t_begin + i));
    }

    const float sum0 = l[0], sum1 = kNarrow ? l[1] : l[2];
    const float inv0 = sum0 == 0.f ? 0.f : 16777216.f / sum0, inv1 = sum1 == 0.f ? 0.f : 16777216.f / sum1;       // a NaN stays one
    const long long row0 = (long long)(tok0 + t0) * a.Hq + head0 + h0, row1 = (long long)(tok0 + t1) * a.Hq + head0 + h1;
    const long long at = ((long long)mine * 2 + (head ? 1 : 0)) * R;     // a row tile's first piece: the share's second place
    auto put = [&](int d, const float4& x, const float4& y) {             // dims d .. d + 3 of both rows
      if (whole) {
        if (ok0) *reinterpret_cast<uint2*>(a.out + row0 * D + d) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
        if (ok1) *reinterpret_cast<uint2*>(a.out + row1 * D + d) = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
      } else {
        if (ok0) *reinterpret_cast<float4*>(a.part + (at + r0) * D + d) = x;
        if (ok1) *reinterpret_cast<float4*>(a.part + (at + r1) * D + d) = y;
      }
    };
    if constexpr (kNarrow) {                                             // dims n D/8 + 4 i ..
#pragma unroll
      for (int i = 0; i < G::nt / 4; i++) {
        const float (&u)[4] = o[2 * i], (&v)[4] = o[2 * i + 1];
        put(n * (D / 8) + 4 * i, make_float4(u[0] * inv0, u[2] * inv0, v[0] * inv0, v[2] * inv0), make_float4(u[1] * inv1, u[3] * inv1, v[1] * inv1, v[3] * inv1));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int i = 0; i < G::nt / 4; i++)                              // dims (2 c + e) D/8 + 4 i ..
          put((2 * c + e) * (D / 8) + 4 * i, make_float4(o[4 * i][e] * inv0, o[4 * i + 1][e] * inv0, o[4 * i + 2][e] * inv0, o[4 * i + 3][e] * inv0),
              make_float4(o[4 * i][2 + e] * inv1, o[4 * i + 1][2 + e] * inv1, o[4 * i + 2][2 + e] * inv1, o[4 * i + 3][2 + e] * inv1));
    }
    if (!whole && (kNarrow ? n == 0 : c == 0)) {
      if (ok0) a.lse2[at + r0] = sum0 == 0.f ? -INFINITY : m0 + log2f(sum0);
      if (ok1) a.lse2[at + r1] = sum1 == 0.f ? -INFINITY : m1 + log2f(sum1);
    }
    if (left == 0) break;
  }
}

// Joins the pieces of row tile x where cuts run through it:  out = sum_p 2^(lse_p - m) part_p / sum_p 2^(lse_p - m).  The first piece sits in its share's second
// place, the others' in their first.  Groups of D / 4 lanes
// take a row each (kSplit false), or the groups of a CTA share the pieces of row y.
constexpr int i4_join_threads(bool split) { return split ? 512 : 128; }
template <int D, bool kSplit>
__global__ void __launch_bounds__(i4_join_threads(kSplit)) gqa_int4_join_kernel(const I4Args a) {
  pdl_wait(); pdl_trigger();
  constexpr int Q = D / 4, GR = i4_join_threads(kSplit) / Q;             // quads of a row; groups
  __shared__ float4 s_acc[kSplit ? GR : 1][Q];
  __shared__ float s_sum[GR], s_max[GR];
  const int4 cut = a.cuts[1 + blockIdx.x];
  if ((int)blockIdx.x >= a.cuts[0].x) return;
  const int rows = cut.y & 255, gh = cut.y >> 8 & 255, pieces = cut.y >> 16, first = cut.w;
  if (pieces <= 1) return;
  const int grp = threadIdx.x / Q, f = threadIdx.x % Q;
  const int r = kSplit ? blockIdx.y : blockIdx.y * GR + grp;
  if (r >= rows) return;                                                 // (kSplit: the whole CTA)
  constexpr int kBatch = 8, step = kSplit ? GR : 1;                      // loads in flight; pieces between a group's
  const int i0 = kSplit ? grp : 0;
  auto place = [&](int i) { return ((long long)(first + i) * 2 + (i == 0)) * a.rows + r; };
  float m = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int b = i0; b < pieces; b += kBatch * step) {
    float lse[kBatch];
    float4 y[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      const int i = b + j * step;
      lse[j] = i < pieces ? a.lse2[place(i)] : -INFINITY;
      y[j] = i < pieces ? *reinterpret_cast<const float4*>(a.part + place(i) * D + 4 * f) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top = m;
#pragma unroll
    for (int j = 0; j < kBatch; j++) top = fmaxf(top, lse[j]);
    const float old = m == -INFINITY ? 0.f : exp2f(m - top);
    sum *= old; acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
    m = top;
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      const float wt = lse[j] == -INFINITY ? 0.f : m == -INFINITY ? lse[j] : exp2f(lse[j] - m);       // scores that are no numbers stay visible
      sum += wt;
      acc.x += wt * y[j].x; acc.y += wt * y[j].y; acc.z += wt * y[j].z; acc.w += wt * y[j].w;
    }
  }
  if (kSplit) {
    s_acc[grp][f] = acc;
    if (f == 0) { s_sum[grp] = sum; s_max[grp] = m; }
    __syncthreads();
    if (grp > 0) return;
    float top = -INFINITY;
    for (int g = 0; g < GR; g++) top = fmaxf(top, s_max[g]);
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    sum = 0.f;
    for (int g = 0; g < GR; g++) {
      if (s_sum[g] == 0.f) continue;                                     // saw no key
      const float wt = s_max[g] == -INFINITY ? 1.f : exp2f(s_max[g] - top);
      const float4 z = s_acc[g][f];
      sum += wt * s_sum[g];
      acc.x += wt * z.x; acc.y += wt * z.y; acc.z += wt * z.z; acc.w += wt * z.w;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const long long row = (long long)(cut.x + r / gh) * a.Hq + cut.z + r % gh;
  *reinterpret_cast<uint2*>(a.out + row * D + 4 * f) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

}  // namespace ne

using namespace ne;

namespace {
template <int D, int R, bool kPlain, bool kSplitP> cudaError_t launch_i4_main(const I4Args& a, cudaStream_t st) {
  static bool configured[64] = {};                                       // per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(gqa_int4_kernel<D, R, kPlain, kSplitP>, cudaFuncAttributeMaxDynamicSharedMemorySize, I4Geo<D, R>::smem);
    if (e != cudaSuccess) return e;
    if (dev < 64) configured[dev] = true;
  }
  return launch_pdl(gqa_int4_kernel<D, R, kPlain, kSplitP>, dim3((unsigned)(a.shares / kI4Warps)), dim3(kI4Threads), I4Geo<D, R>::smem, st, a);
}
template <int D, int R, bool kSplitP> cudaError_t launch_i4_pages(const I4Args& a, cudaStream_t st) {
  return a.block_size % I4Geo<D, R>::keys == 0 ? launch_i4_main<D, R, true, kSplitP>(a, st) : launch_i4_main<D, R, false, kSplitP>(a, st);
}
template <int D, int R> cudaError_t launch_i4_rows(const I4Args& a, cudaStream_t st) {
  if constexpr (D == 128) { if (a.window <= 0) return launch_i4_pages<D, R, false>(a, st); }
  return launch_i4_pages<D, R, true>(a, st);
}
template <int D> int launch_i4(const I4Args& a, int tiles, cudaStream_t st) {
  const cudaError_t e = a.rows == 8 ? launch_i4_rows<D, 8>(a, st) : launch_i4_rows<D, 16>(a, st);
  if (e != cudaSuccess) return (int)e;
  // Many pieces a row tile: a CTA per row shares them.  us of attention with a group per row / a CTA per row, 1184 shares, 64 / 4 heads of 128: 4 row tiles 57 / 34,
  // 8: 62 / 50, 32: 51 / 57, 64: 33 / 48, 512: 86 / 194.
  if (a.shares > 64 * tiles) return (int)launch_pdl(gqa_int4_join_kernel<D, true>, dim3((unsigned)tiles, a.rows), dim3(i4_join_threads(true)), 0, st, a);
  const int rows_a_cta = i4_join_threads(false) / (D / 4);
  return (int)launch_pdl(gqa_int4_join_kernel<D, false>, dim3((unsigned)tiles, (a.rows + rows_a_cta - 1) / rows_a_cta), dim3(i4_join_threads(false)), 0, st, a);
}
}  // namespace

// Shares of the work that an SM's CTAs hold for heads of D and row tiles of `rows` (0: not built for them)
extern "C" int ne_gqa_int4_shares(int D, int rows) {
  if (rows != 8 && rows != 16) return 0;
  return kI4Warps * (D == 64 ? I4Geo<64, 8>::ctas : D == 128 ? (rows == 8 ? I4Geo<128, 8>::ctas : I4Geo<128, 16>::ctas) : D == 256 ? I4Geo<256, 8>::ctas : 0);
}

// q bf16 [T, Hq, D] with rows q_ld elements apart (8-byte aligned); k / v uint8 [num_blocks, Hkv, block_size (D/2 + D/32)].  rows: of a row tile, 8 or 16.  shares: of the work, a multiple of 4, each with
// two places of them in part fp32 [shares, 2, rows, D] and lse2 fp32 [shares, 2, rows].  tiles: an upper bound of the row tiles, the sum over sequences of
// ceil(q_len / tq) Hkv ceil(g / rows), tq = max(1, rows / g); cuts int32 [1 + tiles, 4].
extern "C" int ne_gqa_int4(const void* q, long long q_ld, const void* k, const void* v, int num_blocks, int block_size, const int* block_tables, long long bt_ld, int bt_width,
                           const int* cu_seqlens_q, const int* context_lens, int num_seqs, int T, int Hq, int Hkv, int D, int rows, int shares, int tiles, int window, float scale,
                           void* out, float* part, float* lse2, void* cuts, cudaStream_t st) {
  if (T <= 0 || num_seqs <= 0) return 0;
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv || num_blocks < 1 || bt_width < 1 || shares < kI4Warps || shares % kI4Warps || shares >= 32768 || tiles < 1 || !part || !lse2 || !cuts)
    return 1001;
  if (rows != 8 && rows != 16) return 1003;
  if (!(block_size == 16 || block_size == 32 || (block_size > 0 && block_size % 64 == 0))) return 1002;
  I4Args a{};
  a.q = (const __nv_bfloat16*)q; a.q_ld = q_ld; a.k = (const uint8_t*)k; a.v = (const uint8_t*)v; a.num_blocks = num_blocks; a.block_size = block_size;
  a.block_tables = block_tables; a.bt_ld = bt_ld; a.bt_width = bt_width; a.cu_seqlens_q = cu_seqlens_q; a.context_lens = context_lens; a.num_seqs = num_seqs;
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.g = Hq / Hkv; a.rows = rows; a.tq = a.g >= rows ? 1 : rows / a.g; a.head_tiles = (a.g + rows - 1) / rows; a.shares = shares; a.max_tiles = tiles;
  a.window = window > 0 ? window : 0; a.scale_log2 = scale * 1.4426950408889634f;
  a.out = (__nv_bfloat16*)out; a.part = part; a.lse2 = lse2; a.cuts = (int4*)cuts;
  switch (D) {
    case 64: return launch_i4<64>(a, tiles, st);
    case 128: return launch_i4<128>(a, tiles, st);
    case 256: return launch_i4<256>(a, tiles, st);
    default: return 1004;
  }
}
