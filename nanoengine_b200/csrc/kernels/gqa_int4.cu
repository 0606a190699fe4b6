// Grouped-query paged attention over a key / value cache held in 4 bits (kv4.cuh): decode steps and short portions.
//
//   softmax(q k^T scale) v with k = (c - 8) s of 4-bit codes, a scale per 32 dims; causal, optionally the last `window` keys only
//
// Bound by HBM: D/2 + D/32 bytes a key row, 17/64 of bf16.  One CTA = one KV head x one tile of up to 16 (token, head of the group) rows of one sequence
// x one slice of its keys; its warps take tiles of 64 keys in turn, each with a ring of bulk copies of its own (no barrier among warps until the end).
// A key is unpacked once, in registers, straight into the fragments of mma.m16n8k16: a lane owns a contiguous quarter of a key row and an eighth of a value
// row, the dims of a step of the product and the keys of a step of the second one are permuted to match (query rows and probabilities follow).  tcgen05
// would want the unpacked tile in shared memory or TMEM: 16 rows fill an eighth of its M = 128, and the 64 KB of bf16 a tile of 64 keys would be written and
// read there is seven times what is read from HBM.  Portions with many rows per key run on the tensor-core prompt kernel over expanded pages instead.
//
// Unpacked values (c - 8) s are exact in bf16, scores, maxima, sums and results are 32-bit, probabilities enter the second product as bf16 (2^-9 each) and
// the sum takes them as rounded.  Every byte stands for a finite value, so a masked key (probability 0) adds nothing whatever its page holds.
#include "kv4.cuh"
#include "seq_tile.cuh"

namespace ne {

constexpr int kKernelI4 = 31;
constexpr int kTileKeys = 64;

struct I4Args {
  const __nv_bfloat16* q; long long q_ld;              // [T, Hq, D], rows q_ld apart
  const uint8_t* k; const uint8_t* v; int num_blocks, block_size;
  const int* block_tables; long long bt_ld; int bt_width;
  const int* cu_seqlens_q; const int* context_lens; int num_seqs;
  int T, Hq, Hkv, g, tq, head_tiles, splits, window;   // tq tokens x min(g, 16) heads a tile; head_tiles = ceil(g / 16)
  float scale_log2;
  __nv_bfloat16* out;                                  // [T, Hq, D] (splits == 1)
  float* part; float* lse2;                            // [splits, T, Hq, D], [splits, T, Hq] (splits > 1)
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D> struct I4Geo {
  static constexpr int row = D / 2, srow = D / 32;                      // bytes of a row's codes and scales
  static constexpr int codes = kTileKeys * row, half = codes + kTileKeys * srow, stage = 2 * half;
  static constexpr int words = D / 32;                                  // words of a key row a lane owns (a quarter of the row)
  static constexpr int vwords = D / 64;                                 // words of a value row a lane owns (an eighth)
  static constexpr int ks = D / 16;                                     // k steps of the first product
  static constexpr int nt = D / 8;                                      // column tiles of the second one
};

template <int D, int W, int ST>
__global__ void __launch_bounds__(W * 32, 1) gqa_int4_kernel(const I4Args a) {
  using G = I4Geo<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_bar[W * ST];
  __shared__ uint32_t s_bad[W * ST];                                     // pieces of a slot whose page lies outside the cache
  __shared__ int s_tile[2];
  __shared__ int s_abort;
  __shared__ float s_m[W][16], s_l[W][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = lane & 3, n = lane >> 2;                                 // fragment coordinates: column pair, row
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < W * ST; i++) mbar_init(smem_u32(&s_bar[i]), 1);
    mbar_fence_init();
  }
  pdl_wait(); pdl_trigger();
  if (warp == 0) {
    int seq, tok;
    find_seq_tile(a.cu_seqlens_q, a.num_seqs, a.tq, blockIdx.x, seq, tok);
    if (lane == 0) { s_tile[0] = seq; s_tile[1] = tok; }
  }
  __syncthreads();
  const int seq = s_tile[0], tok0 = s_tile[1];
  if (seq < 0) return;
  const int hkv = blockIdx.y / a.head_tiles, head0 = (blockIdx.y - hkv * a.head_tiles) * 16, split = blockIdx.z;
  const int gh = min(a.g - head0, 16);                                   // heads of this tile
  const int q_beg = a.cu_seqlens_q[seq], q_len = a.cu_seqlens_q[seq + 1] - q_beg;
  const int n_tok = min(min(a.tq, q_beg + q_len - tok0), a.T - tok0);
  if (n_tok <= 0 || tok0 < 0) return;
  const int ctx = (int)min((long long)a.context_lens[seq], (long long)a.bt_width * a.block_size);
  const int base_limit = ctx - q_len + (tok0 - q_beg);                   // last key the tile's first token sees
  const int max_limit = base_limit + n_tok - 1;
  const int first_key = a.window > 0 ? max(0, base_limit - a.window + 1) : 0;
  int t_begin = 0, t_end = 0;                                            // this slice's tiles of 64 keys
  if (max_limit >= first_key) {
    const int lo = first_key / kTileKeys, total = max_limit / kTileKeys + 1 - lo, per = (total + a.splits - 1) / a.splits;
    t_begin = lo + min(split * per, total);
    t_end = lo + min((split + 1) * per, total);
  }
  const int* bt = a.block_tables + (long long)seq * a.bt_ld;
  const int used_pages = (ctx + a.block_size - 1) / a.block_size;
  const long long page_bytes = (long long)a.block_size * (G::row + G::srow);
  uint8_t* ring = smem + warp * (ST * G::stage);

  // this lane's two query rows (fragment rows n and n + 8): token and head
  const int r0 = n, r1 = n + 8;
  const int t0 = r0 / gh, t1 = r1 / gh;
  const bool ok0 = t0 < n_tok, ok1 = t1 < n_tok;
  const int hd0 = hkv * a.g + head0 + r0 % gh, hd1 = hkv * a.g + head0 + r1 % gh;
  const int lim0 = ok0 ? base_limit + t0 : -1, lim1 = ok1 ? base_limit + t1 : -1;

  uint32_t qa[G::ks][4];
  {
    const uint2* p0 = reinterpret_cast<const uint2*>(a.q + (long long)(tok0 + (ok0 ? t0 : 0)) * a.q_ld + (long long)hd0 * D + c * (D / 4));
    const uint2* p1 = reinterpret_cast<const uint2*>(a.q + (long long)(tok0 + (ok1 ? t1 : 0)) * a.q_ld + (long long)hd1 * D + c * (D / 4));
#pragma unroll
    for (int ks = 0; ks < G::ks; ks++) {
      const uint2 u0 = ok0 ? p0[ks] : make_uint2(0, 0), u1 = ok1 ? p1[ks] : make_uint2(0, 0);
      qa[ks][0] = u0.x; qa[ks][1] = u1.x; qa[ks][2] = u0.y; qa[ks][3] = u1.y;
    }
  }

  // copies of one tile into a slot: pieces of one page each; lane 0 only
  const int piece = min(a.block_size, kTileKeys), pieces = kTileKeys / piece;
  auto fetch = [&](int tile, int slot) {
    const uint32_t bar = smem_u32(&s_bar[warp * ST + slot]), dst = smem_u32(ring + slot * G::stage);
    int id[kTileKeys / 16];
    uint32_t bytes = 0, bad = 0;
#pragma unroll
    for (int p = 0; p < kTileKeys / 16; p++) {
      id[p] = -1;
      if (p >= pieces) continue;
      const int pg = (tile * kTileKeys + p * piece) / a.block_size;
      if (pg >= used_pages) continue;                                    // behind the context: masked, whatever the slot holds
      id[p] = bt[pg];
      if (id[p] >= 0 && id[p] < a.num_blocks && NE_INDEX_OK(id[p], BK_CACHE_PAGES, kKernelI4, __LINE__)) bytes += 2 * piece * (G::row + G::srow);
      else { id[p] = -1; bad |= 1u << p; }
    }
    s_bad[warp * ST + slot] = bad;                                       // seen by the others behind the barrier's phase
    if (bytes) mbar_expect_tx(bar, bytes); else mbar_arrive(bar);
#pragma unroll
    for (int p = 0; p < kTileKeys / 16; p++) {
      if (id[p] < 0) continue;
      const int key = tile * kTileKeys + p * piece, tok = key % a.block_size;
      const long long at = ((long long)id[p] * a.Hkv + hkv) * page_bytes;
      if (a.block_size == kTileKeys) {                                   // a page is a tile: codes and scales in one piece
        bulk_load(dst, a.k + at, G::half, bar);
        bulk_load(dst + G::half, a.v + at, G::half, bar);
      } else {
        const long long sc = at + a.block_size * G::row + tok * G::srow;
        const uint32_t d0 = dst + p * piece * G::row, d1 = dst + G::codes + p * piece * G::srow;
        bulk_load(d0, a.k + at + tok * G::row, piece * G::row, bar);
        bulk_load(d1, a.k + sc, piece * G::srow, bar);
        bulk_load(d0 + G::half, a.v + at + tok * G::row, piece * G::row, bar);
        bulk_load(d1 + G::half, a.v + sc, piece * G::srow, bar);
      }
    }
  };

  float o[G::nt][4];
#pragma unroll
  for (int i = 0; i < G::nt; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

  if (lane == 0)
    for (int i = 0; i < ST; i++) if (t_begin + warp + i * W < t_end) fetch(t_begin + warp + i * W, i);
  int slot = 0, phase = 0;
  for (int tile = t_begin + warp; tile < t_end; tile += W) {
    if (!mbar_wait(smem_u32(&s_bar[warp * ST + slot]), phase, (volatile int*)&s_abort, kKernelI4, 100 + slot)) break;
    uint8_t* kt = ring + slot * G::stage;
    const uint8_t* vt = kt + G::half;
    if (const uint32_t bad = s_bad[warp * ST + slot]) {                  // pages outside the cache read as zeros: code 8
      for (int p = 0; p < pieces; p++)
        if (bad >> p & 1)
          for (int i = lane; i < piece * G::row / 4; i += 32) {
            reinterpret_cast<uint32_t*>(kt + p * piece * G::row)[i] = 0x88888888u;
            reinterpret_cast<uint32_t*>(kt + G::half + p * piece * G::row)[i] = 0x88888888u;
          }
      __syncwarp();
    }
    // scores: column tile j = (kk, t) holds for fragment column 2 c' + e the key 16 kk + 4 (2 t + e) + (c' ^ e): neighbouring lanes read neighbouring rows
    float s[8][4];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
      const int key = 16 * (j >> 1) + 4 * (2 * (j & 1) + (n & 1)) + ((n >> 1) ^ (n & 1));
      uint32_t w[G::words];
      const uint8_t* src = kt + key * G::row + c * (G::row / 4);
      if constexpr (D == 64) { const uint2 u = *reinterpret_cast<const uint2*>(src); w[0] = u.x; w[1] = u.y; }
      else {
#pragma unroll
        for (int i = 0; i < G::words / 4; i++) {
          const uint4 u = reinterpret_cast<const uint4*>(src)[i];
          w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
        }
      }
      const uint8_t* sp = kt + G::codes + key * G::srow;
#pragma unroll
      for (int i = 0; i < G::words; i++) {
        uint32_t s2, z;
        if (i % 4 == 0) {
          s2 = kv4_scale_bits(sp[D == 64 ? c >> 1 : D == 128 ? c : 2 * c + i / 4]) * 0x00010001u;
          z = kv4_minus24(s2);
        }
        mma_16816(s[j], qa[2 * i], kv4_pair<0>(w[i], s2, z), kv4_pair<1>(w[i], s2, z));
        mma_16816(s[j], qa[2 * i + 1], kv4_pair<2>(w[i], s2, z), kv4_pair<3>(w[i], s2, z));
      }
    }
    const int key0 = tile * kTileKeys;
    if (key0 + kTileKeys - 1 > base_limit || (a.window > 0 && key0 <= max_limit - a.window)) {
      const int low0 = a.window > 0 ? lim0 - a.window : -1, low1 = a.window > 0 ? lim1 - a.window : -1;
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int key = key0 + 16 * (j >> 1) + 4 * (2 * (j & 1) + e) + (c ^ e);
          if (key > lim0 || key <= low0) s[j][e] = -INFINITY;
          if (key > lim1 || key <= low1) s[j][2 + e] = -INFINITY;
        }
    }
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      x0 = fmaxf(x0, fmaxf(s[j][0], s[j][1]));
      x1 = fmaxf(x1, fmaxf(s[j][2], s[j][3]));
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
    }
    x0 *= a.scale_log2; x1 *= a.scale_log2;
    // the reference maximum moves only when a tile's exceeds it by more than 2^8
    const bool up0 = x0 > m0 + 8.f || m0 == -INFINITY, up1 = x1 > m1 + 8.f || m1 == -INFINITY;
    if (__any_sync(0xffffffffu, (up0 && x0 > m0) || (up1 && x1 > m1))) {
      const float n0 = up0 ? fmaxf(m0, x0) : m0, n1 = up1 ? fmaxf(m1, x1) : m1;
      const float f0 = m0 == -INFINITY ? 0.f : exp2f(m0 - n0), f1 = m1 == -INFINITY ? 0.f : exp2f(m1 - n1);
      m0 = n0; m1 = n1; l0 *= f0; l1 *= f1;
#pragma unroll
      for (int i = 0; i < G::nt; i++) { o[i][0] *= f0; o[i][1] *= f0; o[i][2] *= f1; o[i][3] *= f1; }
    }
    const float z0 = m0 == -INFINITY ? 0.f : -m0, z1 = m1 == -INFINITY ? 0.f : -m1;
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
      uint32_t p[4];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const float (&v)[4] = s[2 * kk + t];
        p[2 * t] = pack_bf16x2(exp2f(fmaf(v[0], a.scale_log2, z0)), exp2f(fmaf(v[1], a.scale_log2, z0)));
        p[2 * t + 1] = pack_bf16x2(exp2f(fmaf(v[2], a.scale_log2, z1)), exp2f(fmaf(v[3], a.scale_log2, z1)));
        const float2 e0 = unpack_bf16x2(p[2 * t]), e1 = unpack_bf16x2(p[2 * t + 1]);
        l0 += e0.x + e0.y; l1 += e1.x + e1.y;
      }
      // values: this lane's four keys of the step, an eighth of each row
      uint32_t w[4][G::vwords], sb[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int key = 16 * kk + 4 * u + (c ^ (u & 1));
        const uint8_t* src = vt + key * G::row + n * (G::row / 8);
        if constexpr (D == 64) w[u][0] = *reinterpret_cast<const uint32_t*>(src);
        else if constexpr (D == 128) { const uint2 x = *reinterpret_cast<const uint2*>(src); w[u][0] = x.x; w[u][1] = x.y; }
        else { const uint4 x = *reinterpret_cast<const uint4*>(src); w[u][0] = x.x; w[u][1] = x.y; w[u][2] = x.z; w[u][3] = x.w; }
        sb[u] = vt[G::codes + key * G::srow + (D == 64 ? n >> 2 : D == 128 ? n >> 1 : n)];
      }
      const uint32_t sa2 = kv4_scale_bits(sb[0]) | kv4_scale_bits(sb[1]) << 16, sb2 = kv4_scale_bits(sb[2]) | kv4_scale_bits(sb[3]) << 16;
      const uint32_t za = kv4_minus24(sa2), zb = kv4_minus24(sb2);
#pragma unroll
      for (int i = 0; i < G::vwords; i++) {
        const uint32_t al = __byte_perm(w[0][i], w[1][i], 0x5410), ah = __byte_perm(w[0][i], w[1][i], 0x7632);
        const uint32_t bl = __byte_perm(w[2][i], w[3][i], 0x5410), bh = __byte_perm(w[2][i], w[3][i], 0x7632);
        mma_16816(o[8 * i + 0], p, kv4_pair<0>(al, sa2, za), kv4_pair<0>(bl, sb2, zb));
        mma_16816(o[8 * i + 1], p, kv4_pair<0>(ah, sa2, za), kv4_pair<0>(bh, sb2, zb));
        mma_16816(o[8 * i + 2], p, kv4_pair<1>(al, sa2, za), kv4_pair<1>(bl, sb2, zb));
        mma_16816(o[8 * i + 3], p, kv4_pair<1>(ah, sa2, za), kv4_pair<1>(bh, sb2, zb));
        mma_16816(o[8 * i + 4], p, kv4_pair<2>(al, sa2, za), kv4_pair<2>(bl, sb2, zb));
        mma_16816(o[8 * i + 5], p, kv4_pair<2>(ah, sa2, za), kv4_pair<2>(bh, sb2, zb));
        mma_16816(o[8 * i + 6], p, kv4_pair<3>(al, sa2, za), kv4_pair<3>(bl, sb2, zb));
        mma_16816(o[8 * i + 7], p, kv4_pair<3>(ah, sa2, za), kv4_pair<3>(bh, sb2, zb));
      }
    }
    __syncwarp();
    if (lane == 0 && tile + ST * W < t_end) fetch(tile + ST * W, slot);
    if (++slot == ST) { slot = 0; phase ^= 1; }
  }

  // join the warps: results and statistics meet in the ring's memory
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) { l0 += __shfl_xor_sync(0xffffffffu, l0, d); l1 += __shfl_xor_sync(0xffffffffu, l1, d); }
  __syncthreads();                                                       // every warp's last tile has been read
  if (s_abort) {                                                         // copies may still be in flight: let them land before the block ends
    if (threadIdx.x == 0) for (int i = 0; i < 2000; i++) __nanosleep(1000);
    __syncthreads();
    return;
  }
  float4* so = reinterpret_cast<float4*>(smem);                          // [W][16][D / 4], a row's quads swizzled within groups of eight
  auto place = [](int row, int f) { return f ^ (((f >> 3) & 3) + 4 * (row & 1)); };
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int i = 0; i < G::nt / 4; i++) {                                // dims (2 c + e) D/8 + 4 i ..
      const int f = (2 * c + e) * (G::nt / 4) + i;
      so[(warp * 16 + r0) * (D / 4) + place(r0, f)] = make_float4(o[4 * i][e], o[4 * i + 1][e], o[4 * i + 2][e], o[4 * i + 3][e]);
      so[(warp * 16 + r1) * (D / 4) + place(r1, f)] = make_float4(o[4 * i][2 + e], o[4 * i + 1][2 + e], o[4 * i + 2][2 + e], o[4 * i + 3][2 + e]);
    }
  if (c == 0) { s_m[warp][r0] = m0; s_m[warp][r1] = m1; s_l[warp][r0] = l0; s_l[warp][r1] = l1; }
  __syncthreads();
  for (int i = threadIdx.x; i < n_tok * gh * (D / 4); i += W * 32) {
    const int r = i / (D / 4), f = i - r * (D / 4);
    float m = -INFINITY, l = 0.f;
    for (int w = 0; w < W; w++) m = fmaxf(m, s_m[w][r]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < W; w++) {
      const float mw = s_m[w][r];
      if (s_l[w][r] == 0.f) continue;                                    // saw no key
      const float x = mw == -INFINITY ? 1.f : exp2f(mw - m);             // -inf: scores that are no numbers, which the sum shows
      const float4 v = so[(w * 16 + r) * (D / 4) + place(r, f)];
      l += x * s_l[w][r];
      acc.x += x * v.x; acc.y += x * v.y; acc.z += x * v.z; acc.w += x * v.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;                          // a NaN stays one
    const long long row = (long long)(tok0 + r / gh) * a.Hq + hkv * a.g + head0 + r % gh;
    if (a.splits == 1) {
      *reinterpret_cast<uint2*>(a.out + row * D + 4 * f) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    } else {
      const long long at = (long long)split * a.T * a.Hq + row;
      *reinterpret_cast<float4*>(a.part + at * D + 4 * f) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      if (f == 0) a.lse2[at] = l == 0.f ? -INFINITY : m + log2f(l);
    }
  }
}

}  // namespace ne

using namespace ne;

namespace {
template <int D, int W, int ST> int launch_i4(const I4Args& a, int tiles, cudaStream_t st) {
  constexpr int ring = W * ST * I4Geo<D>::stage, join = W * 16 * D * 4, smem = ring > join ? ring : join;
  static_assert(smem <= 225 * 1024, "shared memory of a CTA");
  static bool configured[64] = {};                                       // per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(gqa_int4_kernel<D, W, ST>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) configured[dev] = true;
  }
  return (int)launch_pdl(gqa_int4_kernel<D, W, ST>, dim3((unsigned)tiles, (unsigned)(a.Hkv * a.head_tiles), (unsigned)a.splits), dim3(W * 32), smem, st, a);
}
}  // namespace

// q bf16 [T, Hq, D] with rows q_ld elements apart (8-byte aligned); k / v uint8 [num_blocks, Hkv, block_size (D/2 + D/32)].  tiles: an upper bound of the sum over
// sequences of ceil(q_len / tq), tq = max(1, 16 / g).  splits > 1: part / lse2 as ne_attn_merge takes them.
extern "C" int ne_gqa_int4(const void* q, long long q_ld, const void* k, const void* v, int num_blocks, int block_size, const int* block_tables, long long bt_ld, int bt_width,
                           const int* cu_seqlens_q, const int* context_lens, int num_seqs, int T, int Hq, int Hkv, int D, int tiles, int splits, int window, float scale,
                           void* out, float* part, float* lse2, cudaStream_t st) {
  if (T <= 0 || num_seqs <= 0) return 0;
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv || num_blocks < 1 || bt_width < 1 || tiles < 1 || splits < 1 || splits > 65535 || (splits > 1 && (!part || !lse2))) return 1001;
  if (!(block_size == 16 || block_size == 32 || (block_size > 0 && block_size % kTileKeys == 0))) return 1002;
  I4Args a{};
  a.q = (const __nv_bfloat16*)q; a.q_ld = q_ld; a.k = (const uint8_t*)k; a.v = (const uint8_t*)v; a.num_blocks = num_blocks; a.block_size = block_size;
  a.block_tables = block_tables; a.bt_ld = bt_ld; a.bt_width = bt_width; a.cu_seqlens_q = cu_seqlens_q; a.context_lens = context_lens; a.num_seqs = num_seqs;
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.g = Hq / Hkv; a.tq = a.g >= 16 ? 1 : 16 / a.g; a.head_tiles = (a.g + 15) / 16; a.splits = splits;
  a.window = window > 0 ? window : 0; a.scale_log2 = scale * 1.4426950408889634f;
  a.out = (__nv_bfloat16*)out; a.part = part; a.lse2 = lse2;
  if ((long long)Hkv * a.head_tiles > 65535) return 1003;
  switch (D) {
    case 64: return launch_i4<64, 8, 4>(a, tiles, st);
    case 128: return launch_i4<128, 8, 3>(a, tiles, st);
    case 256: return launch_i4<256, 6, 2>(a, tiles, st);
    default: return 1004;
  }
}
