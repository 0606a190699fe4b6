// What lies between a GQA model's qkv projection and its attention, for positions on several axes and for caches held in 4 bits: per-head RMS norm,
// rotation of query and key heads, rows into their cache pages; and 4-bit rows read back as bf16.
//
//   y = x / sqrt(mean x^2 + eps) w ;  pairs (i, i + D/2) of y turned by the angle of position[axis(i)]
//   4 bits, groups of 32 dims:  s = amax / 7 to four significant bits,  c = clamp(rint(y / s), -7, 7) + 8
//
// Bound by HBM: a row is read once and written once (a key or value as D/2 + D/32 bytes).  A lane holds four dims of the lower half of a row and their
// partners in the upper half, so that a rotation stays in the lane; D / 8 lanes share a row, a warp takes 256 / D heads of one token at a time.  Query rows
// go in batches of four such steps, loaded before the first is used, under one fetch of cosines and sines.
//
// The key row that is cut to 4 bits is computed in 64 bits: its codes sit on borders, and a sum taken in another order would move some of them.  Value
// rows are bf16, whose quotients are exact or far from a border in 32 bits.  Built without approximate functions.
#include "kv4.cuh"

namespace ne {

constexpr int kRowsWarps = 8;
constexpr int kRowsBatch = 4;                         // steps of query rows in flight
constexpr double kKv4Most = 7 * 1.875 * 32768;       // largest value of the format

struct RowsArgs {
  const __nv_bfloat16* qkv; long long ld;
  const __nv_bfloat16* qw; const __nv_bfloat16* kw; double eps; float w_offset;
  const long long* positions; long long pos_ld; const float* rope; int max_pos;
  int axes, interleaved, sections[4];
  __nv_bfloat16* q_out; uint8_t* k_cache; uint8_t* v_cache; const long long* slots; long long cache_rows;
  int T, Hq, Hkv, block_size, chunk;                  // chunk: steps of query rows a warp takes
};

// a lane's dims of a row: [4 l, 4 l + 4) and their partners half a row further
struct RowBits { uint2 lo, hi; };
template <int L> __device__ __forceinline__ RowBits load_row(const __nv_bfloat16* row, int l) {
  return {*reinterpret_cast<const uint2*>(row + 4 * l), *reinterpret_cast<const uint2*>(row + 4 * L + 4 * l)};
}
__device__ __forceinline__ void unpack_row(const RowBits& b, float (&x)[8]) {
  const uint32_t u[4] = {b.lo.x, b.lo.y, b.hi.x, b.hi.y};
#pragma unroll
  for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(u[i] << 16); x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
}
template <int L> __device__ __forceinline__ void store_row(__nv_bfloat16* row, int l, const float (&x)[8]) {
  *reinterpret_cast<uint2*>(row + 4 * l) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
  *reinterpret_cast<uint2*>(row + 4 * L + 4 * l) = make_uint2(pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

// norm and rotation of one row in R (float or double), by its L lanes
template <int L, typename R> __device__ __forceinline__ void norm_and_turn(R (&x)[8], const RowBits& w, bool norm, double eps, float w_offset, const float (&cs)[4],
                                                                           const float (&sn)[4]) {
  if (norm) {
    R ss = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) ss += x[e] * x[e];
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const R r = rsqrt(ss / (R)(8 * L) + (R)eps);
    float g[8];
    unpack_row(w, g);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = x[e] * r * ((R)g[e] + (R)w_offset);
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const R a = x[e], b = x[4 + e];
    x[e] = a * (R)cs[e] - b * (R)sn[e];
    x[4 + e] = b * (R)cs[e] + a * (R)sn[e];
  }
}

// Scale byte of a group whose largest magnitude is amax: the nearest scale to amax / 7, ties to the even byte, and the scale itself.  A first guess in 32 bits is
// corrected by comparing amax with seven times the midpoints, products of few bits that are exact.
__device__ __forceinline__ float kv4_scale_value(int b) { return __uint_as_float((uint32_t)(b + (127 - 16) * 8) << 20); }
template <typename R> __device__ __forceinline__ int kv4_scale_of(R amax, float* s) {
  const uint32_t u = __float_as_uint(__fdiv_rn((float)amax, 7.f));
  int b = (int)((u + (1u << 19)) >> 20) - (127 - 16) * 8;
  b = min(max(b, 0), 255);
  const float lo = kv4_scale_value(max(b - 1, 0)), at = kv4_scale_value(b), hi = kv4_scale_value(min(b + 1, 255));
  const R up = (R)3.5 * ((R)at + (R)hi), down = (R)3.5 * ((R)lo + (R)at);
  if (b < 255 && (amax > up || (amax == up && (b & 1)))) b++;
  else if (b > 0 && (amax < down || (amax == down && (b & 1)))) b--;
  *s = kv4_scale_value(b);
  return b;
}
// The nearest multiple of s, ties to even, from -7 to 7: by a product with the reciprocal, corrected with the exact remainder.
__device__ __forceinline__ int kv4_code(float x, float s, float inv) {
  const float t = fmaf(x, inv, 12582912.f);
  int q = __float_as_int(t) - 0x4B400000;
  const float r = fmaf(-(t - 12582912.f), s, x), h = 0.5f * s;
  if (r > h || (r == h && (q & 1))) q++;
  else if (r < -h || (r == -h && (q & 1))) q--;
  return min(max(q, -7), 7);
}
__device__ __forceinline__ int kv4_code(double x, float sf, float inv) {
  const double s = sf, t = fma(x, (double)inv, 6755399441055744.0);
  int q = __double2loint(t);
  const double r = fma(-(t - 6755399441055744.0), s, x), h = 0.5 * s;
  if (r > h || (r == h && (q & 1))) q++;
  else if (r < -h || (r == -h && (q & 1))) q--;
  return min(max(q, -7), 7);
}

// one row [8 L] of a head to its place in a 4-bit page, by its L lanes (all lanes of the warp call; those without a row pass store = false)
template <int L, typename R> __device__ __forceinline__ void store_kv4(uint8_t* page, int tok, int block_size, R (&x)[8], int l, bool store) {
  constexpr int D = 8 * L;
  R m0 = 0, m1 = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    x[e] = x[e] != x[e] ? (R)0 : x[e] > (R)kKv4Most ? (R)kKv4Most : x[e] < -(R)kKv4Most ? -(R)kKv4Most : x[e];
    const R m = x[e] < 0 ? -x[e] : x[e];
    if (e < 4) m0 = m > m0 ? m : m0; else m1 = m > m1 ? m : m1;
  }
  if (L == 4) m0 = m1 = m0 > m1 ? m0 : m1;                               // one group of 32: both halves
#pragma unroll
  for (int o = L == 4 ? 2 : 4; o > 0; o >>= 1) {
    const R a = __shfl_xor_sync(0xffffffffu, m0, o), b = L == 4 ? a : __shfl_xor_sync(0xffffffffu, m1, o);
    m0 = a > m0 ? a : m0;
    m1 = b > m1 ? b : m1;
  }
  float s0, s1;
  const int b0 = kv4_scale_of(m0, &s0), b1 = L == 4 ? b0 : kv4_scale_of(m1, &s1);
  if (L == 4) s1 = s0;
  const float i0 = __fdiv_rn(1.f, s0), i1 = L == 4 ? i0 : __fdiv_rn(1.f, s1);
  int c[8];
#pragma unroll
  for (int e = 0; e < 8; e++) c[e] = kv4_code(x[e], e < 4 ? s0 : s1, e < 4 ? i0 : i1) + 8;
  // four dims of a word of eight: even places in one byte of the low half, odd ones in one of the high half
  const int sh = 8 * (l & 1);
  const uint32_t w0 = (uint32_t)(c[0] | c[2] << 4) << sh | (uint32_t)(c[1] | c[3] << 4) << (16 + sh);
  const uint32_t w1 = (uint32_t)(c[4] | c[6] << 4) << sh | (uint32_t)(c[5] | c[7] << 4) << (16 + sh);
  const uint32_t other = __shfl_xor_sync(0xffffffffu, l & 1 ? w0 : w1, 1);
  if (!store) return;
  // even lanes write the word of the lower half, odd lanes that of the upper half
  *reinterpret_cast<uint32_t*>(page + tok * (D / 2) + (l & 1 ? D / 4 : 0) + (l >> 1) * 4) = (l & 1 ? w1 : w0) | other;
  if (l % 8 < (L == 4 ? 1 : 2)) page[block_size * (D / 2) + tok * (D / 32) + (l & 1 ? D / 64 : 0) + (l >> 3)] = (uint8_t)(l & 1 ? b1 : b0);
}

__device__ __forceinline__ void split_slot(long long slot, int block_size, long long& page, int& tok) {
  if (slot < (1ll << 31)) { page = (unsigned)slot / (unsigned)block_size; tok = (int)((unsigned)slot % (unsigned)block_size); }
  else { page = slot / block_size; tok = (int)(slot % block_size); }
}

// A warp takes `chunk` steps of a token's query heads, or one step of its key heads, or of its value heads; a step is the heads of 32 / L rows.
template <int L, bool kInt4>
__global__ void __launch_bounds__(kRowsWarps * 32) gqa_rows_kernel(const RowsArgs a) {
  pdl_wait(); pdl_trigger();
  constexpr int D = 8 * L, R = 32 / L;
  const int lane = threadIdx.x & 31, l = lane % L, sub = lane / L;
  const int q_steps = (a.Hq + R - 1) / R, kv_steps = (a.Hkv + R - 1) / R, q_warps = (q_steps + a.chunk - 1) / a.chunk, per_token = q_warps + 2 * kv_steps;
  const long long w = (long long)blockIdx.x * kRowsWarps + (threadIdx.x >> 5);
  if (w >= (long long)a.T * per_token) return;
  const int t = (int)(w / per_token), part = (int)(w - (long long)t * per_token);
  const __nv_bfloat16* src = a.qkv + (long long)t * a.ld;
  const bool is_q = part < q_warps, is_v = part >= q_warps + kv_steps;
  float cs[4], sn[4];
  auto angles = [&] {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = 4 * l + e;                                               // angle of the pair (i, i + D/2)
      int ax = 0;
      if (a.axes > 1) {
        if (a.interleaved) {
          const int r = i % a.axes;
          ax = r > 0 && i < a.axes * (r == 1 ? a.sections[1] : r == 2 ? a.sections[2] : a.sections[3]) ? r : 0;
        } else {
          int end = a.sections[0];
          for (ax = 0; ax + 1 < a.axes && i >= end; ax++) end += ax == 0 ? a.sections[1] : ax == 1 ? a.sections[2] : a.sections[3];
        }
      }
      long long pos = a.positions[(long long)ax * a.pos_ld + t];
      pos = pos < 0 ? 0 : pos >= a.max_pos ? a.max_pos - 1 : pos;            // never outside the table
      cs[e] = a.rope[pos * D + i];
      sn[e] = a.rope[pos * D + D / 2 + i];
    }
  };
  if (is_q) {
    RowBits next[kRowsBatch];
    const int s0 = part * a.chunk, s1 = min(s0 + a.chunk, q_steps);
#pragma unroll
    for (int i = 0; i < kRowsBatch; i++) {
      const int h = (s0 + i) * R + sub;
      if (s0 + i < s1 && h < a.Hq) next[i] = load_row<L>(src + (long long)h * D, l); else next[i] = {make_uint2(0, 0), make_uint2(0, 0)};
    }
    RowBits g = {make_uint2(0, 0), make_uint2(0, 0)};
    if (a.qw) g = load_row<L>(a.qw, l);
    angles();
    for (int s = s0; s < s1; s += kRowsBatch) {
      RowBits now[kRowsBatch];
#pragma unroll
      for (int i = 0; i < kRowsBatch; i++) {
        now[i] = next[i];
        const int h = (s + kRowsBatch + i) * R + sub;
        if (s + kRowsBatch + i < s1 && h < a.Hq) next[i] = load_row<L>(src + (long long)h * D, l);
      }
#pragma unroll
      for (int i = 0; i < kRowsBatch; i++) {
        if (s + i >= s1) break;
        float x[8];
        unpack_row(now[i], x);
        norm_and_turn<L, float>(x, g, a.qw != nullptr, a.eps, a.w_offset, cs, sn);
        const int h = (s + i) * R + sub;
        if (h < a.Hq) store_row<L>(a.q_out + ((long long)t * a.Hq + h) * D, l, x);
      }
    }
    return;
  }
  const long long slot = a.slots[t];
  if (slot < 0 || slot >= a.cache_rows || !NE_INDEX_OK(slot, BK_CACHE_ROWS, 30, __LINE__)) return;
  const int h = (part - q_warps - (is_v ? kv_steps : 0)) * R + sub;
  const bool live = h < a.Hkv;
  RowBits bits = {make_uint2(0, 0), make_uint2(0, 0)}, g = bits;
  if (live) bits = load_row<L>(src + (long long)(a.Hq + (is_v ? a.Hkv : 0) + h) * D, l);
  if (!is_v) {
    if (a.kw) g = load_row<L>(a.kw, l);
    angles();
  }
  float x[8];
  unpack_row(bits, x);
  uint8_t* cache = is_v ? a.v_cache : a.k_cache;
  if constexpr (kInt4) {
    long long page; int tok;
    split_slot(slot, a.block_size, page, tok);
    uint8_t* dst = cache + (page * a.Hkv + (live ? h : 0)) * ((long long)a.block_size * (D / 2 + D / 32));
    if (is_v) {
      store_kv4<L, float>(dst, tok, a.block_size, x, l, live);
    } else {
      double y[8];
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = x[e];
      norm_and_turn<L, double>(y, g, a.kw != nullptr, a.eps, a.w_offset, cs, sn);
      store_kv4<L, double>(dst, tok, a.block_size, y, l, live);
    }
  } else {
    if (!is_v) norm_and_turn<L, float>(x, g, a.kw != nullptr, a.eps, a.w_offset, cs, sn);
    if (live) store_row<L>(reinterpret_cast<__nv_bfloat16*>(cache) + (slot * a.Hkv + h) * D, l, x);
  }
}

// Rows of k and v [T, Hkv, D] as they are into 4-bit pages: a warp per (token, step of heads, key or value).
template <int L>
__global__ void __launch_bounds__(kRowsWarps * 32) kv4_store_kernel(const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, long long k_ld, long long v_ld,
                                                                   uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache, const long long* __restrict__ slots,
                                                                   long long cache_rows, int T, int Hkv, int block_size) {
  pdl_wait(); pdl_trigger();
  constexpr int D = 8 * L, R = 32 / L;
  const int lane = threadIdx.x & 31, l = lane % L, steps = (Hkv + R - 1) / R;
  const long long w = (long long)blockIdx.x * kRowsWarps + (threadIdx.x >> 5);
  if (w >= (long long)T * 2 * steps) return;
  const int t = (int)(w / (2 * steps)), r = (int)(w - (long long)t * 2 * steps), h = (r >> 1) * R + lane / L;
  const long long slot = slots[t];
  if (slot < 0 || slot >= cache_rows || !NE_INDEX_OK(slot, BK_CACHE_ROWS, 30, __LINE__)) return;
  const bool live = h < Hkv;
  RowBits bits = {make_uint2(0, 0), make_uint2(0, 0)};
  if (live) bits = load_row<L>((r & 1 ? v + (long long)t * v_ld : k + (long long)t * k_ld) + h * D, l);
  float x[8];
  unpack_row(bits, x);
  long long page; int tok;
  split_slot(slot, block_size, page, tok);
  store_kv4<L, float>((r & 1 ? v_cache : k_cache) + (page * Hkv + (live ? h : 0)) * ((long long)block_size * (D / 2 + D / 32)), tok, block_size, x, l, live);
}

// 4-bit rows as bf16 [T, Hkv, D]: a thread per word of 8 dims of a key and a value row.  Slots outside the cache give zeros.
__global__ void __launch_bounds__(256) kv4_gather_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const long long* __restrict__ slots,
                                                        long long cache_rows, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int T, int Hkv, int D,
                                                        int block_size) {
  pdl_wait(); pdl_trigger();
  const int words = D / 8;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)T * Hkv * words) return;
  const int t = (int)(i / (Hkv * words)), r = (int)(i - (long long)t * Hkv * words), h = r / words, j = r - h * words;
  const long long slot = slots[t];
  uint4 kv = make_uint4(0, 0, 0, 0), vv = kv;
  if (slot >= 0 && slot < cache_rows && NE_INDEX_OK(slot, BK_CACHE_ROWS, 30, __LINE__)) {
    const int tok = (int)(slot % block_size);
    const long long base = (slot / block_size * Hkv + h) * ((long long)block_size * (D / 2 + D / 32));
    const long long code = base + tok * (D / 2) + 4 * j, scale = base + block_size * (D / 2) + tok * (D / 32) + j / 4;
    kv = kv4_word(*reinterpret_cast<const uint32_t*>(k_cache + code), k_cache[scale]);
    vv = kv4_word(*reinterpret_cast<const uint32_t*>(v_cache + code), v_cache[scale]);
  }
  *reinterpret_cast<uint4*>(k_out + i * 8) = kv;
  *reinterpret_cast<uint4*>(v_out + i * 8) = vv;
}

// The contexts of all sequences as bf16 pages of 64 tokens of their own, [B * width, 64, Hkv, D], page p of sequence i at i * width + p, with that table and
// the context lengths (cut off where their block tables end).  Pages outside the cache read as zeros, and so do keys behind a context that share a page
// with it; pages behind a context are left out.
__global__ void __launch_bounds__(256) kv4_expand_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, int num_blocks,
                                                        const int* __restrict__ tables, long long bt_ld, int bt_width, const int* __restrict__ ctx,
                                                        __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int* __restrict__ out_tables,
                                                        int* __restrict__ out_ctx, int width, int Hkv, int D, int block_size) {
  pdl_wait(); pdl_trigger();
  const int seq = blockIdx.y, p = blockIdx.x, h = blockIdx.z;
  const long long at = (long long)seq * width + p;
  const int n = (int)min((long long)ctx[seq], (long long)bt_width * block_size);
  if (h == 0 && threadIdx.x == 0) {
    out_tables[at] = (int)at;
    if (p == 0) out_ctx[seq] = n;
  }
  if (p * 64 >= n) return;
  const int words = D / 8;
  constexpr int kFlight = 4;                                             // words of a thread in flight
  for (int i0 = threadIdx.x; i0 < 64 * words; i0 += 256 * kFlight) {
    uint32_t kw[kFlight], vw[kFlight], ks[kFlight], vs[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; u++) {
      const int i = i0 + u * 256, r = i / words, j = i - r * words, key = p * 64 + r;
      kw[u] = vw[u] = 0x88888888u;                                       // zeros
      ks[u] = vs[u] = 0;
      if (r < 64 && key < n) {
        const int id = tables[(long long)seq * bt_ld + key / block_size], tok = key % block_size;
        if (id >= 0 && id < num_blocks && NE_INDEX_OK(id, BK_CACHE_PAGES, 30, __LINE__)) {
          const long long base = ((long long)id * Hkv + h) * ((long long)block_size * (D / 2 + D / 32));
          const long long code = base + tok * (D / 2) + 4 * j, scale = base + block_size * (D / 2) + tok * (D / 32) + j / 4;
          kw[u] = *reinterpret_cast<const uint32_t*>(k_cache + code); ks[u] = k_cache[scale];
          vw[u] = *reinterpret_cast<const uint32_t*>(v_cache + code); vs[u] = v_cache[scale];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kFlight; u++) {
      const int i = i0 + u * 256, r = i / words, j = i - r * words;
      if (r >= 64) break;
      const long long dst = ((at * 64 + r) * Hkv + h) * D + 8 * j;
      *reinterpret_cast<uint4*>(k_out + dst) = kv4_word(kw[u], ks[u]);
      *reinterpret_cast<uint4*>(v_out + dst) = kv4_word(vw[u], vs[u]);
    }
  }
}

}  // namespace ne

using namespace ne;

namespace {
template <int L> int launch_rows(const RowsArgs& a, bool int4, cudaStream_t st) {
  constexpr int R = 32 / L;
  const int q_steps = (a.Hq + R - 1) / R, kv_steps = (a.Hkv + R - 1) / R;
  const long long warps = (long long)a.T * ((q_steps + a.chunk - 1) / a.chunk + 2 * kv_steps);
  const dim3 grid((unsigned)((warps + kRowsWarps - 1) / kRowsWarps));
  return (int)(int4 ? launch_pdl(gqa_rows_kernel<L, true>, grid, dim3(kRowsWarps * 32), 0, st, a) : launch_pdl(gqa_rows_kernel<L, false>, grid, dim3(kRowsWarps * 32), 0, st, a));
}
}  // namespace

// qkv bf16 [T, (Hq + 2 Hkv) D], rows ld apart and aligned to 8 bytes; positions int64 [axes, T], rows pos_ld apart; rope fp32 [max_pos, D] (cos | sin);
// caches: int4 != 0: uint8 [blocks, Hkv, block_size (D/2 + D/32)], else bf16 [blocks, block_size, Hkv, D].
extern "C" int ne_gqa_rows(const void* qkv, long long ld, int Hq, int Hkv, int D, const void* qw, const void* kw, double eps, float w_offset, const long long* positions,
                           long long pos_ld, const float* rope, int max_pos, int axes, const int* sections, int interleaved, void* q_out, void* k_cache, void* v_cache,
                           const long long* slots, long long cache_rows, int block_size, int int4, int T, cudaStream_t st) {
  if (T <= 0) return 0;
  if (Hq < 0 || Hkv < 1 || axes < 1 || axes > 4 || max_pos < 1 || block_size < 1) return 1001;
  RowsArgs a{};
  a.qkv = (const __nv_bfloat16*)qkv; a.ld = ld; a.qw = (const __nv_bfloat16*)qw; a.kw = (const __nv_bfloat16*)kw; a.eps = eps; a.w_offset = w_offset;
  a.positions = positions; a.pos_ld = pos_ld; a.rope = rope; a.max_pos = max_pos; a.axes = axes; a.interleaved = interleaved;
  for (int i = 0; i < axes; i++) a.sections[i] = sections[i];
  a.q_out = (__nv_bfloat16*)q_out; a.k_cache = (uint8_t*)k_cache; a.v_cache = (uint8_t*)v_cache; a.slots = slots; a.cache_rows = cache_rows;
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.block_size = block_size;
  // few rows: a warp per step, so that all SMs work; many: eight steps under one fetch of the angles
  a.chunk = (long long)T * Hq * D >= 148ll * 64 * 256 * 4 ? 8 : 1;
  switch (D) {
    case 32: return launch_rows<4>(a, int4, st);
    case 64: return launch_rows<8>(a, int4, st);
    case 128: return launch_rows<16>(a, int4, st);
    case 256: return launch_rows<32>(a, int4, st);
    default: return 1002;
  }
}

extern "C" int ne_kv4_store(const void* k, const void* v, long long k_ld, long long v_ld, void* k_cache, void* v_cache, const long long* slots, long long cache_rows, int T,
                            int Hkv, int D, int block_size, cudaStream_t st) {
  if (T <= 0) return 0;
  if (Hkv < 1 || block_size < 1 || (D != 32 && D != 64 && D != 128 && D != 256)) return 1001;
  const int per_step = 256 / D, steps = (Hkv + per_step - 1) / per_step;
  const dim3 grid((unsigned)(((long long)T * 2 * steps + kRowsWarps - 1) / kRowsWarps));
  auto go = [&](auto kern) {
    return (int)launch_pdl(kern, grid, dim3(kRowsWarps * 32), 0, st, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, k_ld, v_ld, (uint8_t*)k_cache, (uint8_t*)v_cache, slots,
                           cache_rows, T, Hkv, block_size);
  };
  return D == 32 ? go(kv4_store_kernel<4>) : D == 64 ? go(kv4_store_kernel<8>) : D == 128 ? go(kv4_store_kernel<16>) : go(kv4_store_kernel<32>);
}

extern "C" int ne_kv4_gather(const void* k_cache, const void* v_cache, const long long* slots, long long cache_rows, void* k_out, void* v_out, int T, int Hkv, int D,
                             int block_size, cudaStream_t st) {
  if (T <= 0) return 0;
  if (Hkv < 1 || block_size < 1 || D < 32 || D % 32) return 1001;
  const long long n = (long long)T * Hkv * (D / 8);
  return (int)launch_pdl(kv4_gather_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, (const uint8_t*)k_cache, (const uint8_t*)v_cache, slots, cache_rows,
                         (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, T, Hkv, D, block_size);
}

// width: pages of 64 tokens per sequence, at least ceil(bt_width * block_size / 64)
extern "C" int ne_kv4_expand(const void* k_cache, const void* v_cache, int num_blocks, const int* tables, long long bt_ld, int bt_width, const int* ctx, int seqs, int width,
                             void* k_out, void* v_out, int* out_tables, int* out_ctx, int Hkv, int D, int block_size, cudaStream_t st) {
  if (seqs <= 0 || width <= 0) return 0;
  if (num_blocks < 1 || Hkv < 1 || block_size < 1 || D < 32 || D % 32 || seqs > 65535 || Hkv > 65535 || (long long)width * 64 < (long long)bt_width * block_size ||
      (long long)seqs * width >= (1ll << 31)) return 1001;
  return (int)launch_pdl(kv4_expand_kernel, dim3((unsigned)width, (unsigned)seqs, (unsigned)Hkv), dim3(256), 0, st, (const uint8_t*)k_cache, (const uint8_t*)v_cache, num_blocks,
                         tables, bt_ld, bt_width, ctx, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, out_tables, out_ctx, width, Hkv, D, block_size);
}
