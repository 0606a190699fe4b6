// What lies between a GQA model's qkv projection and its attention, for positions on several axes and for caches held in 4 bits: per-head RMS norm,
// rotation of query and key heads, rows into their cache pages; and 4-bit rows read back as bf16.
//
//   y = x / sqrt(mean x^2 + eps) w ;  pairs (i, i + D/2) of y turned by the angle of position[axis(i)]
//   4 bits, groups of 32 dims:  s = amax / 7 to four significant bits,  c = clamp(rint(y / s), -7, 7) + 8
//
// Bound by HBM: a row is read once and written once (a key or value as D/2 + D/32 bytes).  One warp takes the heads of one token one after the other:
// lane l holds the dims [l E, l E + E), E = D / 32, so that a row is one load per lane, its rotation partner sits in lane l ^ 16, a group of 32
// dims in 32 / E neighbouring lanes, and the cosines and sines are fetched once for all heads.
//
// The key row that is cut to 4 bits is computed in 64 bits: its codes sit on borders, and a sum taken in another order would move some of them.  Value
// rows are bf16, whose quotients are exact or far from a border in 32 bits.  Built without approximate functions.
#include "kv4.cuh"

namespace ne {

constexpr int kRowsWarps = 8;
constexpr double kKv4Most = 7 * 1.875 * 32768;       // largest value of the format

struct RowsArgs {
  const __nv_bfloat16* qkv; long long ld;
  const __nv_bfloat16* qw; const __nv_bfloat16* kw; double eps; float w_offset;
  const long long* positions; long long pos_ld; const float* rope; int max_pos;
  int axes, interleaved, sections[4];
  __nv_bfloat16* q_out; uint8_t* k_cache; uint8_t* v_cache; const long long* slots; long long cache_rows;
  int T, Hq, Hkv, block_size, chunk;                  // chunk: heads of a warp
};

template <int E> struct RowBits { uint32_t u[(E + 1) / 2]; };

template <int E> __device__ __forceinline__ RowBits<E> load_bits(const __nv_bfloat16* p) {
  RowBits<E> r;
  if constexpr (E == 1) r.u[0] = *reinterpret_cast<const uint16_t*>(p);
  else if constexpr (E == 2) r.u[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (E == 4) { const uint2 v = *reinterpret_cast<const uint2*>(p); r.u[0] = v.x; r.u[1] = v.y; }
  else { const uint4 v = *reinterpret_cast<const uint4*>(p); r.u[0] = v.x; r.u[1] = v.y; r.u[2] = v.z; r.u[3] = v.w; }
  return r;
}
template <int E> __device__ __forceinline__ float bits_at(const RowBits<E>& r, int e) {
  return __uint_as_float(e & 1 ? r.u[e >> 1] & 0xffff0000u : r.u[e >> 1] << 16);
}
template <int E> __device__ __forceinline__ void store_bf16(__nv_bfloat16* p, const float (&v)[E]) {
  if constexpr (E == 1) *p = __float2bfloat16(v[0]);
  else {
    uint32_t u[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; i++) u[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    if constexpr (E == 2) *reinterpret_cast<uint32_t*>(p) = u[0];
    else if constexpr (E == 4) *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// norm and rotation of one row in R (float or double); all lanes of the warp
template <int E, typename R> __device__ __forceinline__ void norm_and_turn(R (&x)[E], const __nv_bfloat16* w, double eps, float w_offset, const float (&cs)[E],
                                                                           const float (&sn)[E], int lane) {
  if (w) {
    R ss = 0;
#pragma unroll
    for (int e = 0; e < E; e++) ss += x[e] * x[e];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const R r = rsqrt(ss / (R)(32 * E) + (R)eps);
    const RowBits<E> g = load_bits<E>(w + lane * E);
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = x[e] * r * ((R)bits_at(g, e) + (R)w_offset);
  }
  const bool low = lane < 16;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const R other = __shfl_xor_sync(0xffffffffu, x[e], 16);
    x[e] = low ? x[e] * (R)cs[e] - other * (R)sn[e] : x[e] * (R)cs[e] + other * (R)sn[e];
  }
}

// Scale byte of a group whose largest magnitude is amax, and the scale itself: amax / 7 to four significant bits, ties to even.
__device__ __forceinline__ int kv4_scale_of(double amax, double* s) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(amax / 7.0);
  const long long r = (long long)((u + ((1ull << 48) - 1) + ((u >> 49) & 1)) >> 49) - (1023 - 16) * 8;
  const int b = (int)(r < 0 ? 0 : r > 255 ? 255 : r);
  *s = __longlong_as_double((long long)(b + (1023 - 16) * 8) << 49);
  return b;
}
__device__ __forceinline__ int kv4_scale_of(float amax, float* s) {
  const uint32_t u = __float_as_uint(__fdiv_rn(amax, 7.f));
  const int r = (int)((u + ((1u << 19) - 1) + ((u >> 20) & 1)) >> 20) - (127 - 16) * 8;
  const int b = r < 0 ? 0 : r > 255 ? 255 : r;
  *s = __uint_as_float((uint32_t)(b + (127 - 16) * 8) << 20);
  return b;
}
__device__ __forceinline__ int kv4_code(double x, double s) { return (int)rint(x / s); }
__device__ __forceinline__ int kv4_code(float x, float s) { return (int)rintf(__fdiv_rn(x, s)); }

// one row [32 E] of a head to its place in a 4-bit page; all lanes of the warp
template <int E, typename R> __device__ __forceinline__ void store_kv4(uint8_t* page, int tok, int block_size, R (&x)[E], int lane) {
  R amax = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    x[e] = x[e] != x[e] ? (R)0 : x[e] > (R)kKv4Most ? (R)kKv4Most : x[e] < -(R)kKv4Most ? -(R)kKv4Most : x[e];
    const R m = x[e] < 0 ? -x[e] : x[e];
    amax = m > amax ? m : amax;
  }
#pragma unroll
  for (int o = 16 / E; o > 0; o >>= 1) { const R m = __shfl_xor_sync(0xffffffffu, amax, o); amax = m > amax ? m : amax; }
  R s;
  const int b = kv4_scale_of(amax, &s);
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int c = min(max(kv4_code(x[e], s), -7), 7) + 8, d = (lane * E + e) & 7;
    w |= (uint32_t)c << (4 * ((d >> 1) + 4 * (d & 1)));
  }
#pragma unroll
  for (int o = 4 / E; o > 0; o >>= 1) w |= __shfl_xor_sync(0xffffffffu, w, o);
  constexpr int D = 32 * E;
  if ((lane * E) % 8 == 0) *reinterpret_cast<uint32_t*>(page + tok * (D / 2) + lane * E / 2) = w;
  if ((lane * E) % 32 == 0) page[block_size * (D / 2) + tok * (D / 32) + lane * E / 32] = (uint8_t)b;
}

template <int E, bool kInt4>
__global__ void __launch_bounds__(kRowsWarps * 32) gqa_rows_kernel(const RowsArgs a) {
  pdl_wait(); pdl_trigger();
  constexpr int D = 32 * E;
  const int heads = a.Hq + 2 * a.Hkv, lane = threadIdx.x & 31;
  const int chunks = (heads + a.chunk - 1) / a.chunk;
  const long long w = (long long)blockIdx.x * kRowsWarps + (threadIdx.x >> 5);
  if (w >= (long long)a.T * chunks) return;
  const int t = (int)(w / chunks), h0 = (int)(w - (long long)t * chunks) * a.chunk, h1 = min(h0 + a.chunk, heads);
  const __nv_bfloat16* src = a.qkv + (long long)t * a.ld + lane * E;
  RowBits<E> next = load_bits<E>(src + (long long)h0 * D);
  float cs[E], sn[E];
  if (h0 < a.Hq + a.Hkv) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int i = (lane & 15) * E + e;                                     // angle of the pair (i, i + D/2)
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
  }
  const long long slot = h1 > a.Hq ? a.slots[t] : -1;
  const bool store = slot >= 0 && slot < a.cache_rows && NE_INDEX_OK(slot, BK_CACHE_ROWS, 30, __LINE__);
  long long page = 0; int tok = 0;
  if (kInt4 && store) {
    if (slot < (1ll << 31)) { page = (unsigned)slot / (unsigned)a.block_size; tok = (int)((unsigned)slot % (unsigned)a.block_size); }
    else { page = slot / a.block_size; tok = (int)(slot % a.block_size); }
  }
  for (int h = h0; h < h1; h++) {
    const RowBits<E> now = next;
    if (h + 1 < h1) next = load_bits<E>(src + (long long)(h + 1) * D);
    const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + a.Hkv;
    if (!is_q && !store) break;                                              // keys and values come last: nothing more to do
    float x[E];
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = bits_at(now, e);
    if (is_q) {
      norm_and_turn<E, float>(x, a.qw, a.eps, a.w_offset, cs, sn, lane);
      store_bf16<E>(a.q_out + ((long long)t * a.Hq + h) * D + lane * E, x);
      continue;
    }
    const int kh = is_k ? h - a.Hq : h - a.Hq - a.Hkv;
    uint8_t* cache = is_k ? a.k_cache : a.v_cache;
    if constexpr (kInt4) {
      uint8_t* dst = cache + (page * a.Hkv + kh) * ((long long)a.block_size * (D / 2 + D / 32));
      if (is_k) {
        double y[E];
#pragma unroll
        for (int e = 0; e < E; e++) y[e] = x[e];
        norm_and_turn<E, double>(y, a.kw, a.eps, a.w_offset, cs, sn, lane);
        store_kv4<E, double>(dst, tok, a.block_size, y, lane);
      } else {
        store_kv4<E, float>(dst, tok, a.block_size, x, lane);
      }
    } else {
      if (is_k) norm_and_turn<E, float>(x, a.kw, a.eps, a.w_offset, cs, sn, lane);
      store_bf16<E>(reinterpret_cast<__nv_bfloat16*>(cache) + (slot * a.Hkv + kh) * D + lane * E, x);
    }
  }
}

// Rows of k and v [T, Hkv, D] as they are into 4-bit pages: a warp per (token, head, key or value).
template <int E>
__global__ void __launch_bounds__(kRowsWarps * 32) kv4_store_kernel(const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, long long k_ld, long long v_ld,
                                                                   uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache, const long long* __restrict__ slots,
                                                                   long long cache_rows, int T, int Hkv, int block_size) {
  pdl_wait(); pdl_trigger();
  constexpr int D = 32 * E;
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * kRowsWarps + (threadIdx.x >> 5);
  if (w >= (long long)T * 2 * Hkv) return;
  const int t = (int)(w / (2 * Hkv)), r = (int)(w - (long long)t * 2 * Hkv), h = r >> 1;
  const long long slot = slots[t];
  if (slot < 0 || slot >= cache_rows || !NE_INDEX_OK(slot, BK_CACHE_ROWS, 30, __LINE__)) return;
  const RowBits<E> bits = load_bits<E>((r & 1 ? v + (long long)t * v_ld : k + (long long)t * k_ld) + h * D + lane * E);
  float x[E];
#pragma unroll
  for (int e = 0; e < E; e++) x[e] = bits_at(bits, e);
  store_kv4<E, float>((r & 1 ? v_cache : k_cache) + (slot / block_size * Hkv + h) * ((long long)block_size * (D / 2 + D / 32)), (int)(slot % block_size), block_size, x, lane);
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
  for (int i = threadIdx.x; i < 64 * words; i += 256) {
    const int r = i / words, j = i - r * words, key = p * 64 + r;
    uint4 kv = make_uint4(0, 0, 0, 0), vv = kv;
    if (key < n) {
      const int id = tables[(long long)seq * bt_ld + key / block_size], tok = key % block_size;
      if (id >= 0 && id < num_blocks && NE_INDEX_OK(id, BK_CACHE_PAGES, 30, __LINE__)) {
        const long long base = ((long long)id * Hkv + h) * ((long long)block_size * (D / 2 + D / 32));
        const long long code = base + tok * (D / 2) + 4 * j, scale = base + block_size * (D / 2) + tok * (D / 32) + j / 4;
        kv = kv4_word(*reinterpret_cast<const uint32_t*>(k_cache + code), k_cache[scale]);
        vv = kv4_word(*reinterpret_cast<const uint32_t*>(v_cache + code), v_cache[scale]);
      }
    }
    const long long dst = ((at * 64 + r) * Hkv + h) * D + 8 * j;
    *reinterpret_cast<uint4*>(k_out + dst) = kv;
    *reinterpret_cast<uint4*>(v_out + dst) = vv;
  }
}

}  // namespace ne

using namespace ne;

namespace {
template <int E> cudaError_t launch_rows(const RowsArgs& a, bool int4, cudaStream_t st) {
  const long long warps = (long long)a.T * ((a.Hq + 2 * a.Hkv + a.chunk - 1) / a.chunk);
  const dim3 grid((unsigned)((warps + kRowsWarps - 1) / kRowsWarps));
  return int4 ? launch_pdl(gqa_rows_kernel<E, true>, grid, dim3(kRowsWarps * 32), 0, st, a) : launch_pdl(gqa_rows_kernel<E, false>, grid, dim3(kRowsWarps * 32), 0, st, a);
}
}  // namespace

// qkv bf16 [T, (Hq + 2 Hkv) D], rows ld apart and aligned to 2 D / 32 bytes; positions int64 [axes, T], rows pos_ld apart; rope fp32 [max_pos, D] (cos | sin);
// caches: int4 != 0: uint8 [blocks, Hkv, block_size (D/2 + D/32)], else bf16 [blocks, block_size, Hkv, D].  chunk: heads a warp takes one after the other.
extern "C" int ne_gqa_rows(const void* qkv, long long ld, int Hq, int Hkv, int D, const void* qw, const void* kw, double eps, float w_offset, const long long* positions,
                           long long pos_ld, const float* rope, int max_pos, int axes, const int* sections, int interleaved, void* q_out, void* k_cache, void* v_cache,
                           const long long* slots, long long cache_rows, int block_size, int int4, int chunk, int T, cudaStream_t st) {
  if (T <= 0) return 0;
  if (Hq < 0 || Hkv < 1 || axes < 1 || axes > 4 || max_pos < 1 || block_size < 1 || chunk < 1) return 1001;
  RowsArgs a{};
  a.qkv = (const __nv_bfloat16*)qkv; a.ld = ld; a.qw = (const __nv_bfloat16*)qw; a.kw = (const __nv_bfloat16*)kw; a.eps = eps; a.w_offset = w_offset;
  a.positions = positions; a.pos_ld = pos_ld; a.rope = rope; a.max_pos = max_pos; a.axes = axes; a.interleaved = interleaved;
  for (int i = 0; i < axes; i++) a.sections[i] = sections[i];
  a.q_out = (__nv_bfloat16*)q_out; a.k_cache = (uint8_t*)k_cache; a.v_cache = (uint8_t*)v_cache; a.slots = slots; a.cache_rows = cache_rows;
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.block_size = block_size; a.chunk = chunk;
  switch (D) {
    case 32: return (int)launch_rows<1>(a, int4, st);
    case 64: return (int)launch_rows<2>(a, int4, st);
    case 128: return (int)launch_rows<4>(a, int4, st);
    case 256: return (int)launch_rows<8>(a, int4, st);
    default: return 1002;
  }
}

extern "C" int ne_kv4_store(const void* k, const void* v, long long k_ld, long long v_ld, void* k_cache, void* v_cache, const long long* slots, long long cache_rows, int T,
                            int Hkv, int D, int block_size, cudaStream_t st) {
  if (T <= 0) return 0;
  if (Hkv < 1 || block_size < 1) return 1001;
  const dim3 grid((unsigned)(((long long)T * 2 * Hkv + kRowsWarps - 1) / kRowsWarps));
  auto go = [&](auto kern) {
    return (int)launch_pdl(kern, grid, dim3(kRowsWarps * 32), 0, st, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, k_ld, v_ld, (uint8_t*)k_cache, (uint8_t*)v_cache, slots,
                           cache_rows, T, Hkv, block_size);
  };
  switch (D) {
    case 32: return go(kv4_store_kernel<1>);
    case 64: return go(kv4_store_kernel<2>);
    case 128: return go(kv4_store_kernel<4>);
    case 256: return go(kv4_store_kernel<8>);
    default: return 1002;
  }
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
