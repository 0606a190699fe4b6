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
// The codes of a key row are those of the row in 64 bits, whatever order its norm is summed in: it is computed in 32 bits with a bound of its error, and where
// an element or a scale lies nearer to a border than that (one step of two rows in a hundred), its warp computes it again in 64.  Value rows are bf16,
// whose quotients are exact or far from a border in 32 bits.  Built without approximate functions.
//
// Measured (B200, us, calls in a graph over inputs larger than L2; bytes at 6540 GB/s): 64 / 4 heads of 128 into 4 bits, three axes: 128 tokens 5.0, 4096: 39 (22), one
// position: 34; 16 / 2 of 256: 26 (12); 32 / 8 heads into bf16, three axes: 4096: 24 (15); bound there by the chain position, table row, rotation of few resident warps: eight CTAs
// per SM cap them at 64 registers, where the 4-bit forms spill 172 to 184 bytes (the 64-bit pass of key rows), the bf16 ones 16 to 44.  Rows stored as they are: 4096
// of 8 heads of 128: 19 (3.2), of 2 heads of 256: 10 (1.6); read back: 6.5 and 3.9.  Expanding 32 x 4096 keys of 4 heads: 79 (52): a page's rows are found behind a barrier,
// codes come as 4 bytes and scales as single ones.
#include "kv4.cuh"

namespace ne {

constexpr int kRowsWarps = 4;
constexpr int kRowsBatch = 4;                         // steps of query rows in flight
constexpr double kKv4Most = 7 * 1.875 * 32768;       // largest value of the format

struct RowsArgs {
  const __nv_bfloat16* qkv; long long ld;
  const __nv_bfloat16* qw; const __nv_bfloat16* kw; double eps; float w_offset;
  const long long* positions; long long pos_ld; const float* rope; int max_pos;
  int axes, interleaved, sections[4];
  __nv_bfloat16* q_out; uint8_t* k_cache; uint8_t* v_cache; const long long* slots; long long cache_rows;
  int T, Hq, Hkv, block_size, chunk, kv_chunk;        // steps of query rows, of key or value rows, that a warp takes
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

// What a row is turned by, with its norm weights: lower half a w_a cos - b w_b sin, upper half b w_b cos + a w_a sin
template <typename R> struct Turn { R ca[4], sb[4], cb[4], sa[4]; };
template <typename R> __device__ __forceinline__ void make_turn(Turn<R>& t, const RowBits& w, float w_offset, const float (&cs)[4], const float (&sn)[4]) {
  float g[8];
  unpack_row(w, g);
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const R ga = (R)g[e] + (R)w_offset, gb = (R)g[4 + e] + (R)w_offset, c = cs[e], s = sn[e];
    t.ca[e] = ga * c; t.sa[e] = ga * s; t.cb[e] = gb * c; t.sb[e] = gb * s;
  }
}
// norm and rotation of one row in R (float or double), by its L lanes
template <int L, typename R> __device__ __forceinline__ void norm_and_turn(R (&x)[8], const Turn<R>& t, bool norm, R eps, float* off = nullptr) {
  R ss = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) ss += x[e] * x[e];
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const R mean = ss / (R)(8 * L) + eps, r = norm ? rsqrt(mean) : (R)1;
  const bool lost = norm && !(mean > (R)1e-30 && mean < (R)1e37);        // squares that 32 bits do not hold: no bound
  // Error in 32 bits, relative to the sum of the two magnitudes, in units of 2^-24: 8 of the mean (a product, 13 additions, eps rounded and added: 16, halved by the
  // root), 4 of the root (two units in the last place), one each for the weight, its factor, the product, the sum and the scaling: 17.  20 are taken: the rest
  // is for the products of errors and for the roundings of `off` itself
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const R a = x[e], b = x[4 + e];
    x[e] = r * (a * t.ca[e] - b * t.sb[e]);
    x[4 + e] = r * (b * t.cb[e] + a * t.sa[e]);
    if (off) {
      off[e] = lost ? INFINITY : (float)(r * (fabs(a * t.ca[e]) + fabs(b * t.sb[e]))) * 0x1.4p-20f;
      off[4 + e] = lost ? INFINITY : (float)(r * (fabs(b * t.cb[e]) + fabs(a * t.sa[e]))) * 0x1.4p-20f;
    }
  }
}

// The same for query rows, two elements an instruction
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 f2(float a, float b) { f32x2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float2 un2(f32x2 v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
struct Turn2 { f32x2 ca[2], nsb[2], cb[2], sa[2]; };
__device__ __forceinline__ Turn2 pair_turn(const Turn<float>& t) {
  Turn2 p;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    p.ca[i] = f2(t.ca[2 * i], t.ca[2 * i + 1]); p.nsb[i] = f2(-t.sb[2 * i], -t.sb[2 * i + 1]);
    p.cb[i] = f2(t.cb[2 * i], t.cb[2 * i + 1]); p.sa[i] = f2(t.sa[2 * i], t.sa[2 * i + 1]);
  }
  return p;
}
template <int L> __device__ __forceinline__ void query_row(const RowBits& bits, __nv_bfloat16* row, int l, bool store, const Turn2& t, bool norm, float eps) {
  const uint32_t u[4] = {bits.lo.x, bits.lo.y, bits.hi.x, bits.hi.y};
  f32x2 x[4];
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = f2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
  const float2 q = un2(fma2(x[0], x[0], fma2(x[1], x[1], fma2(x[2], x[2], mul2(x[3], x[3])))));
  float ss = q.x + q.y;
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float r = norm ? rsqrtf(ss * (1.f / (8 * L)) + eps) : 1.f;
  const f32x2 rr = f2(r, r);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const float2 lo = un2(mul2(rr, fma2(x[2 + i], t.nsb[i], mul2(x[i], t.ca[i])))), hi = un2(mul2(rr, fma2(x[i], t.sa[i], mul2(x[2 + i], t.cb[i]))));
    w[i] = pack_bf16x2(lo.x, lo.y);
    w[2 + i] = pack_bf16x2(hi.x, hi.y);
  }
  if (store) {
    *reinterpret_cast<uint2*>(row + 4 * l) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(row + 4 * L + 4 * l) = make_uint2(w[2], w[3]);
  }
}

// Scale byte of a group whose largest magnitude is amax: the nearest scale to amax / 7, ties to the even byte.  A first guess in 32 bits is corrected by comparing
// amax with seven times the midpoints, products of few bits that are exact.  open is set if a midpoint lies within `off` of it.
__device__ __forceinline__ float kv4_scale_value(int b) { return __uint_as_float((uint32_t)(b + (127 - 16) * 8) << 20); }
template <typename R> __device__ __forceinline__ int kv4_scale_of(R amax, float off, bool& open) {
  const uint32_t u = __float_as_uint((float)amax * (1.f / 7.f));
  int b = (int)((u + (1u << 19)) >> 20) - (127 - 16) * 8;
  b = min(max(b, 0), 255);
  const float lo = kv4_scale_value(max(b - 1, 0)), at = kv4_scale_value(b), hi = kv4_scale_value(min(b + 1, 255));
  const R up = (R)3.5 * ((R)at + (R)hi), down = (R)3.5 * ((R)lo + (R)at);
  const bool odd = b & 1, more = b < 255 && (amax > up || (amax == up && odd)), less = b > 0 && (amax < down || (amax == down && odd));
  open |= fabs((float)(amax - up)) <= off || fabs((float)(amax - down)) <= off;
  return b + more - less;
}
// The nearest multiples of s, ties to even: x / s by a product with the reciprocal (an error that no quotient is as close to a border as, but for the borders
// themselves, or one that `off` covers), rounded by an addition whose sum has them in its last bits.  The exact remainder shows what lies on a border (tie)
// or within `off` of one (open).
__device__ __forceinline__ uint32_t kv4_round(float x, float s, float inv, float off, bool& tie, bool& open) {
  const float t = fmaf(x, inv, 12582912.f), r = fabsf(fmaf(-(t - 12582912.f), s, x)), h = 0.5f * s;
  tie |= r == h;
  open |= h - r < off;
  return __float_as_uint(t);
}
__device__ __forceinline__ uint32_t kv4_round(double x, double s, double inv, float, bool& tie, bool&) {
  const double t = fma(x, inv, 6755399441055744.0), r = fabs(fma(-(t - 6755399441055744.0), s, x));
  tie |= r == 0.5 * s;
  return (uint32_t)__double2loint(t);
}
template <typename R> __device__ __forceinline__ uint32_t kv4_even(uint32_t t, R x, R s) {      // of a quotient on a border, the even neighbour
  const int q = (int)(t << 28) >> 28;
  const R r = x - (R)q * s;
  return (r < 0 ? -r : r) == (R)0.5 * s && (q & 1) ? (uint32_t)(r > 0 ? q + 1 : q - 1) : t;
}
__device__ __forceinline__ float rcp_approx(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// The codes of one row [8 L] (the low four bits of c, signed) and its two scale bytes, by its L lanes (all lanes of the warp call).  Infinities and values past the
// largest become the largest, a NaN becomes 0; no quotient is past 7.47 then.  Returns whether `off`, the error of every element, leaves a code or a scale open.
template <int L, typename R> __device__ __forceinline__ bool code_kv4(R (&x)[8], const float* off, uint32_t (&c)[8], int& b0, int& b1) {
  R m0 = 0, m1 = 0;
  float d0 = 0.f, d1 = 0.f;
  bool wild = false;
#pragma unroll
  for (int e = 0; e < 8; e++) wild |= !(fabs(x[e]) <= (R)kKv4Most);
  if (wild) {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = x[e] > (R)kKv4Most ? (R)kKv4Most : x[e] < -(R)kKv4Most ? -(R)kKv4Most : x[e] == x[e] ? x[e] : (R)0;
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    m0 = fmax(m0, fabs(x[e]));
    m1 = fmax(m1, fabs(x[4 + e]));
    if (off) { d0 = fmaxf(d0, off[e]); d1 = fmaxf(d1, off[4 + e]); }
  }
  if (L == 4) { m0 = m1 = fmax(m0, m1); d0 = d1 = fmaxf(d0, d1); }       // one group of 32: both halves
#pragma unroll
  for (int o = L == 4 ? 2 : 4; o > 0; o >>= 1) {
    m0 = fmax(m0, __shfl_xor_sync(0xffffffffu, m0, o));
    m1 = L == 4 ? m0 : fmax(m1, __shfl_xor_sync(0xffffffffu, m1, o));
    if (off) {
      d0 = fmaxf(d0, __shfl_xor_sync(0xffffffffu, d0, o));
      d1 = L == 4 ? d0 : fmaxf(d1, __shfl_xor_sync(0xffffffffu, d1, o));
    }
  }
  bool open = false, tie = false;
  b0 = kv4_scale_of(m0, d0, open);
  b1 = L == 4 ? b0 : kv4_scale_of(m1, d1, open);
  const float f0 = kv4_scale_value(b0), f1 = kv4_scale_value(b1);
  const R s0 = f0, s1 = f1;
  R i0 = rcp_approx(f0), i1 = rcp_approx(f1);
  if (sizeof(R) == 8) {                                                  // to 2^-44
    i0 = i0 * ((R)2 - s0 * i0);
    i1 = i1 * ((R)2 - s1 * i1);
  }
#pragma unroll
  for (int e = 0; e < 8; e++) c[e] = kv4_round(x[e], e < 4 ? s0 : s1, e < 4 ? i0 : i1, off ? off[e] : -1.f, tie, open);
  if (tie) {
#pragma unroll
    for (int e = 0; e < 8; e++) c[e] = kv4_even(c[e], x[e], e < 4 ? s0 : s1);
  }
  return open;
}
// one row to its place in a 4-bit page; lanes without a row pass store = false
template <int L> __device__ __forceinline__ void store_kv4(uint8_t* page, int tok, int block_size, const uint32_t (&c)[8], int b0, int b1, int l, bool store) {
  constexpr int D = 8 * L;
  // four dims of a word of eight: even places in one byte of the low half, odd ones in one of the high half; code 8 is zero
  uint32_t n[8];
#pragma unroll
  for (int e = 0; e < 8; e++) n[e] = c[e] & 15;
  const int sh = 8 * (l & 1);
  const uint32_t w0 = ((n[0] | n[2] << 4 | n[1] << 16 | n[3] << 20) ^ 0x00880088u) << sh, w1 = ((n[4] | n[6] << 4 | n[5] << 16 | n[7] << 20) ^ 0x00880088u) << sh;
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
__global__ void __launch_bounds__(kRowsWarps * 32, 8) gqa_rows_kernel(const RowsArgs a) {
  pdl_wait(); pdl_trigger();
  constexpr int D = 8 * L, R = 32 / L;
  const int lane = threadIdx.x & 31, l = lane % L, sub = lane / L;
  const int q_steps = (a.Hq + R - 1) / R, kv_steps = (a.Hkv + R - 1) / R, q_warps = (q_steps + a.chunk - 1) / a.chunk, kv_warps = (kv_steps + a.kv_chunk - 1) / a.kv_chunk, per_token = q_warps + 2 * kv_warps;
  const unsigned w = blockIdx.x * kRowsWarps + (threadIdx.x >> 5);
  const int t = (int)(w / (unsigned)per_token), part = (int)(w - (unsigned)t * per_token);
  if (t >= a.T) return;
  const __nv_bfloat16* src = a.qkv + (long long)t * a.ld;
  const bool is_q = part < q_warps, is_v = part >= q_warps + kv_warps;
  const uint2 ones = make_uint2(0x3F803F80u, 0x3F803F80u);
  float cs[4], sn[4];
  auto angles = [&] {                                                        // of the pairs (i, i + D/2), i = 4 l ..
    const float* row[4];
#pragma unroll
    for (int x = 0; x < 4; x++) {
      long long pos = a.positions[(long long)(x < a.axes ? x : 0) * a.pos_ld + t];
      pos = pos < 0 ? 0 : pos >= a.max_pos ? a.max_pos - 1 : pos;            // never outside the table
      row[x] = a.rope + pos * D + 4 * l;
    }
    if (a.axes == 1) {
      const float4 c = *reinterpret_cast<const float4*>(row[0]), s = *reinterpret_cast<const float4*>(row[0] + D / 2);
      cs[0] = c.x; cs[1] = c.y; cs[2] = c.z; cs[3] = c.w;
      sn[0] = s.x; sn[1] = s.y; sn[2] = s.z; sn[3] = s.w;
      return;
    }
    int turn = a.interleaved ? 4 * l % a.axes : 0;
    const int e0 = a.sections[0], e1 = e0 + a.sections[1], e2 = e1 + a.sections[2];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = 4 * l + e;
      int ax;
      if (a.interleaved) {
        ax = turn > 0 && i < a.axes * (turn == 1 ? a.sections[1] : turn == 2 ? a.sections[2] : a.sections[3]) ? turn : 0;
        if (++turn == a.axes) turn = 0;
      } else {
        ax = (i >= e0) + (i >= e1 && a.axes > 2) + (i >= e2 && a.axes > 3);
      }
      const float* r = ax == 0 ? row[0] : ax == 1 ? row[1] : ax == 2 ? row[2] : row[3];
      cs[e] = r[e];
      sn[e] = r[D / 2 + e];
    }
  };
  if (is_q) {
    const int s0 = part * a.chunk, s1 = min(s0 + a.chunk, q_steps);
    const __nv_bfloat16* in = src + (long long)(s0 * R + sub) * D;
    __nv_bfloat16* out = a.q_out + ((long long)t * a.Hq + s0 * R + sub) * D;
    const bool norm = a.qw != nullptr;
    const float eps = (float)a.eps;
    // whole batches first, without a test per row; the next one is loaded while one is worked on
    const int full = min(s1 - s0, a.Hq / R - s0) / kRowsBatch;
    RowBits next[kRowsBatch];
    if (full > 0) {
#pragma unroll
      for (int i = 0; i < kRowsBatch; i++) next[i] = load_row<L>(in + i * R * D, l);
    }
    RowBits g = {ones, ones};
    if (norm) g = load_row<L>(a.qw, l);
    angles();
    Turn<float> one;
    make_turn(one, g, norm ? a.w_offset : 0.f, cs, sn);
    const Turn2 turn = pair_turn(one);
    for (int b = 0; b < full; b++) {
      in += kRowsBatch * R * D;
#pragma unroll
      for (int i = 0; i < kRowsBatch; i++) {
        const RowBits now = next[i];
        if (b + 1 < full) next[i] = load_row<L>(in + i * R * D, l);
        query_row<L>(now, out + i * R * D, l, true, turn, norm, eps);
      }
      out += kRowsBatch * R * D;
    }
    for (int s = s0 + full * kRowsBatch; s < s1; s++) {
      const bool live = s * R + sub < a.Hq;
      RowBits now = {make_uint2(0, 0), make_uint2(0, 0)};
      if (live) now = load_row<L>(in, l);
      query_row<L>(now, out, l, live, turn, norm, eps);
      in += R * D;
      out += R * D;
    }
    return;
  }
  const long long slot = a.slots[t];
  if (slot < 0 || slot >= a.cache_rows || !NE_INDEX_OK(slot, BK_CACHE_ROWS, 30, __LINE__)) return;
  const int s0 = (part - q_warps - (is_v ? kv_warps : 0)) * a.kv_chunk, s1 = min(s0 + a.kv_chunk, kv_steps);
  const __nv_bfloat16* in = src + (long long)(a.Hq + (is_v ? a.Hkv : 0)) * D;
  uint8_t* cache = is_v ? a.v_cache : a.k_cache;
  const bool norm = a.kw != nullptr;
  int h = s0 * R + sub;
  RowBits next = {make_uint2(0, 0), make_uint2(0, 0)}, g = {ones, ones};
  if (h < a.Hkv) next = load_row<L>(in + h * D, l);
  Turn<float> turn;
  if (!is_v) {
    if (norm) g = load_row<L>(a.kw, l);
    angles();
    make_turn(turn, g, norm ? a.w_offset : 0.f, cs, sn);
  }
  long long page = 0; int tok = 0;
  if (kInt4) split_slot(slot, a.block_size, page, tok);
  for (int s = s0; s < s1; s++, h += R) {
    const RowBits bits = next;
    const bool live = h < a.Hkv;
    if (s + 1 < s1 && h + R < a.Hkv) next = load_row<L>(in + (h + R) * D, l);
    float x[8], off[8];
    unpack_row(bits, x);
    if (!is_v) norm_and_turn<L, float>(x, turn, norm, (float)a.eps, off);
    if constexpr (kInt4) {
      uint32_t c[8];
      int b0, b1;
      if (is_v) {
        code_kv4<L, float>(x, nullptr, c, b0, b1);
      } else if (__any_sync(0xffffffffu, code_kv4<L, float>(x, off, c, b0, b1) && live)) {
        RowBits again = bits, weights = g;
        // (opaque, or what does not change from step to step moves in front of them all)
        asm volatile("" : "+r"(weights.lo.x), "+r"(weights.lo.y), "+r"(weights.hi.x), "+r"(weights.hi.y), "+r"(again.lo.x), "+r"(again.lo.y), "+r"(again.hi.x), "+r"(again.hi.y));
        float f[8];
        double y[8];
        unpack_row(again, f);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = f[e];
        Turn<double> wide;
        make_turn(wide, weights, norm ? a.w_offset : 0.f, cs, sn);
        norm_and_turn<L, double>(y, wide, norm, a.eps);
        code_kv4<L, double>(y, nullptr, c, b0, b1);
      }
      store_kv4<L>(cache + (page * a.Hkv + (live ? h : 0)) * ((long long)a.block_size * (D / 2 + D / 32)), tok, a.block_size, c, b0, b1, l, live);
    } else {
      if (live) store_row<L>(reinterpret_cast<__nv_bfloat16*>(cache) + (slot * a.Hkv + h) * D, l, x);
    }
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
  uint32_t c[8];
  int b0, b1;
  code_kv4<L, float>(x, nullptr, c, b0, b1);
  store_kv4<L>((r & 1 ? v_cache : k_cache) + (page * Hkv + (live ? h : 0)) * ((long long)block_size * (D / 2 + D / 32)), tok, block_size, c, b0, b1, l, live);
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
// with it; pages behind a context are left out.  A CTA takes a page of a head: its threads find the rows' places once, then each unpacks words of 8 dims, so that
// neighbouring lanes store neighbouring 16 bytes.
template <int D>
__global__ void __launch_bounds__(256) kv4_expand_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, int num_blocks,
                                                        const int* __restrict__ tables, long long bt_ld, int bt_width, const int* __restrict__ ctx,
                                                        __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int* __restrict__ out_tables,
                                                        int* __restrict__ out_ctx, int width, int Hkv, int block_size) {
  pdl_wait(); pdl_trigger();
  constexpr int words = D / 8, items = 64 * words / 256, kFlight = items < 4 ? items : 4;        // words of a thread, in flight
  __shared__ long long s_code[64], s_scale[64];                          // where a row's codes and scales begin, -1: zeros
  const int seq = blockIdx.y, p = blockIdx.x, h = blockIdx.z;
  const long long at = (long long)seq * width + p;
  const int n = (int)min((long long)ctx[seq], (long long)bt_width * block_size);
  if (h == 0 && threadIdx.x == 0) {
    out_tables[at] = (int)at;
    if (p == 0) out_ctx[seq] = n;
  }
  if (p * 64 >= n) return;
  if (threadIdx.x < 64) {
    const int key = p * 64 + threadIdx.x;
    long long code = -1, scale = -1;
    if (key < n) {
      const int page = key / block_size, tok = key - page * block_size, id = tables[(long long)seq * bt_ld + page];
      if (id >= 0 && id < num_blocks && NE_INDEX_OK(id, BK_CACHE_PAGES, 30, __LINE__)) {
        const long long base = ((long long)id * Hkv + h) * ((long long)block_size * (D / 2 + D / 32));
        code = base + tok * (D / 2);
        scale = base + block_size * (D / 2) + tok * (D / 32);
      }
    }
    s_code[threadIdx.x] = code;
    s_scale[threadIdx.x] = scale;
  }
  __syncthreads();
#pragma unroll
  for (int i0 = 0; i0 < items; i0 += kFlight) {
    uint32_t kw[kFlight], vw[kFlight], ks[kFlight], vs[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; u++) {
      const int i = threadIdx.x + (i0 + u) * 256, r = i / words, j = i % words;
      const long long code = s_code[r], scale = s_scale[r] + j / 4;
      kw[u] = vw[u] = 0x88888888u;                                       // zeros
      ks[u] = vs[u] = 0;
      if (code >= 0) {
        kw[u] = *reinterpret_cast<const uint32_t*>(k_cache + code + 4 * j); ks[u] = k_cache[scale];
        vw[u] = *reinterpret_cast<const uint32_t*>(v_cache + code + 4 * j); vs[u] = v_cache[scale];
      }
    }
#pragma unroll
    for (int u = 0; u < kFlight; u++) {
      const int i = threadIdx.x + (i0 + u) * 256, r = i / words, j = i % words;
      const long long dst = ((at * 64 + r) * Hkv + h) * D + 8 * j;
      *reinterpret_cast<uint4*>(k_out + dst) = kv4_word(kw[u], ks[u]);
      *reinterpret_cast<uint4*>(v_out + dst) = kv4_word(vw[u], vs[u]);
    }
  }
}

}  // namespace ne

using namespace ne;

namespace {
// The kernels read and write words of eight codes: a head's part of a page has to be whole words (heads of 32: pages of a multiple of 4 tokens, of 64: of 2)
bool kv4_words(int block_size, int D) { return ((long long)block_size * (D / 2 + D / 32)) % 4 == 0; }

template <int L> int launch_rows(const RowsArgs& a, bool int4, cudaStream_t st) {
  constexpr int R = 32 / L;
  const int q_steps = (a.Hq + R - 1) / R, kv_steps = (a.Hkv + R - 1) / R;
  const long long warps = (long long)a.T * ((q_steps + a.chunk - 1) / a.chunk + 2 * ((kv_steps + a.kv_chunk - 1) / a.kv_chunk));
  if (warps >= (1ll << 31)) return 1003;
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
  if ((int4 && !kv4_words(block_size, D)) || (ld & 3) || ((uintptr_t)qkv & 7) || (((uintptr_t)qw | (uintptr_t)kw) & 7) || ((uintptr_t)rope & 15)) return 1004;
  RowsArgs a{};
  a.qkv = (const __nv_bfloat16*)qkv; a.ld = ld; a.qw = (const __nv_bfloat16*)qw; a.kw = (const __nv_bfloat16*)kw; a.eps = eps; a.w_offset = w_offset;
  a.positions = positions; a.pos_ld = pos_ld; a.rope = rope; a.max_pos = max_pos; a.axes = axes; a.interleaved = interleaved;
  for (int i = 0; i < axes; i++) a.sections[i] = sections[i];
  a.q_out = (__nv_bfloat16*)q_out; a.k_cache = (uint8_t*)k_cache; a.v_cache = (uint8_t*)v_cache; a.slots = slots; a.cache_rows = cache_rows;
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.block_size = block_size;
  // Few rows: a warp per step, so that all SMs work; many: several steps under one fetch of the angles.  us of few / many: 64 / 4 heads of 128 into 4 bits, three axes:
  // 16 tokens 3.4 / 4.2, 128: 5.3 / 4.6, 1024: 25 / 12; 32 / 8 heads: 128: 4.9 / 5.9, 256: 6.1 / 6.3, 512: 9.5 / 7.4; 16 / 2 heads of 256: 128: 4.6 / 4.4, 256: 5.2 / 4.6.
  const bool many = (long long)T * Hq * D >= 1 << 20;
  a.chunk = many ? 8 : 1;
  a.kv_chunk = many ? 4 : 1;
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
  if (!kv4_words(block_size, D) || ((k_ld | v_ld) & 3) || (((uintptr_t)k | (uintptr_t)v) & 7)) return 1004;
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
  if (Hkv < 1 || block_size < 1 || D < 32 || D % 32 || !kv4_words(block_size, D)) return 1001;
  const long long n = (long long)T * Hkv * (D / 8);
  return (int)launch_pdl(kv4_gather_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, (const uint8_t*)k_cache, (const uint8_t*)v_cache, slots, cache_rows,
                         (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, T, Hkv, D, block_size);
}

// width: pages of 64 tokens per sequence, at least ceil(bt_width * block_size / 64)
extern "C" int ne_kv4_expand(const void* k_cache, const void* v_cache, int num_blocks, const int* tables, long long bt_ld, int bt_width, const int* ctx, int seqs, int width,
                             void* k_out, void* v_out, int* out_tables, int* out_ctx, int Hkv, int D, int block_size, cudaStream_t st) {
  if (seqs <= 0 || width <= 0) return 0;
  if (!kv4_words(block_size, D)) return 1004;
  if (num_blocks < 1 || Hkv < 1 || block_size < 1 || seqs > 65535 || Hkv > 65535 || (long long)width * 64 < (long long)bt_width * block_size ||
      (long long)seqs * width >= (1ll << 31)) return 1001;
  auto go = [&](auto kern) {
    return (int)launch_pdl(kern, dim3((unsigned)width, (unsigned)seqs, (unsigned)Hkv), dim3(256), 0, st, (const uint8_t*)k_cache, (const uint8_t*)v_cache, num_blocks, tables,
                           bt_ld, bt_width, ctx, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, out_tables, out_ctx, width, Hkv, block_size);
  };
  return D == 64 ? go(kv4_expand_kernel<64>) : D == 128 ? go(kv4_expand_kernel<128>) : D == 256 ? go(kv4_expand_kernel<256>) : 1002;
}
