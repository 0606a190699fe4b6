// Tables of a paged step from its sequences' lengths: cumulative query lengths, context lengths, positions, cache slots, padded block tables and
// last-token rows, with the padding rows of a captured batch behind the sequences.
//
//   cu[i + 1] = cu[i] + q[i] ; position(t) = n[i] - q[i] + t - cu[i] ; slot(t) = page[position / bs] * bs + position % bs
//
// Bound by latency: a decode step reads and writes tens of KB.  One launch: every CTA takes the prefix sum of all rows itself (a few hundred values
// that sit in L2) instead of a scan kernel in front, then the CTAs share tokens and table entries; a token finds its sequence by a binary search in
// shared memory.  Measured (B200, in a graph): 128 decode rows of 64 pages 3.3 us, 13 portions of 1260 tokens 2.9, one row of 2048 pages 2.9.
#include "ptx.cuh"

namespace ne {

constexpr int kStepThreads = 256;

struct StepArgs {
  const int* q_lens; const int* seq_lens; const int* ids; const int* offsets;
  int seqs, rows, n_ids, block_size, tokens, width, pad_len, scratch;
  int* cu; int* ctx; long long* positions; long long* slots; int* tables; long long table_ld; int* last;
};

__global__ void __launch_bounds__(kStepThreads) step_tables_kernel(const StepArgs a) {
  pdl_wait(); pdl_trigger();
  extern __shared__ int s_cu[];                    // [rows + 1]
  __shared__ int s_warp[kStepThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int carry = 0;
  for (int r0 = 0; r0 < a.rows; r0 += kStepThreads) {
    const int r = r0 + tid;
    int v = r < a.seqs ? max(a.q_lens[r], 0) : (r < a.rows ? a.pad_len : 0);
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += u; }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int before = carry, total = 0;
#pragma unroll
    for (int w = 0; w < kStepThreads / 32; w++) { before += w < warp ? s_warp[w] : 0; total += s_warp[w]; }
    if (r < a.rows) s_cu[r + 1] = before + incl;
    carry += total;
    __syncthreads();
  }
  if (tid == 0) s_cu[0] = 0;
  __syncthreads();
  const long long stride = (long long)gridDim.x * kStepThreads, first = (long long)blockIdx.x * kStepThreads + tid;
  for (long long r = first; r <= a.rows; r += stride) {
    a.cu[r] = s_cu[r];
    if (r < a.rows) { a.ctx[r] = r < a.seqs ? a.seq_lens[r] : a.pad_len; a.last[r] = s_cu[r + 1] - 1; }
  }
  for (long long t = first; t < a.tokens; t += stride) {
    long long pos = 0, slot = -1;
    if (a.rows > 0 && t < s_cu[a.rows]) {
      int lo = 0, hi = a.rows;                     // the row with cu[lo] <= t < cu[lo + 1]
      while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (s_cu[mid] <= t) lo = mid; else hi = mid; }
      const int j = (int)t - s_cu[lo];
      if (lo >= a.seqs) {
        pos = j;
        slot = j / a.block_size < a.width ? (long long)a.scratch * a.block_size + j % a.block_size : -1;
      } else {
        const long long p = (long long)a.seq_lens[lo] - (s_cu[lo + 1] - s_cu[lo]) + j;
        if (p >= 0) {
          pos = p;
          const int o0 = min(max(a.offsets[lo], 0), a.n_ids), o1 = min(max(a.offsets[lo + 1], 0), a.n_ids);
          const int at = (int)p / a.block_size;
          const int page = at < o1 - o0 ? a.ids[o0 + at] : -1;
          if (page >= 0) slot = (long long)page * a.block_size + (int)p % a.block_size;
        }
      }
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
  const long long cells = (long long)a.rows * a.width;
  for (long long c = first; c < cells; c += stride) {
    const int r = (int)(c / a.width), col = (int)(c - (long long)r * a.width);
    int id = a.scratch;
    if (r < a.seqs) {
      const int o0 = min(max(a.offsets[r], 0), a.n_ids), o1 = min(max(a.offsets[r + 1], 0), a.n_ids);
      id = col < o1 - o0 ? a.ids[o0 + col] : 0;
    }
    a.tables[(long long)r * a.table_ld + col] = id;
  }
}

}  // namespace ne

using namespace ne;

// q_lens / seq_lens int32 [seqs], ids int32 [n_ids], offsets int32 [seqs + 1]; outputs as the kernel's arguments name them, tables rows table_ld apart.
extern "C" int ne_step_tables(const int* q_lens, const int* seq_lens, const int* ids, const int* offsets, int seqs, int rows, int n_ids, int block_size,
                              int tokens, int width, int pad_len, int scratch, int* cu, int* ctx, long long* positions, long long* slots, int* tables,
                              long long table_ld, int* last, cudaStream_t st) {
  if (seqs < 0 || rows < seqs || n_ids < 0 || block_size < 1 || tokens < 0 || width < 1 || pad_len < 1 || table_ld < width) return 1001;
  if (rows > 12000) return 1002;                   // the prefix sums sit in the 48 KB of shared memory every launch may have
  StepArgs a{q_lens, seq_lens, ids, offsets, seqs, rows, n_ids, block_size, tokens, width, pad_len, scratch, cu, ctx, positions, slots, tables, table_ld, last};
  const long long work = (long long)rows * width + tokens;
  const unsigned grid = (unsigned)min(296ll, (work + kStepThreads - 1) / kStepThreads + 1);
  return (int)launch_pdl(step_tables_kernel, dim3(grid), dim3(kStepThreads), (size_t)(rows + 1) * sizeof(int), st, a);
}
