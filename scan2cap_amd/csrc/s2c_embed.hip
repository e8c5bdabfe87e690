// s2c_embed.hip -- embedding lookup with scaling (s2c_embed_fwd) and the table's gradient
// (s2c_embed_grad).
//
// Lookup: out[n] = scale table[token[n]], one rounding; bound by writing N D elements and reading the
// distinct rows.
// Gradient: d_table[v] = scale sum_{n: token[n] = v} g[n]; every row is written, so the floor is reading
// N D and writing V D elements.  A wave owns a table row's columns and adds the row's places in their
// order in 32-bit registers: no atomics, the same bits every time.  Where a row's places are comes from
//  * looking through all tokens (few tokens: one launch), or
//  * a stable sort of (word, place) by word; padding and bad tokens sort behind the last word.  The sorted
//    order is cut into chunks, a wave each, whatever words are in them (a word's run may be most of the
//    batch, or one place): the wave has 4 to 8 of its rows under way and writes a word's sum when its run ends.
//    A run that passes a chunk's border leaves partial sums, which a last launch joins in order, 16 waves to a
//    long run (10^6 x 256 bf16 whose most frequent word takes 4 %: 30 us, 73 with 4).  The rows of the
//    words that are not in the batch are written beside the sums.
// Measured (kernel times, MI355X): 131072 tokens x 1024 bf16, 50001 words: lookup 80 us (4.1 TB/s),
// gradient 120 us = sort 27 + runs 83 + join 10 (floor 73 us at 5.1 TB/s); 8191 x 515 fp16, 10007 words:
// lookup 5.7 us, gradient 35 us = sort 18 + 10 + 7.
#include "s2c_words_common.h"

#include <stdio.h>

#include <type_traits>

using namespace s2c;

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;

// VEC elements of a row that ends at D, from column col
template <int DT>
__device__ __forceinline__ Raw load_part(const void *p, long long i, int valid) {
  typedef Elem<DT> E;
  Raw r = {{0u, 0u, 0u, 0u}};
  if (valid >= E::VEC) return load16<DT>(p, i);
  if (valid <= 0) return r;
#pragma unroll
  for (int e = 0; e < E::VEC; ++e)
    if (e < valid) E::put(r, e, E::bits(p, i + e));
  return r;
}
template <int DT>
__device__ __forceinline__ void store_part(void *p, long long i, int valid, const float (&f)[Elem<DT>::VEC]) {
  typedef Elem<DT> E;
  if (valid >= E::VEC) {
    store16<DT>(p, i, E::pack(f));
  } else {
#pragma unroll
    for (int e = 0; e < E::VEC; ++e)
      if (e < valid) E::store(p, i + e, f[e]);
  }
}

// lpr lanes per row (a power of two <= 64), ROWS rows under way per lane
template <int DT, int ROWS>
__global__ __launch_bounds__(THREADS) void embed_fwd_kernel(long long N, int V, int D, long long ld,
                                                            const long long *__restrict__ token,
                                                            const void *__restrict__ table, float scale,
                                                            long long padding, void *__restrict__ out,
                                                            int lpr, bool past_cache) {
  typedef Elem<DT> E;
  const int sub = threadIdx.x & (lpr - 1), per = THREADS / lpr;
  const long long step = (long long)gridDim.x * per * ROWS;
  for (long long n0 = (long long)blockIdx.x * per * ROWS + threadIdx.x / lpr; n0 < N; n0 += step) {
    long long t[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) t[i] = n0 + i * per < N ? token[n0 + i * per] : padding;
    for (int c = sub * E::VEC; c < D; c += lpr * E::VEC) {
      Raw r[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const bool good = t[i] != padding && t[i] >= 0 && t[i] < V;
        r[i] = load_part<DT>(table, good ? t[i] * ld + c : 0, good ? D - c : 0);
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const long long n = n0 + i * per;
        if (n >= N) break;
        const bool pad = t[i] == padding && padding != S2C_WORDS_NO_PADDING;
        const bool bad = !pad && (t[i] < 0 || t[i] >= V);
        float f[E::VEC];
#pragma unroll
        for (int e = 0; e < E::VEC; ++e) f[e] = bad ? NAN : pad ? 0.0f : scale * E::at(r[i], e);
        if (past_cache) store16_past_cache(out, (n * D + c) * E::ES, E::pack(f));
        else store_part<DT>(out, n * D + c, D - c, f);
      }
    }
  }
}

// ---- gradient ------------------------------------------------------------------------------------------
// A lane's VEC columns of one row, from column col
template <int DT>
struct Acc {
  typedef Elem<DT> E;
  float f[E::VEC];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int e = 0; e < E::VEC; ++e) f[e] = 0.0f;
  }
  __device__ __forceinline__ void add(const Raw &r) {
#pragma unroll
    for (int e = 0; e < E::VEC; ++e) f[e] += E::at(r, e);
  }
  // row: the element that the row starts at
  __device__ __forceinline__ void store(void *d, long long row, int col, int D, float scale) {
#pragma unroll
    for (int e = 0; e < E::VEC; ++e) f[e] *= scale;
    if (col < D) store_part<DT>(d, row + col, D - col, f);
  }
};

struct GradArgs {
  long long N, ldg, padding;
  int V, D, pieces;              // pieces: waves to a row's columns
  float scale;
  const long long *token;
  const void *g;
  void *dt;
  // the sorted order
  u32 *key, *pos;                // (N) each
  int chunk;                     // places of it that a wave takes, <= 64
  float *partial;                // (chunks, 2, ldp): a chunk's run that began before it, one that goes on
  int ldp;                       // D, up to a multiple of 8
};

// a token as a sort key: its word, or V
__device__ __forceinline__ u32 word_key(long long t, int V, long long padding) {
  return t != padding && t >= 0 && t < V ? (u32)t : (u32)V;
}

constexpr int STAGE = 512;        // tokens that are looked through
constexpr int AHEAD = 8;          // rows under way per wave

// a wave per word and piece of its columns
template <int DT>
__global__ __launch_bounds__(THREADS) void embed_grad_scan_kernel(GradArgs a) {
  typedef Elem<DT> E;
  __shared__ u32 s_tok[STAGE];
  __shared__ u16 s_at[WAVES][STAGE];                 // the places of a wave's word
  const int lane = lane_id(), w = threadIdx.x >> 6;
  const int n = (int)a.N, n64 = (n + 63) & ~63;
  for (int i = threadIdx.x; i < n64; i += THREADS)
    s_tok[i] = i < n ? word_key(a.token[i], a.V, a.padding) : (u32)a.V;
  __syncthreads();
  const long long units = (long long)a.V * a.pieces;
  for (long long un = (long long)blockIdx.x * WAVES + w; un < units; un += (long long)gridDim.x * WAVES) {
    const u32 v = (u32)(un / a.pieces);
    const int col = ((int)(un % a.pieces) * 64 + lane) * E::VEC;
    int m = 0;
    for (int i0 = 0; i0 < n; i0 += 64) {
      const u64 mask = __ballot(s_tok[i0 + lane] == v);
      if ((mask >> lane) & 1) s_at[w][m + mask_rank_below(mask)] = (u16)(i0 + lane);
      m += __popcll(mask);
    }
    wave_lds_fence();
    Acc<DT> acc;
    acc.clear();
    for (int j0 = 0; j0 < m; j0 += AHEAD) {
      Raw r[AHEAD];
#pragma unroll
      for (int q = 0; q < AHEAD; ++q)
        if (j0 + q < m) r[q] = load_part<DT>(a.g, s_at[w][j0 + q] * a.ldg + col, a.D - col);
#pragma unroll
      for (int q = 0; q < AHEAD; ++q)
        if (j0 + q < m) acc.add(r[q]);
    }
    wave_lds_fence();
    acc.store(a.dt, (long long)v * a.D, col, a.D, a.scale);
  }
}

// ---- the sort: least significant digit first, 8 bits at most a pass -------------------------------------
constexpr int RADIX = 256;

// lanes of the wave with the same digit (of `bits` bits), among `valid`
__device__ __forceinline__ u64 same_digit(u32 d, int bits, u64 valid) {
  u64 peers = valid;
  for (int b = 0; b < bits; ++b) {
    const u64 on = __ballot((d >> b) & 1);
    peers &= (d >> b) & 1 ? on : ~on;
  }
  return peers;
}

// exclusive prefix sum over the first 256 threads; all threads of the workgroup call it
__device__ __forceinline__ u32 scan256(u32 v, u32 *s_wave) {
  const int lane = lane_id(), w = threadIdx.x >> 6;
  u32 x = v;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const u32 o = __shfl_up(x, k);
    if (lane >= k) x += o;
  }
  if (lane == 63 && w < 4) s_wave[w] = x;
  __syncthreads();
  u32 base = 0;
  for (int i = 0; i < 4; ++i)
    if (i < w) base += s_wave[i];
  __syncthreads();
  return base + x - v;
}

constexpr int SMALL = 8192, SMALL_THREADS = 1024;

// up to SMALL_THREADS ITEMS tokens by one workgroup, all passes in registers and LDS
template <int ITEMS>
__global__ __launch_bounds__(SMALL_THREADS) void sort_small_kernel(GradArgs a, int passes, int bits) {
  constexpr int W = SMALL_THREADS / 64;
  __shared__ u32 s_x[SMALL_THREADS * ITEMS];
  __shared__ u32 s_cnt[W][RADIX];
  __shared__ u32 s_wave[4];
  const int tid = threadIdx.x, lane = lane_id(), w = tid >> 6;
  const int n = (int)a.N;
  u32 key[ITEMS], pos[ITEMS], at[ITEMS];
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = (w * ITEMS + r) * 64 + lane;
    key[r] = i < n ? word_key(a.token[i], a.V, a.padding) : 0xFFFFFFFFu;       // (sorts behind everything)
    pos[r] = i;
  }
  for (int p = 0; p < passes; ++p) {
    for (int i = tid; i < W * RADIX; i += SMALL_THREADS) (&s_cnt[0][0])[i] = 0;
    __syncthreads();
    const u32 dmask = (1u << bits) - 1;
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const u32 d = (key[r] >> (p * bits)) & dmask;
      const u64 peers = same_digit(d, bits, ~0ull);
      const u32 before = s_cnt[w][d];
      at[r] = before + mask_rank_below(peers);
      wave_lds_fence();
      if (mask_rank_below(peers) == 0) s_cnt[w][d] = before + __popcll(peers);
      wave_lds_fence();
    }
    __syncthreads();
    u32 total = 0;
    if (tid < RADIX)
      for (int i = 0; i < W; ++i) total += s_cnt[i][tid];
    u32 base = scan256(total, s_wave);
    if (tid < RADIX)
      for (int i = 0; i < W; ++i) {
        const u32 c = s_cnt[i][tid];
        s_cnt[i][tid] = base;
        base += c;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      at[r] += s_cnt[w][(key[r] >> (p * bits)) & dmask];
      s_x[at[r]] = key[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) key[r] = s_x[(w * ITEMS + r) * 64 + lane];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) s_x[at[r]] = pos[r];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) pos[r] = s_x[(w * ITEMS + r) * 64 + lane];
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = (w * ITEMS + r) * 64 + lane;
    if (i < n) {
      a.key[i] = key[r];
      a.pos[i] = pos[r];
    }
  }
}

// many tokens: per pass a histogram of every workgroup's stretch, then a stable scatter
constexpr int TILE_ITEMS = 4, TILE = THREADS * TILE_ITEMS, MAX_SORT_GRID = 256;

struct SortArgs {
  long long N, per;              // tokens, tokens per workgroup (a multiple of TILE)
  int shift, bits;
  // the first pass reads tokens, later ones (key, place)
  const long long *token;
  long long padding;
  int V;
  const u32 *key_in, *pos_in;
  u32 *key_out, *pos_out;
  u32 *counts;                   // (gridDim.x, RADIX)
};

__device__ __forceinline__ u32 sort_key(const SortArgs &a, long long i) {
  return a.token ? word_key(a.token[i], a.V, a.padding) : a.key_in[i];
}

__global__ __launch_bounds__(THREADS) void sort_count_kernel(SortArgs a) {
  __shared__ u32 s_cnt[RADIX];
  s_cnt[threadIdx.x] = 0;
  __syncthreads();
  const long long b = blockIdx.x * a.per, e = min(a.N, b + a.per);
  const u32 dmask = (1u << a.bits) - 1;
  for (long long i = b + threadIdx.x; i < e; i += THREADS) atomicAdd(&s_cnt[(sort_key(a, i) >> a.shift) & dmask], 1u);
  __syncthreads();
  a.counts[(size_t)blockIdx.x * RADIX + threadIdx.x] = s_cnt[threadIdx.x];
}

__global__ __launch_bounds__(THREADS) void sort_scatter_kernel(SortArgs a) {
  static_assert(RADIX == THREADS, "a thread per digit");
  __shared__ u32 s_base[RADIX];
  __shared__ u32 s_cnt[WAVES][RADIX];
  __shared__ u32 s_wave[4];
  const int tid = threadIdx.x, lane = lane_id(), w = tid >> 6;
  const u32 dmask = (1u << a.bits) - 1;
  {
    // this workgroup's first place of digit tid: all smaller digits, then the workgroups before it
    u32 total = 0, before = 0;
#pragma unroll 32
    for (u32 i = 0; i < gridDim.x; ++i) {
      const u32 x = a.counts[(size_t)i * RADIX + tid];
      total += x;
      before += i < blockIdx.x ? x : 0u;
    }
    s_base[tid] = scan256(total, s_wave) + before;
  }
  const long long b = blockIdx.x * a.per, e = min(a.N, b + a.per);
  for (long long t0 = b; t0 < e; t0 += TILE) {
    for (int i = 0; i < WAVES; ++i) s_cnt[i][tid] = 0;
    __syncthreads();
    u32 key[TILE_ITEMS], pos[TILE_ITEMS], at[TILE_ITEMS];
#pragma unroll
    for (int r = 0; r < TILE_ITEMS; ++r) {
      const long long i = t0 + (w * TILE_ITEMS + r) * 64 + lane;
      key[r] = i < e ? sort_key(a, i) : 0u;
      pos[r] = i < e ? (a.token ? (u32)i : a.pos_in[i]) : 0u;
    }
#pragma unroll
    for (int r = 0; r < TILE_ITEMS; ++r) {
      const bool valid = t0 + (w * TILE_ITEMS + r) * 64 + lane < e;
      const u32 d = (key[r] >> a.shift) & dmask;
      const u64 peers = same_digit(d, a.bits, __ballot(valid));
      const u32 before = s_cnt[w][d];
      at[r] = before + mask_rank_below(peers);
      wave_lds_fence();
      if (valid && mask_rank_below(peers) == 0) s_cnt[w][d] = before + __popcll(peers);
      wave_lds_fence();
    }
    __syncthreads();
    u32 base = s_base[tid];
    for (int i = 0; i < WAVES; ++i) {
      const u32 c = s_cnt[i][tid];
      s_cnt[i][tid] = base;
      base += c;
    }
    s_base[tid] = base;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TILE_ITEMS; ++r) {
      if (t0 + (w * TILE_ITEMS + r) * 64 + lane < e) {
        const u32 to = s_cnt[w][(key[r] >> a.shift) & dmask] + at[r];
        a.key_out[to] = key[r];
        a.pos_out[to] = pos[r];
      }
    }
    __syncthreads();
  }
}

constexpr int BATCH = 4;          // rows of a chunk that are asked for together

constexpr int WORDS = 32, GROUP = 8;      // of a workgroup that looks for absent words: words, pieces of their columns

// which of the WORDS words from v0 are in the batch (a bit each).  A trip to memory takes about 0.7 us, so
// the places of the words' keys are narrowed 64 fold a trip, and few keys are all read at once.
__device__ __forceinline__ u64 present_words(const GradArgs &a, u32 v0, int lane) {
  const u32 v[2] = {v0, v0 + WORDS}, end = (u32)a.N;
  u32 at[2] = {0u, 0u};                              // the first key that is not below v[t]: at .. at + span
  for (u32 span = end; span;) {
    const u32 step = (span + 63) / 64, last = (lane + 1) * step - 1;
    u32 key[2];                                      // (no condition on a load: they go together)
#pragma unroll
    for (int t = 0; t < 2; ++t) key[t] = a.key[min(at[t] + last, end - 1)];
#pragma unroll
    for (int t = 0; t < 2; ++t) at[t] += __popcll(__ballot(at[t] + last < end && key[t] < v[t])) * step;
    span = step - 1;
  }
  u64 present = 0;
  if (at[1] - at[0] <= 8 * 64) {
    u32 key[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const u32 j = at[0] + i * 64 + lane;
      const u32 k = a.key[min(j, end - 1u)];
      key[i] = j < at[1] ? k : 0xFFFFFFFFu;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (key[i] != 0xFFFFFFFFu) present |= 1ull << (key[i] - v0);
    for (int k = 1; k < 64; k <<= 1) present |= __shfl_xor(present, k);
    return present;
  }
  u32 lo = at[0], hi = at[1];
  while (lo < hi) {
    const u32 mid = lo + (hi - lo) / 2;
    if (a.key[mid] < v0 + lane) lo = mid + 1; else hi = mid;
  }
  return __ballot(lo < at[1] && a.key[lo < at[1] ? lo : at[0]] == v0 + lane);
}

// The rows of the words that are not in the batch.  A wave writes few of them, one after the other: 64 words to
// a workgroup take longer where the table is small (8192 tokens, 3500 rows of 8 KB: runs 24 us, 22 with 32), 8 where
// it is large (2048 tokens, 131072 rows of 1 KB: 36 us, 22).
template <int DT>
__device__ __forceinline__ void absent_rows(const GradArgs &a, long long first, long long step) {
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int groups = (a.pieces + GROUP - 1) / GROUP;
  const long long units = ((long long)a.V + WORDS - 1) / WORDS * groups;
  for (long long un = first; un < units; un += step) {
    const long long part = groups == 1 ? un : un / groups;
    const int v0 = (int)(part * WORDS), p0 = (int)(un - part * groups) * GROUP, p1 = min(a.pieces, p0 + GROUP);
    u64 absent = ~present_words(a, (u32)v0, lane);
    absent &= __ballot(lane < WORDS && lane < a.V - v0 && (lane & (WAVES - 1)) == w);
    for (; absent; absent &= absent - 1) {
      const long long row = (long long)(v0 + __builtin_ctzll(absent)) * a.D;
      for (int p = p0; p < p1; ++p) {
        Acc<DT> zero;
        zero.clear();
        zero.store(a.dt, row, (p * 64 + lane) * Elem<DT>::VEC, a.D, 1.0f);
      }
    }
  }
}

// The first `sums` workgroups: the sums of the chunks' runs.  The others: the rows of the absent words.
template <int DT>
__global__ __launch_bounds__(THREADS) void embed_runs_kernel(GradArgs a, int sums) {
  typedef Elem<DT> E;
  if ((int)blockIdx.x >= sums) {
    absent_rows<DT>(a, (long long)blockIdx.x - sums, (long long)gridDim.x - sums);
    return;
  }
  const int lane = lane_id(), w = threadIdx.x >> 6;
  const long long units = (a.N + a.chunk - 1) / a.chunk * a.pieces;
  for (long long un = (long long)blockIdx.x * WAVES + w; un < units; un += (long long)sums * WAVES) {
    const long long c = un / a.pieces, i0 = c * a.chunk, i1 = min(a.N, i0 + a.chunk);
    const int m = (int)(i1 - i0);
    const u32 key = lane < m ? a.key[i0 + lane] : 0xFFFFFFFFu;
    const u32 pos = lane < m ? a.pos[i0 + lane] : 0u;
    const u32 before = i0 > 0 ? a.key[i0 - 1] : 0xFFFFFFFFu, after = i1 < a.N ? a.key[i1] : 0xFFFFFFFFu;
    const int n = __popcll(__ballot(key < (u32)a.V));             // (padding and bad tokens come last)
    const int col = ((int)(un % a.pieces) * 64 + lane) * E::VEC;
    Acc<DT> acc;
    acc.clear();
    bool began_before = n > 0 && (u32)__builtin_amdgcn_readlane((int)key, 0) == before;
    auto row = [&](int j) {
      return load_part<DT>(a.g, (long long)(u32)__builtin_amdgcn_readlane((int)pos, j) * a.ldg + col, a.D - col);
    };
    Raw r[BATCH], next[BATCH];                        // these are added while the next are under way
#pragma unroll
    for (int q = 0; q < BATCH; ++q)
      if (q < n) next[q] = row(q);
    for (int j0 = 0; j0 < n; j0 += BATCH) {
#pragma unroll
      for (int q = 0; q < BATCH; ++q) r[q] = next[q];
#pragma unroll
      for (int q = 0; q < BATCH; ++q)
        if (j0 + BATCH + q < n) next[q] = row(j0 + BATCH + q);
#pragma unroll
      for (int q = 0; q < BATCH; ++q) {
        const int j = j0 + q;
        if (j >= n) break;
        acc.add(r[q]);
        const u32 word = (u32)__builtin_amdgcn_readlane((int)key, j);
        const u32 next = j + 1 < m ? (u32)__builtin_amdgcn_readlane((int)key, j + 1) : after;
        const bool goes_on = j + 1 == m && next == word;
        if (next == word && !goes_on) continue;
        if (began_before || goes_on) {
          float *out = a.partial + (size_t)(2 * c + (began_before ? 0 : 1)) * a.ldp + col;
          if (col < a.D) {
#pragma unroll
            for (int e = 0; e < E::VEC; e += 4)
              *reinterpret_cast<float4 *>(out + e) = make_float4(acc.f[e], acc.f[e + 1], acc.f[e + 2], acc.f[e + 3]);
          }
        } else {
          acc.store(a.dt, (long long)word * a.D, col, a.D, a.scale);
        }
        acc.clear();
        began_before = false;
      }
    }
  }
}

// partial sums of the chunks [c0, c1) of a run whose first chunk is `first`
template <int DT>
__device__ __forceinline__ void add_partials(Acc<DT> &acc, const GradArgs &a, u32 first, u32 c0, u32 c1, int col) {
  typedef Elem<DT> E;
  if (col >= a.D) return;
#pragma unroll 8
  for (u32 c = c0; c < c1; ++c) {
    const float *in = a.partial + (2 * (size_t)c + (c == first ? 1 : 0)) * a.ldp + col;
#pragma unroll
    for (int e = 0; e < E::VEC; e += 4) {
      const float4 x = *reinterpret_cast<const float4 *>(in + e);
      acc.f[e] += x.x;
      acc.f[e + 1] += x.y;
      acc.f[e + 2] += x.z;
      acc.f[e + 3] += x.w;
    }
  }
}

constexpr int JOIN_WAVES = 16;
constexpr u32 LONG = 16;          // chunks of a run that the waves of a workgroup join together, more than

// the chunks [c, end) of the run that begins in chunk c and passes its end; end = c: none does
__device__ __forceinline__ u32 run_end(const GradArgs &a, long long c, u32 &word) {
  const long long i0 = c * a.chunk, i1 = i0 + a.chunk;
  if (i1 >= a.N) return (u32)c;
  // the next 64 chunks at once: most runs end there (no condition on a load: all go together)
  const long long j = (c + 1 + lane_id()) * a.chunk;
  const u32 next = a.key[i1], before = a.key[max(i0, 1LL) - 1], begin = a.key[min(j, a.N - 1)];
  word = a.key[i1 - 1];
  if (word >= (u32)a.V || next != word || (i0 > 0 && before == word)) return (u32)c;
  const u64 more = __ballot(j < a.N && begin == word);
  if (~more) return (u32)(c + 1 + __builtin_ctzll(~more));
  long long lo = c + 65, hi = (a.N + a.chunk - 1) / a.chunk;       // the first chunk that begins otherwise
  while (lo < hi) {
    const long long mid = (lo + hi) / 2;
    if (a.key[mid * a.chunk] == word) lo = mid + 1; else hi = mid;
  }
  return (u32)lo;
}

// a workgroup: the runs that begin in JOIN_WAVES chunks and pass their ends, one piece of their columns; chunks far
// apart, since the words of long runs may be neighbours
template <int DT>
__global__ __launch_bounds__(64 * JOIN_WAVES) void embed_join_kernel(GradArgs a) {
  typedef Elem<DT> E;
  __shared__ u32 s_c0[JOIN_WAVES], s_c1[JOIN_WAVES];                        // the long runs
  __shared__ float s_sum[JOIN_WAVES][E::VEC][64];
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const long long chunks = (a.N + a.chunk - 1) / a.chunk;
  const long long per = (chunks + JOIN_WAVES - 1) / JOIN_WAVES, units = per * a.pieces;
  for (long long un = blockIdx.x; un < units; un += gridDim.x) {
    const u32 c0 = (u32)(w * per + un / a.pieces);
    const int col = ((int)(un % a.pieces) * 64 + lane) * E::VEC;
    u32 word = 0;
    const u32 c1 = run_end(a, c0, word);
    const bool many = c1 - c0 > LONG;
    if (lane == 0) {
      s_c0[w] = many ? c0 : 0;
      s_c1[w] = many ? c1 : 0;
    }
    Acc<DT> acc;
    acc.clear();
    if (c1 > c0 && !many) {
      add_partials<DT>(acc, a, c0, c0, c1, col);
      acc.store(a.dt, (long long)word * a.D, col, a.D, a.scale);
    }
    __syncthreads();
    for (u64 runs = __ballot(lane < JOIN_WAVES && s_c1[lane & (JOIN_WAVES - 1)] != 0); runs; runs &= runs - 1) {
      const int i = __builtin_ctzll(runs);
      const u32 b = s_c0[i], n = s_c1[i] - b;
      acc.clear();
      add_partials<DT>(acc, a, b, b + (u32)((u64)n * w / JOIN_WAVES), b + (u32)((u64)n * (w + 1) / JOIN_WAVES), col);
#pragma unroll
      for (int q = 0; q < E::VEC; ++q) s_sum[w][q][lane] = acc.f[q];
      __syncthreads();
      if (w == i) {
#pragma unroll
        for (int q = 0; q < E::VEC; ++q) {
          float x = s_sum[0][q][lane];
          for (int k = 1; k < JOIN_WAVES; ++k) x += s_sum[k][q][lane];
          acc.f[q] = x;
        }
        acc.store(a.dt, (long long)word * a.D, col, a.D, a.scale);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

int launched(const char *what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    fprintf(stderr, "s2c: %s launch failed: %s\n", what, hipGetErrorString(e));
    return (int)e;
  }
  return 0;
}

constexpr int MAX_GRID = 1 << 22;       // workgroups of 256: below 2^32 work-items
int grid_of(long long units) { return (int)(units < 1 ? 1 : units < MAX_GRID ? units : MAX_GRID); }

bool bad_array(const void *p, int dtype) { return !p || ((uintptr_t)p & (dtype == S2C_F32 ? 3 : 1)); }

}  // namespace

extern "C" int s2c_embed_fwd(long long N, int V, int D, int dtype, long long ld, const long long *token,
                             const void *table, float scale, long long padding, void *out, void *stream) {
  if (N < 0 || V <= 0 || D <= 0 || D > S2C_WORDS_MAX_DIM || dtype < 0 || dtype > 2 || ld < 0) return S2C_EINVAL;
  if (N == 0) return 0;
  if (!token || bad_array(table, dtype) || bad_array(out, dtype)) return S2C_EINVAL;
  const int vec = dtype == S2C_F32 ? 4 : 8;
  int lpr = 1;
  while (lpr < 64 && lpr * vec < D) lpr *= 2;
  hipStream_t st = (hipStream_t)stream;
  // an output that the 256 MB cache cannot hold is stored past it, in whole vectors (131072 x 4096 bf16: 228 us,
  // 258 us through it; and what runs next finds no lines to be written back)
  const long long row_bytes = (long long)D * (dtype == S2C_F32 ? 4 : 2);
  const bool past_cache = N * row_bytes >= (256LL << 20) && row_bytes % 16 == 0 && ((uintptr_t)out & 15) == 0;
  auto go = [&](auto dt, auto rows) {
    const long long per = (long long)THREADS / lpr * rows.value;
    hipLaunchKernelGGL((embed_fwd_kernel<dt.value, rows.value>), dim3(grid_of((N + per - 1) / per)), dim3(THREADS), 0,
                       st, N, V, D, ld, token, table, scale, padding, out, lpr, past_cache);
  };
  auto by_rows = [&](auto dt) {
    // many rows: a lane has 4 of them under way (in a training step, 131072 rows of 2 KB from a table of 3500 rows:
    // 59 us, 68 with one; from one of 50001: 80 and 81; 10^6 rows of 512 bytes from 32000: 138 and 158.  Lookups
    // alone: 49 and 46, 60 and 59, 94 and 105), else as many waves as there are (32768 rows of 2 KB, alone: 15.6
    // us, 16.7 with four)
    if (N * lpr >= (1LL << 22)) go(dt, std::integral_constant<int, 4>());
    else go(dt, std::integral_constant<int, 1>());
  };
  if (dtype == S2C_F32) by_rows(std::integral_constant<int, S2C_F32>());
  else if (dtype == S2C_BF16) by_rows(std::integral_constant<int, S2C_BF16>());
  else by_rows(std::integral_constant<int, S2C_F16>());
  return launched("embed_fwd");
}

// Looking through the tokens is one launch; where a word has many places its wave reads them alone, so
// only few tokens (256 tokens, 3500 words of 300 columns: 4.5 us; the sort's three launches: 15.4 us).
static bool by_scan(long long N, int V) { return N <= STAGE && N * V <= (1LL << 26); }

static long long align16(long long n) { return (n + 15) & ~15LL; }

static int pieces_of(int D, int vec) { return (D + 64 * vec - 1) / (64 * vec); }

// About 4096 waves, and 64 places (a lane each) at most: shorter chunks leave more partial sums (131072
// rows of 1024 bf16: runs 82 + join 10 us, 98 + 12 us with twice the waves).
static int chunk_of(long long N, int D) {
  const long long want = N * pieces_of(D, 8) / 4096;
  return want >= 64 ? 64 : want >= 32 ? 32 : want >= 16 ? 16 : 8;
}

// key and place twice, the histograms, the chunks' partial sums
extern "C" long long s2c_embed_grad_workspace_bytes(long long N, int V, int D) {
  if (N <= 0 || V <= 0 || D <= 0 || by_scan(N, V)) return 0;
  const int chunk = chunk_of(N, D);
  return 4 * align16(4 * N) + 4LL * RADIX * MAX_SORT_GRID +
         8 * ((N + chunk - 1) / chunk) * ((D + 7) & ~7);
}

template <int DT>
static void grad_launch(GradArgs &a, bool scan, hipStream_t st) {
  const dim3 block(THREADS);
  a.pieces = pieces_of(a.D, Elem<DT>::VEC);
  a.ldp = (a.D + 7) & ~7;
  if (scan) {
    const long long units = (long long)a.V * a.pieces;
    hipLaunchKernelGGL((embed_grad_scan_kernel<DT>), dim3(grid_of((units + WAVES - 1) / WAVES)), block, 0, st, a);
    return;
  }
  const long long chunks = (a.N + a.chunk - 1) / a.chunk;
  const int sums = grid_of((chunks * a.pieces + WAVES - 1) / WAVES);
  const long long absent = ((long long)a.V + WORDS - 1) / WORDS * ((a.pieces + GROUP - 1) / GROUP);
  hipLaunchKernelGGL((embed_runs_kernel<DT>), dim3(sums + (int)(absent < 65536 ? absent : 65536)), block, 0, st, a, sums);
  if (chunks > 1)
    hipLaunchKernelGGL((embed_join_kernel<DT>), dim3(min(grid_of((chunks + JOIN_WAVES - 1) / JOIN_WAVES * a.pieces), 1 << 16)),
                       dim3(64 * JOIN_WAVES), 0, st, a);
}

static void sort_tokens(GradArgs &a, u32 *const *key, u32 *const *pos, u32 *counts, hipStream_t st) {
  int total = 1;
  while (total < 32 && ((u32)a.V >> total) != 0) ++total;              // the key V has this many bits
  const int passes = (total + 7) / 8, bits = (total + passes - 1) / passes;
  if (a.N <= SMALL) {
    a.key = key[0];
    a.pos = pos[0];
    const dim3 one(1), block(SMALL_THREADS);
    if (a.N <= 2 * SMALL_THREADS) hipLaunchKernelGGL(sort_small_kernel<2>, one, block, 0, st, a, passes, bits);
    else if (a.N <= 4 * SMALL_THREADS) hipLaunchKernelGGL(sort_small_kernel<4>, one, block, 0, st, a, passes, bits);
    else hipLaunchKernelGGL(sort_small_kernel<8>, one, block, 0, st, a, passes, bits);
    return;
  }
  const long long tiles = (a.N + TILE - 1) / TILE, per = (tiles + MAX_SORT_GRID - 1) / MAX_SORT_GRID * TILE;
  const dim3 grid((int)((a.N + per - 1) / per)), block(THREADS);
  SortArgs s = {};
  s.N = a.N;
  s.per = per;
  s.bits = bits;
  s.padding = a.padding;
  s.V = a.V;
  s.counts = counts;
  for (int p = 0; p < passes; ++p) {
    s.token = p == 0 ? a.token : nullptr;
    s.shift = p * bits;
    s.key_in = key[(p + 1) & 1];
    s.pos_in = pos[(p + 1) & 1];
    s.key_out = key[p & 1];
    s.pos_out = pos[p & 1];
    hipLaunchKernelGGL(sort_count_kernel, grid, block, 0, st, s);
    hipLaunchKernelGGL(sort_scatter_kernel, grid, block, 0, st, s);
  }
  a.key = key[(passes - 1) & 1];
  a.pos = pos[(passes - 1) & 1];
}

extern "C" int s2c_embed_grad(long long N, int V, int D, int dtype, long long ldg, const long long *token,
                              const void *g, float scale, long long padding, void *d_table, void *ws,
                              void *stream) {
  if (N < 0 || N >= (1LL << 31) || V <= 0 || D <= 0 || D > S2C_WORDS_MAX_DIM || dtype < 0 || dtype > 2 ||
      ldg < 0 || bad_array(d_table, dtype))
    return S2C_EINVAL;
  if (N > 0 && (!token || bad_array(g, dtype))) return S2C_EINVAL;
  const bool scan = by_scan(N, V);
  if (!scan && (!ws || ((uintptr_t)ws & 15))) return S2C_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  GradArgs a = {};
  a.N = N;
  a.ldg = ldg;
  a.padding = padding;
  a.V = V;
  a.D = D;
  a.scale = scale;
  a.token = token;
  a.g = g;
  a.dt = d_table;
  a.chunk = chunk_of(N, D);
  if (!scan) {
    char *p = (char *)ws;
    u32 *key[2], *pos[2];
    for (int i = 0; i < 2; ++i) {
      key[i] = (u32 *)p;
      pos[i] = (u32 *)(p + align16(4 * N));
      p += 2 * align16(4 * N);
    }
    u32 *counts = (u32 *)p;
    p += 4LL * RADIX * MAX_SORT_GRID;
    a.partial = (float *)p;
    sort_tokens(a, key, pos, counts, st);
  }
  if (dtype == S2C_F32) grad_launch<S2C_F32>(a, scan, st);
  else if (dtype == S2C_BF16) grad_launch<S2C_BF16>(a, scan, st);
  else grad_launch<S2C_F16>(a, scan, st);
  return launched("embed_grad");
}
