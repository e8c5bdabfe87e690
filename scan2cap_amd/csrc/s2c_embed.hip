// s2c_embed.hip -- embedding lookup with scaling (s2c_embed_fwd) and the table's gradient
// (s2c_embed_grad).
//
// Lookup: out[n] = scale table[token[n]], one rounding; bound by writing N D elements and reading the
// distinct rows.
// Gradient: d_table[v] = scale sum_{n: token[n] = v} g[n]; every row is written, so the floor is reading
// N D and writing V D elements.  A wave owns a row's stretch of columns and adds the row's places in
// their order in 32-bit registers: no atomics, the same bits every time.
#include "s2c_words_common.h"

#include <stdio.h>

using namespace s2c;

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;

// VEC elements of a row that ends at D, from column col
template <int DT>
__device__ __forceinline__ Raw load_part(const void *p, long long i, int valid) {
  typedef Elem<DT> E;
  Raw r = {{0u, 0u, 0u, 0u}};
  if (valid >= E::VEC) return load16<DT>(p, i);
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

// LPR lanes per row (a power of two <= 64), 64 / LPR rows per wave
template <int DT>
__global__ __launch_bounds__(THREADS) void embed_fwd_kernel(long long N, int V, int D, long long ld,
                                                            const long long *__restrict__ token,
                                                            const void *__restrict__ table, float scale,
                                                            long long padding, void *__restrict__ out,
                                                            int lpr) {
  typedef Elem<DT> E;
  const int sub = threadIdx.x & (lpr - 1);
  const long long rows = (long long)gridDim.x * (THREADS / lpr);
  for (long long n = (long long)blockIdx.x * (THREADS / lpr) + threadIdx.x / lpr; n < N; n += rows) {
    const long long t = token[n];
    const bool pad = t == padding, bad = !pad && (t < 0 || t >= V);
    const float fill = bad ? NAN : 0.0f;
    for (int c = sub * E::VEC; c < D; c += lpr * E::VEC) {
      float f[E::VEC];
      if (pad || bad) {
#pragma unroll
        for (int e = 0; e < E::VEC; ++e) f[e] = fill;
      } else {
        const Raw r = load_part<DT>(table, t * ld + c, D - c);
#pragma unroll
        for (int e = 0; e < E::VEC; ++e) f[e] = scale * E::at(r, e);
      }
      store_part<DT>(out, n * D + c, D - c, f);
    }
  }
}

constexpr int STAGE = 2048;       // tokens looked through at a time

template <int DT>
__global__ __launch_bounds__(THREADS) void embed_grad_kernel(long long N, int V, int D, long long ldg,
                                                             const long long *__restrict__ token,
                                                             const void *__restrict__ g, float scale,
                                                             long long padding, void *__restrict__ dt,
                                                             int chunks) {
  typedef Elem<DT> E;
  __shared__ int s_tok[STAGE];
  const int lane = lane_id(), w = threadIdx.x >> 6;
  const long long units = (long long)V * chunks;
  for (long long u0 = (long long)blockIdx.x * WAVES; u0 < units; u0 += (long long)gridDim.x * WAVES) {
    const long long un = u0 + w;
    const int v = (int)(un / chunks), c = (int)(un % chunks) * 64 * E::VEC + lane * E::VEC;
    float acc[E::VEC];
#pragma unroll
    for (int e = 0; e < E::VEC; ++e) acc[e] = 0.0f;
    for (long long n0 = 0; n0 < N; n0 += STAGE) {
      __syncthreads();
      for (int i = threadIdx.x; i < STAGE; i += THREADS) {
        int id = -1;
        if (n0 + i < N) {
          const long long t = token[n0 + i];
          if (t != padding && t >= 0 && t < V) id = (int)t;
        }
        s_tok[i] = id;
      }
      __syncthreads();
      if (un < units) {
        for (int i0 = 0; i0 < STAGE; i0 += 64) {
          u64 mask = __ballot(s_tok[i0 + lane] == v);
          while (mask) {
            const int b = __builtin_ctzll(mask);
            mask &= mask - 1;
            if (c < D) {
              const Raw r = load_part<DT>(g, (n0 + i0 + b) * ldg + c, D - c);
#pragma unroll
              for (int e = 0; e < E::VEC; ++e) acc[e] += E::at(r, e);
            }
          }
        }
      }
    }
    if (un < units && c < D) {
#pragma unroll
      for (int e = 0; e < E::VEC; ++e) acc[e] *= scale;
      store_part<DT>(dt, (long long)v * D + c, D - c, acc);
    }
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
  const dim3 grid(grid_of((N * lpr + THREADS - 1) / THREADS)), block(THREADS);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == S2C_F32)
    hipLaunchKernelGGL(embed_fwd_kernel<S2C_F32>, grid, block, 0, st, N, V, D, ld, token, table, scale, padding, out, lpr);
  else if (dtype == S2C_BF16)
    hipLaunchKernelGGL(embed_fwd_kernel<S2C_BF16>, grid, block, 0, st, N, V, D, ld, token, table, scale, padding, out, lpr);
  else
    hipLaunchKernelGGL(embed_fwd_kernel<S2C_F16>, grid, block, 0, st, N, V, D, ld, token, table, scale, padding, out, lpr);
  return launched("embed_fwd");
}

extern "C" long long s2c_embed_grad_workspace_bytes(long long, int, int) { return 0; }

extern "C" int s2c_embed_grad(long long N, int V, int D, int dtype, long long ldg, const long long *token,
                              const void *g, float scale, long long padding, void *d_table, void *,
                              void *stream) {
  if (N < 0 || V <= 0 || D <= 0 || D > S2C_WORDS_MAX_DIM || dtype < 0 || dtype > 2 || ldg < 0 || bad_array(d_table, dtype))
    return S2C_EINVAL;
  if (N > 0 && (!token || bad_array(g, dtype))) return S2C_EINVAL;
  const int cols = 64 * (dtype == S2C_F32 ? 4 : 8);
  const int chunks = (D + cols - 1) / cols;
  const dim3 grid(grid_of(((long long)V * chunks + WAVES - 1) / WAVES)), block(THREADS);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == S2C_F32)
    hipLaunchKernelGGL(embed_grad_kernel<S2C_F32>, grid, block, 0, st, N, V, D, ldg, token, g, scale, padding, d_table, chunks);
  else if (dtype == S2C_BF16)
    hipLaunchKernelGGL(embed_grad_kernel<S2C_BF16>, grid, block, 0, st, N, V, D, ldg, token, g, scale, padding, d_table, chunks);
  else
    hipLaunchKernelGGL(embed_grad_kernel<S2C_F16>, grid, block, 0, st, N, V, D, ldg, token, g, scale, padding, d_table, chunks);
  return launched("embed_grad");
}
