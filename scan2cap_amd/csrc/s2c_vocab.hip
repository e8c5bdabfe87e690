// s2c_vocab.hip -- softmax statistics of word logits: token log probabilities with entropy and the
// best alternatives (s2c_token_scores_*), distillation from a teacher's top logits (s2c_distill_*).
//
// Both need, per row, m = max x, s0 = sum 2^d and (scores) s1 = sum 2^d d with d = (x - m) c,
// c = inv_t log2 e:
//   log p_v = (x_v - m) inv_t - ln 2 log2 s0        entropy = -sum p log p = ln 2 (log2 s0 - s1 / s0)
// in ONE pass: every lane keeps its own running (m, s0, s1); a larger m rescales s0' = a s0,
// s1' = a (s1 + delta s0) with delta = (m_old - m_new) c, a = 2^delta.  x - m is formed before the
// product with c: type-lowest masks (-3.4e38) would overflow in x c, and a row of nothing but them is
// uniform.  -inf contributes e = 0 (its d is held at -160, whose 2^d is 0, so that 0 * d is 0).
// NaN and +inf reach s0 and with it every output of the row.
//
// The k best: keys (order-preserving 32 bits of the value | ~index) make equal values unique, lowest
// index first.  A wave keeps candidates in LDS and a threshold tau: the k-th best value it is sure of.
// The first tile takes tau from the 64 lanes' tile maxima (k-th largest of them, a binary search over
// ballots), later tiles are entered only if some lane's tile maximum is above tau, and the buffer is cut
// back to its k best, by counting ranks, when it fills.  Later elements equal to tau lose their tie: a
// wave walks its tiles in index order.
//
// All of it is bound by reading the logits (and, backward, reading them again and writing the
// gradient).
#include "s2c_words_common.h"

#include <limits.h>
#include <stdio.h>

using namespace s2c;

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr int KMAX = S2C_WORDS_MAX_TOP;
constexpr int SLOTS = S2C_WORDS_MAX_SLOTS;
constexpr int BUF = 192;          // candidates of a wave: cut back when more than BUF - 64 are held
constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int U = 4;              // 16-byte loads in flight per lane

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
constexpr float D_MIN = -160.0f;

__device__ __forceinline__ const char *row_ptr(const s2c_logits &lg, int es, int r) {
  const int i2 = r % lg.n2, t = r / lg.n2, i1 = t % lg.n1, i0 = t / lg.n1;
  return (const char *)lg.x + es * (i0 * lg.s0 + i1 * lg.s1 + i2 * lg.s2);
}

// ---- order-preserving keys ---------------------------------------------------------------------------
__device__ __forceinline__ u32 ord(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const u32 b = __builtin_bit_cast(u32, x + 0.0f);        // -0 -> +0
  return b ^ ((u32)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unord(u32 k) {
  return __builtin_bit_cast(float, (k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
// !(x <= above(k))  <=>  ord(x) > k
__device__ __forceinline__ float above(u32 k) { return unord(k); }
// !(x <= from(k))  <=>  ord(x) >= k   (0x7FFFFFFF would be -0, which compares equal to +0)
__device__ __forceinline__ float from(u32 k) {
  u32 t = k ? k - 1 : 0;
  if (t == 0x7FFFFFFFu) --t;
  return unord(t);
}
// a lower bound of the k-th largest of the 64 lanes' keys, its upper 20 bits (0: fewer than k keys)
__device__ __forceinline__ u32 kth_of_lanes(u32 key, int k) {
  u32 cur = 0;
#pragma unroll
  for (int b = 31; b >= 12; --b) {
    const u32 trial = cur | (1u << b);
    if (__popcll(__ballot(key >= trial)) >= k) cur = trial;
  }
  return cur;
}

// a wave's candidates (LDS)
struct Best {
  u64 *buf;
  int cnt, k;
  u32 tau;           // keys above tau are wanted
  u64 kth;           // the k-th best key held after the last cut, 0 if fewer are held

  __device__ __forceinline__ void init(u64 *b, int k_) { buf = b; k = k_; cnt = 0; tau = 0; kth = 0; }

  // keep the k best, in descending order
  __device__ __forceinline__ void cut(int lane) {
    wave_lds_fence();
    u64 e[3];
    int rank[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < 3; ++i) e[i] = lane + 64 * i < cnt ? buf[lane + 64 * i] : 0;
    for (int j = 0; j < cnt; ++j) {
      const u64 o = buf[j];
#pragma unroll
      for (int i = 0; i < 3; ++i) rank[i] += o > e[i];
    }
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (lane + 64 * i < cnt && rank[i] < k) buf[rank[i]] = e[i];
    wave_lds_fence();
    if (cnt >= k) {
      cnt = k;
      kth = buf[k - 1];
      const u32 t = (u32)(kth >> 32);
      if (t > tau) tau = t;
    }
  }
  // lanes with `f` add `key`; true if the buffer was cut for it
  __device__ __forceinline__ bool add(u64 mask, u64 key, int lane) {
    bool was_cut = false;
    if (cnt > BUF - 64) { cut(lane); was_cut = true; }
    if ((mask >> lane) & 1) buf[cnt + mask_rank_below(mask)] = key;
    cnt += __popcll(mask);
    return was_cut;
  }
};

// the k best of L (a power of two <= 64) sorted lists, key(list, pos); 64 / L places of every list at a
// time, so that a round that adds nothing ends it.  b.buf holds them in descending order afterwards.
template <class F>
__device__ __forceinline__ void merge_lists(Best &b, int L, int lane, F key) {
  const int ppl = 64 / L;
  const int list = lane & (L - 1), sub = lane / L;
  u64 thr = 0;
  for (int p0 = 0; p0 < b.k; p0 += ppl) {
    const int pos = p0 + sub;
    const u64 v = pos < b.k ? key(list, pos) : 0;
    if (p0 == 0) {
      const u32 cur = kth_of_lanes((u32)(v >> 32), b.k);
      thr = cur ? ((u64)cur << 32) - 1 : 0;
    }
    const u64 mask = __ballot(v > thr);
    if (mask == 0) break;
    if (b.add(mask, v, lane) && b.kth) thr = b.kth;
  }
  b.cut(lane);
}

// ---- per-row softmax statistics --------------------------------------------------------------------------
struct Stat { float m, s0, s1; };

__device__ __forceinline__ float finite_or_0(float m) { return m == -INFINITY ? 0.0f : m; }

// combine the lanes' statistics; every lane gets the result
__device__ __forceinline__ Stat wave_combine(Stat s, float c) {
  const float m = wave_max(s.m);
  const float delta = fmaxf((s.m - m) * c, D_MIN), a = exp2_(delta);
  Stat o;
  o.m = m;
  o.s1 = wave_sum(a * (s.s1 + delta * s.s0));
  o.s0 = wave_sum(a * s.s0);
  return o;
}

// one wave's share of a row: tiles of 64 U vectors, wave `w` of `nw`, vectors [vb, ve) of the row
template <int DT, bool TOP, bool ENT>
__device__ __forceinline__ Stat stream_row(const char *xr, int V, int vb, int ve, int w, int nw, float c,
                                           Best &best) {
  typedef Elem<DT> E;
  constexpr int VEC = E::VEC;
  const int lane = lane_id();
  const int shift = (int)(((uintptr_t)xr / E::ES) & (VEC - 1));   // vector i = elements i VEC - shift ..
  Stat s = {-INFINITY, 0.0f, 0.0f};
  bool first = true;
  for (int t0 = vb + w * 64 * U; t0 < ve; t0 += nw * 64 * U) {
    Raw r[U];
    if ((long long)t0 * VEC - shift >= 0 && (long long)(t0 + 64 * U) * VEC - shift <= V && t0 + 64 * U <= ve) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        r[u] = *reinterpret_cast<const Raw *>(xr + ((long long)(t0 + u * 64 + lane) * VEC - shift) * E::ES);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int vi = t0 + u * 64 + lane;
        const long long e0 = (long long)vi * VEC - shift;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[u].w[i] = E::NEG_INF;
        if (vi < ve) {
          if (e0 >= 0 && e0 + VEC <= V) {
            r[u] = *reinterpret_cast<const Raw *>(xr + e0 * E::ES);
          } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
              if (e0 + e >= 0 && e0 + e < V) E::put(r[u], e, E::bits(xr, e0 + e));
          }
        }
      }
    }
    float tmax = E::at(r[0], 0);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) tmax = nan_max(tmax, E::at(r[u], e));

    if (TOP) {
      bool enter = true;
      float thr;
      u32 next = best.tau;
      if (first) {
        const long long e0 = (long long)(t0 + lane) * VEC - shift;     // the lane's lowest element
        const bool any = t0 + lane < ve && e0 < V;
        next = kth_of_lanes(any ? ord(tmax) : 0u, best.k);
        thr = from(next);
      } else {
        thr = above(best.tau);
        enter = __ballot(!(tmax <= thr)) != 0;
      }
      if (enter) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float v = E::at(r[u], e);
            u64 mask = __ballot(!(v <= thr));
            if (mask) {
              const int vi = t0 + u * 64 + lane;
              const long long idx = (long long)vi * VEC - shift + e;
              mask &= __ballot(vi < ve && idx >= 0 && idx < V);
              const u64 key = ((u64)ord(v) << 32) | (u32)~(u32)idx;
              // after a cut inside a tile, elements equal to the new tau may still win by their index
              if (mask && best.add(mask, key, lane)) thr = from(best.tau > next ? best.tau : next);
            }
          }
        }
      }
      if (next > best.tau) best.tau = next;
      first = false;
    }

    const float m_new = nan_max(s.m, tmax);
    const float delta = fmaxf((s.m - m_new) * c, D_MIN), a = exp2_(delta);
    const float mref = finite_or_0(m_new);
    s.s1 = a * (s.s1 + delta * s.s0);
    s.s0 = a * s.s0;
    s.m = m_new;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float p0 = 0.0f, p1 = 0.0f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = (E::at(r[u], e) - mref) * c;
        const float ex = exp2_(d);
        p0 += ex;
        if (ENT) p1 = __builtin_fmaf(ex, fmaxf(d, D_MIN), p1);
      }
      s.s0 += p0;
      if (ENT) s.s1 += p1;
    }
  }
  return wave_combine(s, c);
}

// ---- what is written for a row ---------------------------------------------------------------------------
// stats: {mref, log2 s0, ., .}; log2 s0 = +inf marks a row without gradient, NaN one whose gradient is NaN
__device__ __forceinline__ float log2_sum(const Stat &s) {
  return s.s0 == 0.0f ? INFINITY : log2f(s.s0);        // (0: every logit is -inf)
}

__device__ __forceinline__ bool scores_dead(const s2c_token_scores_args &a, int r) {
  return a.has_ignore && a.token && a.token[r] == a.ignore;
}

__device__ __forceinline__ void scores_write_dead(const s2c_token_scores_args &a, int r, int lane) {
  if (lane == 0) {
    if (a.logp) a.logp[r] = 0.0f;
    a.entropy[r] = 0.0f;
    *reinterpret_cast<float4 *>(a.stats + 4 * (size_t)r) = make_float4(0.0f, INFINITY, 0.0f, 0.0f);
  }
  for (int j = lane; j < a.k; j += 64) {
    a.top_logp[(size_t)r * a.k + j] = 0.0f;
    a.top_ids[(size_t)r * a.k + j] = -1;
  }
}

template <int DT>
__device__ __forceinline__ void scores_write(const s2c_token_scores_args &a, int r, const char *xr,
                                             const Stat &s, const u64 *top, int lane) {
  const float mref = finite_or_0(s.m);
  const float l2s = log2_sum(s);
  const bool dead = l2s == INFINITY;
  const float sub = dead ? 0.0f : l2s;
  const float h = dead ? 0.0f : LN2 * (l2s - s.s1 / s.s0);
  if (lane == 0) {
    bool bad = false;
    if (a.token) {
      const long long t = a.token[r];
      bad = t < 0 || t >= a.lg.V;
      a.logp[r] = bad ? NAN : (Elem<DT>::load(xr, bad ? 0 : t) - mref) * a.lg.inv_t - LN2 * sub;
    }
    a.entropy[r] = h < 0.0f ? 0.0f : h;
    *reinterpret_cast<float4 *>(a.stats + 4 * (size_t)r) =
        make_float4(mref, bad ? NAN : l2s, h < 0.0f ? 0.0f : h, 0.0f);
  }
  if (lane < a.k) {
    const u64 key = top[lane];
    a.top_logp[(size_t)r * a.k + lane] = (unord((u32)(key >> 32)) - mref) * a.lg.inv_t - LN2 * sub;
    a.top_ids[(size_t)r * a.k + lane] = (long long)(u32)~(u32)key;
  }
}

template <int DT>
__global__ __launch_bounds__(THREADS) void scores_fwd_kernel(s2c_token_scores_args a) {
  __shared__ u64 s_buf[WAVES + 1][BUF];
  __shared__ Stat s_part[WAVES];
  const int lane = lane_id(), w = threadIdx.x >> 6;
  const float c = a.lg.inv_t * LOG2E;
  for (int r = blockIdx.x; r < a.lg.rows; r += gridDim.x) {
    if (scores_dead(a, r)) {
      if (w == 0) scores_write_dead(a, r, lane);
      continue;
    }
    const char *xr = row_ptr(a.lg, Elem<DT>::ES, r);
    const int shift = (int)(((uintptr_t)xr / Elem<DT>::ES) & (Elem<DT>::VEC - 1));
    const int nvec = (int)(((long long)a.lg.V + shift + Elem<DT>::VEC - 1) / Elem<DT>::VEC);
    Best best;
    best.init(s_buf[w], a.k);
    Stat s;
    if (a.k) {
      s = stream_row<DT, true, true>(xr, a.lg.V, 0, nvec, w, WAVES, c, best);
      best.cut(lane);
      for (int j = best.cnt + lane; j < a.k; j += 64) s_buf[w][j] = 0;
    } else {
      s = stream_row<DT, false, true>(xr, a.lg.V, 0, nvec, w, WAVES, c, best);
    }
    if (lane == 0) s_part[w] = s;
    __syncthreads();
    if (w == 0) {
      Stat o = {-INFINITY, 0.0f, 0.0f};
      if (lane < WAVES) o = s_part[lane];
      o = wave_combine(o, c);
      if (a.k) {
        Best all;
        all.init(s_buf[WAVES], a.k);
        merge_lists(all, WAVES, lane, [&](int list, int pos) { return s_buf[list][pos]; });
      }
      scores_write<DT>(a, r, xr, o, s_buf[WAVES], lane);
    }
    __syncthreads();
  }
}

// ---- distillation --------------------------------------------------------------------------------------
// the teacher's softmax over a row's slots, slot j of lane l = l + 64 i: log q and q
struct Slots {
  long long id[SLOTS / 64];
  float lq[SLOTS / 64], q[SLOTS / 64];
  float wm, l2w;          // l2w = +inf: no slot is used
};

__device__ __forceinline__ Slots load_slots(const s2c_distill_args &a, int r, float c, int lane) {
  Slots s;
  float w[SLOTS / 64];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < SLOTS / 64; ++i) {
    const int j = lane + 64 * i;
    s.id[i] = -1;
    w[i] = -INFINITY;
    if (j < a.K) {
      s.id[i] = a.ids[(size_t)r * a.K + j];
      if (s.id[i] >= 0) w[i] = load_any(a.teacher, (long long)r * a.K + j, a.teacher_dtype);
    }
    m = nan_max(m, w[i]);
  }
  s.wm = finite_or_0(wave_max(m));
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < SLOTS / 64; ++i) sum += exp2_((w[i] - s.wm) * c);
  sum = wave_sum(sum);
  s.l2w = sum == 0.0f ? INFINITY : log2f(sum);
#pragma unroll
  for (int i = 0; i < SLOTS / 64; ++i) {
    s.lq[i] = (w[i] - s.wm) * a.lg.inv_t - LN2 * s.l2w;
    s.q[i] = exp2_((w[i] - s.wm) * c - s.l2w);
  }
  return s;
}

__device__ __forceinline__ void distill_write_dead(const s2c_distill_args &a, int r, int lane) {
  if (lane == 0) {
    a.loss[r] = 0.0f;
    *reinterpret_cast<float4 *>(a.stats + 4 * (size_t)r) = make_float4(0.0f, INFINITY, 0.0f, INFINITY);
  }
}

template <int DT>
__device__ __forceinline__ void distill_write(const s2c_distill_args &a, int r, const char *xr,
                                              const Stat &s, const Slots &t, int lane) {
  const float mref = finite_or_0(s.m);
  const float l2s = log2_sum(s);
  const float sub = l2s == INFINITY ? 0.0f : l2s;
  float part = 0.0f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < SLOTS / 64; ++i) {
    if (t.q[i] != 0.0f) {                       // (empty slots and vanishing ones add nothing; NaN does)
      if (t.id[i] >= a.lg.V) bad = true;
      else part += t.q[i] * (t.lq[i] - ((Elem<DT>::load(xr, t.id[i]) - mref) * a.lg.inv_t - LN2 * sub));
    }
  }
  part = wave_sum(part);
  bad = __ballot(bad) != 0;
  if (lane == 0) {
    a.loss[r] = bad ? NAN : part;
    *reinterpret_cast<float4 *>(a.stats + 4 * (size_t)r) = make_float4(mref, bad ? NAN : l2s, t.wm, t.l2w);
  }
}

template <int DT>
__global__ __launch_bounds__(THREADS) void distill_fwd_kernel(s2c_distill_args a) {
  __shared__ Stat s_part[WAVES];
  const int lane = lane_id(), w = threadIdx.x >> 6;
  const float c = a.lg.inv_t * LOG2E;
  for (int r = blockIdx.x; r < a.lg.rows; r += gridDim.x) {
    bool dead = a.mask && a.mask[r] == 0;
    Slots t;
    if (!dead) {
      t = load_slots(a, r, c, lane);
      dead = t.l2w == INFINITY;
    }
    if (dead) {
      if (w == 0) distill_write_dead(a, r, lane);
      continue;
    }
    const char *xr = row_ptr(a.lg, Elem<DT>::ES, r);
    const int shift = (int)(((uintptr_t)xr / Elem<DT>::ES) & (Elem<DT>::VEC - 1));
    const int nvec = (int)(((long long)a.lg.V + shift + Elem<DT>::VEC - 1) / Elem<DT>::VEC);
    Best none;
    const Stat s = stream_row<DT, false, false>(xr, a.lg.V, 0, nvec, w, WAVES, c, none);
    if (lane == 0) s_part[w] = s;
    __syncthreads();
    if (w == 0) {
      Stat o = {-INFINITY, 0.0f, 0.0f};
      if (lane < WAVES) o = s_part[lane];
      distill_write<DT>(a, r, xr, wave_combine(o, c), t, lane);
    }
    __syncthreads();
  }
}

// ---- gradients -------------------------------------------------------------------------------------------
// dx_v = p_v (A + B max(d_v - log2 s0, D_MIN)) + the sparse entries of v:
//   scores  A = -(g + sum g_top + g_H H) inv_t, B = -g_H ln 2 inv_t, entries g inv_t at the token and
//           g_top_j inv_t at top_ids_j
//   distill A = g inv_t, B = 0, entries -g q_j inv_t at id_j
// A workgroup writes the dense part of a stretch of a row, then the first entry of every word in the
// stretch recomputes that element with all entries of the same word added, in slot order, and stores it
// again (rounded once; no atomics).
template <int DT>
__device__ __forceinline__ void dense_row(const char *xr, void *dx, long long o0, int V, int vb, int ve,
                                          int shift, float mref, float l2s, float A, float B, float c) {
  typedef Elem<DT> E;
  constexpr int VEC = E::VEC;
  auto grad = [&](float x) {
    const float d = (x - mref) * c - l2s;
    return exp2_(d) * __builtin_fmaf(B, fmaxf(d, D_MIN), A);
  };
  for (int vi = vb + (int)threadIdx.x; vi < ve; vi += THREADS) {
    const long long e0 = (long long)vi * VEC - shift;
    if (e0 >= 0 && e0 + VEC <= V) {
      const Raw r = load16<DT>(xr, e0);
      float f[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = grad(E::at(r, e));
      store16<DT>(dx, o0 + e0, E::pack(f));
    } else {
      for (int e = 0; e < VEC; ++e)
        if (e0 + e >= 0 && e0 + e < V) E::store(dx, o0 + e0 + e, grad(E::load(xr, e0 + e)));
    }
  }
}

template <int DT>
__device__ __forceinline__ void zero_row(void *dx, long long o0, int V, int vb, int ve, int shift) {
  typedef Elem<DT> E;
  constexpr int VEC = E::VEC;
  const Raw z = {{0u, 0u, 0u, 0u}};
  for (int vi = vb + (int)threadIdx.x; vi < ve; vi += THREADS) {
    const long long e0 = (long long)vi * VEC - shift;
    if (e0 >= 0 && e0 + VEC <= V) {
      store16<DT>(dx, o0 + e0, z);
    } else {
      for (int e = 0; e < VEC; ++e)
        if (e0 + e >= 0 && e0 + e < V) E::store(dx, o0 + e0 + e, 0.0f);
    }
  }
}

template <int DT>
__device__ __forceinline__ void sparse_row(const char *xr, void *dx, long long o0, int V, int vb, int ve,
                                           int shift, float mref, float l2s, float A, float B, float c,
                                           const int *s_id, const float *s_val, int n) {
  typedef Elem<DT> E;
  for (int j = threadIdx.x; j < n; j += THREADS) {
    const int id = s_id[j];
    if (id < 0 || id >= V) continue;
    const int vi = (int)(((long long)id + shift) / E::VEC);
    if (vi < vb || vi >= ve) continue;
    bool seen = false;
    for (int i = 0; i < j; ++i) seen |= s_id[i] == id;
    if (seen) continue;
    float sum = 0.0f;
    for (int i = j; i < n; ++i)
      if (s_id[i] == id) sum += s_val[i];
    const float d = (E::load(xr, id) - mref) * c - l2s;
    E::store(dx, o0 + id, exp2_(d) * __builtin_fmaf(B, fmaxf(d, D_MIN), A) + sum);
  }
}

struct GradArgs {
  s2c_logits lg;
  const float *stats;
  void *dx;
  int segs, vps;         // stretches per row, vectors per stretch
  // scores
  const long long *token, *top_ids;
  const float *g_logp, *g_entropy, *g_top;
  int k;
  // distillation
  const long long *ids;
  const void *teacher;
  const float *g_loss;
  int K, teacher_dtype;
};

template <int DT, bool DISTILL>
__global__ __launch_bounds__(THREADS) void vocab_bwd_kernel(GradArgs a) {
  __shared__ int s_id[SLOTS];
  __shared__ float s_val[SLOTS];
  static_assert(SLOTS >= KMAX + 1, "entries of a row");
  const int tid = threadIdx.x;
  const float c = a.lg.inv_t * LOG2E, it = a.lg.inv_t;
  const int V = a.lg.V;
  const long long units = (long long)a.lg.rows * a.segs;
  for (long long un = blockIdx.x; un < units; un += gridDim.x) {
    const int r = (int)(un / a.segs), seg = (int)(un % a.segs);
    const char *xr = row_ptr(a.lg, Elem<DT>::ES, r);
    const long long o0 = (long long)r * V;
    const int shift = (int)((((uintptr_t)a.dx / Elem<DT>::ES) + o0) & (Elem<DT>::VEC - 1));
    const int nvec = (int)(((long long)V + shift + Elem<DT>::VEC - 1) / Elem<DT>::VEC);
    const int vb = seg * a.vps, ve = min(nvec, vb + a.vps);
    const float4 st = *reinterpret_cast<const float4 *>(a.stats + 4 * (size_t)r);
    const float mref = st.x, l2s = st.y;
    if (l2s == INFINITY) {
      zero_row<DT>(a.dx, o0, V, vb, ve, shift);
      continue;
    }
    float A, B;
    int n = 0;
    if (DISTILL) {
      n = a.K;
      const float g = a.g_loss[r] * it;
      for (int j = tid; j < n; j += THREADS) {
        const long long id = a.ids[(size_t)r * n + j];
        s_id[j] = id < 0 ? -1 : (int)(id < V ? id : -1);
        s_val[j] = id < 0 ? 0.0f
                          : -g * exp2_((load_any(a.teacher, (long long)r * n + j, a.teacher_dtype) - st.z) * c - st.w);
      }
      __syncthreads();
      A = g;
      B = 0.0f;
    } else {
      const float g = (a.g_logp && a.token) ? a.g_logp[r] : 0.0f;
      const float ge = a.g_entropy ? a.g_entropy[r] : 0.0f;
      const int k = a.g_top ? a.k : 0;
      n = k + 1;
      if (tid == 0) {
        s_id[0] = a.token ? (int)a.token[r] : -1;
        s_val[0] = g * it;
      } else if (tid <= k) {
        s_id[tid] = (int)a.top_ids[(size_t)r * k + tid - 1];
        s_val[tid] = a.g_top[(size_t)r * k + tid - 1] * it;
      }
      __syncthreads();
      float sum = 0.0f;
      for (int j = 0; j < n; ++j) sum += s_val[j];
      A = -(sum + ge * st.z * it);
      B = -ge * LN2 * it;
    }
    dense_row<DT>(xr, a.dx, o0, V, vb, ve, shift, mref, l2s, A, B, c);
    __syncthreads();
    sparse_row<DT>(xr, a.dx, o0, V, vb, ve, shift, mref, l2s, A, B, c, s_id, s_val, n);
    __syncthreads();
  }
}

// ---- host --------------------------------------------------------------------------------------------------
int launched(const char *what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    fprintf(stderr, "s2c: %s launch failed: %s\n", what, hipGetErrorString(e));
    return (int)e;
  }
  return 0;
}

bool bad_logits(const s2c_logits &l) {
  return l.rows < 0 || l.V <= 0 || l.dtype < 0 || l.dtype > 2 || l.n1 <= 0 || l.n2 <= 0 ||
         !(l.inv_t > 0.0f) || l.inv_t > 3.0e38f || (l.rows > 0 && !l.x) ||
         ((uintptr_t)l.x & (l.dtype == S2C_F32 ? 3 : 1));
}

constexpr int MAX_GRID = 1 << 22;       // workgroups of 256: below 2^32 work-items

int grid_of(long long units) { return (int)(units < MAX_GRID ? units : MAX_GRID); }

template <bool DISTILL>
int backward(GradArgs &a, const char *what, hipStream_t st) {
  const int vec = a.lg.dtype == S2C_F32 ? 4 : 8;
  const long long nvec = ((long long)a.lg.V + 2 * vec - 2) / vec;      // at any alignment
  a.vps = 4 * THREADS;
  a.segs = (int)((nvec + a.vps - 1) / a.vps);
  const dim3 grid(grid_of((long long)a.lg.rows * a.segs)), block(THREADS);
  if (a.lg.dtype == S2C_F32) hipLaunchKernelGGL((vocab_bwd_kernel<S2C_F32, DISTILL>), grid, block, 0, st, a);
  else if (a.lg.dtype == S2C_BF16) hipLaunchKernelGGL((vocab_bwd_kernel<S2C_BF16, DISTILL>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((vocab_bwd_kernel<S2C_F16, DISTILL>), grid, block, 0, st, a);
  return launched(what);
}

bool bad_scores(const s2c_token_scores_args *a) {
  return !a || bad_logits(a->lg) || a->k < 0 || a->k > KMAX || a->k > a->lg.V || (a->k && !a->top_ids) ||
         !a->stats;
}

bool bad_distill(const s2c_distill_args *a) {
  return !a || bad_logits(a->lg) || a->K <= 0 || a->K > SLOTS || a->teacher_dtype < 0 ||
         a->teacher_dtype > 2 || !a->ids || !a->teacher || !a->stats;
}

}  // namespace

extern "C" long long s2c_words_args_sizeof(int which) {
  return which == 0 ? sizeof(s2c_logits) : which == 1 ? sizeof(s2c_token_scores_args)
         : which == 2 ? sizeof(s2c_distill_args) : 0;
}

extern "C" long long s2c_token_scores_workspace_bytes(int, int, int, int) { return 0; }

extern "C" int s2c_token_scores_fwd(const s2c_token_scores_args *a, void *stream) {
  if (bad_scores(a) || !a->entropy || (a->token && !a->logp) || (a->k && !a->top_logp)) return S2C_EINVAL;
  if (a->lg.rows == 0) return 0;
  const dim3 grid(grid_of(a->lg.rows)), block(THREADS);
  hipStream_t st = (hipStream_t)stream;
  if (a->lg.dtype == S2C_F32) hipLaunchKernelGGL(scores_fwd_kernel<S2C_F32>, grid, block, 0, st, *a);
  else if (a->lg.dtype == S2C_BF16) hipLaunchKernelGGL(scores_fwd_kernel<S2C_BF16>, grid, block, 0, st, *a);
  else hipLaunchKernelGGL(scores_fwd_kernel<S2C_F16>, grid, block, 0, st, *a);
  return launched("token_scores_fwd");
}

extern "C" int s2c_token_scores_bwd(const s2c_token_scores_args *a, const float *g_logp,
                                    const float *g_entropy, const float *g_top, void *dx, void *stream) {
  if (bad_scores(a) || !dx) return S2C_EINVAL;
  if (a->lg.rows == 0) return 0;
  GradArgs g = {};
  g.lg = a->lg;
  g.stats = a->stats;
  g.dx = dx;
  g.token = a->token;
  g.top_ids = a->top_ids;
  g.g_logp = g_logp;
  g.g_entropy = g_entropy;
  g.g_top = g_top;
  g.k = a->k;
  return backward<false>(g, "token_scores_bwd", (hipStream_t)stream);
}

extern "C" long long s2c_distill_workspace_bytes(int, int, int) { return 0; }

extern "C" int s2c_distill_fwd(const s2c_distill_args *a, void *stream) {
  if (bad_distill(a) || !a->loss) return S2C_EINVAL;
  if (a->lg.rows == 0) return 0;
  const dim3 grid(grid_of(a->lg.rows)), block(THREADS);
  hipStream_t st = (hipStream_t)stream;
  if (a->lg.dtype == S2C_F32) hipLaunchKernelGGL(distill_fwd_kernel<S2C_F32>, grid, block, 0, st, *a);
  else if (a->lg.dtype == S2C_BF16) hipLaunchKernelGGL(distill_fwd_kernel<S2C_BF16>, grid, block, 0, st, *a);
  else hipLaunchKernelGGL(distill_fwd_kernel<S2C_F16>, grid, block, 0, st, *a);
  return launched("distill_fwd");
}

extern "C" int s2c_distill_bwd(const s2c_distill_args *a, const float *g_loss, void *dx, void *stream) {
  if (bad_distill(a) || !g_loss || !dx) return S2C_EINVAL;
  if (a->lg.rows == 0) return 0;
  GradArgs g = {};
  g.lg = a->lg;
  g.stats = a->stats;
  g.dx = dx;
  g.ids = a->ids;
  g.teacher = a->teacher;
  g.g_loss = g_loss;
  g.K = a->K;
  g.teacher_dtype = a->teacher_dtype;
  return backward<true>(g, "distill_bwd", (hipStream_t)stream);
}
