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
// index first.  A wave keeps candidates in LDS and enters a tile only where some lane's tile maximum
// passes a threshold, a lower bound of the row's k-th best value.  The first bound is the k-th largest of
// 64 maxima (a binary search over ballots), each over one lane's elements in the first tiles of all waves
// of the group; an element equal to it may still win by its index.  When the buffer fills it is cut back
// to its k best, by counting ranks; later elements equal to a wave's own k-th have lost, since a wave
// walks its tiles in index order.
//
// All of it is bound by reading the logits and, backward, reading them again and writing the gradient; a
// copy of 1 GiB reaches 5.1 TB/s here.  Kernel times on MI355X: 59392 x 3500 fp32 with 5 alternatives 158 us
// (5.3 TB/s; 151 where nothing else runs between); 4096 x 50001 bf16 with 8 alternatives, a tenth of the rows
// ignored, 85 to 88 us forward (4.3 TB/s: about half of it is the VALU's, 8 instructions an element) and 126 us
// backward; distillation over 4096 x 65536 bf16 with 64 slots 115 us and 186 us (5.8 TB/s); one row of 32768 bf16
// words 7.4 us (a launch, a trip to memory and the selection's chain of ballots).
#include "s2c_words_common.h"

#include <stdio.h>

#include <type_traits>

using namespace s2c;

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr int KMAX = S2C_WORDS_MAX_TOP;
constexpr int SLOTS = S2C_WORDS_MAX_SLOTS;
constexpr int BUF = 192;          // candidates of a wave: cut back when more than BUF - 64 are held
constexpr int U = 4;              // 16-byte loads in flight per lane
constexpr int MAX_SPLIT = 64;     // stretches of a row (the lanes that join them)

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
constexpr float D_MIN = -160.0f;

__device__ __forceinline__ const char *row_ptr(const s2c_logits &lg, int es, int r) {
  if (lg.n2 == lg.rows) return (const char *)lg.x + es * (r * lg.s2);      // (no divisions for rows of one stride)
  const int i2 = r % lg.n2, t = r / lg.n2, i1 = t % lg.n1, i0 = t / lg.n1;
  return (const char *)lg.x + es * (i0 * lg.s0 + i1 * lg.s1 + i2 * lg.s2);
}

// a wave's number in its workgroup, in a scalar register: what follows from it (rows, addresses, conditions)
// is then computed once for the wave
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// unit `un` = (row, stretch) of rows in `n` stretches
__device__ __forceinline__ void row_and_stretch(long long un, int n, int &r, int &seg) {
  if (n == 1) {
    r = (int)un;
    seg = 0;
  } else {
    r = (int)(un / n);
    seg = (int)(un - (long long)r * n);
  }
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
// a lower bound of the k-th largest of the 64 lanes' keys, its upper 16 bits (0: fewer than k keys)
__device__ __forceinline__ u32 kth_of_lanes(u32 key, int k) {
  u32 cur = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const u32 trial = cur | (1u << b);
    if (__popcll(__ballot(key >= trial)) >= k) cur = trial;
  }
  return cur;
}

// a wave's candidates (LDS)
struct Best {
  u64 *buf;
  int cnt, k;
  u32 bound;         // keys below it are not wanted
  u64 kth;           // the k-th best key held at the last cut, 0 if fewer were held

  __device__ __forceinline__ void init(u64 *b, int k_) { buf = b; k = k_; cnt = 0; bound = 0; kth = 0; }
  // values that pass: !(x <= threshold)
  __device__ __forceinline__ float threshold() const {
    const u32 t = (u32)(kth >> 32);
    return kth && t >= bound ? above(t) : from(bound);
  }

  // keep the k best, in descending order: an entry's rank is the number of greater ones
  __device__ __forceinline__ void cut(int lane) {
    wave_lds_fence();
    u64 e[3];
    int rank[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < 3; ++i) e[i] = lane + 64 * i < cnt ? buf[lane + 64 * i] : 0;
    if (cnt <= 64) {            // the common case stays in registers
      for (int j = 0; j < cnt; j += 4) {                        // (lanes from cnt on hold 0)
#pragma unroll
        for (int q = 0; q < 4; ++q) rank[0] += readlane_u64(e[0], j + q) > e[0];
      }
    } else {
      for (int j = 0; j < cnt; ++j) {
        const u64 o = buf[j];
#pragma unroll
        for (int i = 0; i < 3; ++i) rank[i] += o > e[i];
      }
    }
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (lane + 64 * i < cnt && rank[i] < k) buf[rank[i]] = e[i];
    wave_lds_fence();
    if (cnt >= k) {
      cnt = k;
      kth = buf[k - 1];
    }
  }
  // the lanes of `mask` add `key`
  __device__ __forceinline__ void add(u64 mask, u64 key, int lane) {
    if (cnt > BUF - 64) {
      cut(lane);
      mask &= __ballot(key > kth);
    }
    if ((mask >> lane) & 1) buf[cnt + mask_rank_below(mask)] = key;
    cnt += __popcll(mask);
  }
};

// what the waves of a group share: their lane maxima, the number of their candidates
struct Shared {
  u32 max[64];
  int n;
};

// the k best of L (a power of two <= 64) sorted lists, key(list, pos); 64 / L places of every list at a
// time, so that a round that adds nothing ends it.  b.buf holds them in descending order afterwards.
template <class F>
__device__ __forceinline__ void merge_lists(Best &b, int L, int lane, F key) {
  const int ppl = 64 / L;
  const int list = lane & (L - 1), sub = lane / L;
  u64 thr = 0;
  u64 next = sub < b.k ? key(list, sub) : 0;
  for (int p0 = 0; p0 < b.k; p0 += ppl) {
    const u64 v = next;
    const int ahead = p0 + ppl + sub;
    next = ahead < b.k ? key(list, ahead) : 0;
    if (p0 == 0) {
      const u32 bound = kth_of_lanes((u32)(v >> 32), b.k);
      thr = bound ? ((u64)bound << 32) - 1 : 0;
    }
    const u64 mask = __ballot(v > thr);
    if (mask == 0) break;
    b.add(mask, v, lane);
    if (b.kth > thr) thr = b.kth;
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

// One tile of a row: 64 U vectors from vector t0.  INSIDE: all of it lies in the row and the stretch [.., ve),
// its loads carry no condition and are under way together; else `nu` of its U vectors a lane may.
template <int DT, int G, bool TOP, bool ENT, bool INSIDE>
__device__ __forceinline__ void stream_tile(const char *xr, int V, int shift, int t0, int ve, float c, bool first,
                                            Stat &s, Best &best, u32 *s_max) {
  typedef Elem<DT> E;
  constexpr int VEC = E::VEC;
  const int lane = lane_id();
  const int nu = INSIDE ? U : t0 < ve ? min(U, (ve - t0 + 63) >> 6) : 0;
  Raw r[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int vi = t0 + u * 64 + lane;
    const long long e0 = (long long)vi * VEC - shift;
    if (INSIDE) {
      r[u] = *reinterpret_cast<const Raw *>(xr + e0 * E::ES);
    } else {
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
  float tmax = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!INSIDE && u >= nu) break;
#pragma unroll
    for (int e = 0; e < VEC; ++e) tmax = nan_max(tmax, E::at(r[u], e));
  }

  if (TOP) {
    if (first) {
      const long long e0 = (long long)(t0 + lane) * VEC - shift;     // the lane's lowest element
      u32 key = t0 + lane < ve && e0 < V ? ord(tmax) : 0u;
      if (G > 1) {
        atomicMax(&s_max[lane], key);
        __syncthreads();
        key = s_max[lane];
      }
      best.bound = kth_of_lanes(key, best.k);
    }
    const float thr = best.threshold();
    const bool enter = __ballot(!(tmax <= thr)) != 0;
    if (enter && G > 1) {
      // few rows: what passes is rare and the code's length counts -- a mask of every lane's elements, then
      // one of each lane at a time, read again (512 rows of 32000 words, 8 alternatives: 13.4 us, 14.1 with the
      // elements unrolled as below).  A wave of its own per row meets more of them (59392 rows of 3500, 5
      // alternatives: 150 us unrolled, 155 to 161 with masks).
      u32 hits = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < VEC; ++e) hits |= (!(E::at(r[u], e) <= thr) ? 1u : 0u) << (u * VEC + e);
      while (__ballot(hits != 0)) {
        const int b = __builtin_ctz(hits | 0x80000000u);
        const int vi = t0 + (b / VEC) * 64 + lane;
        const u32 idx = (u32)vi * VEC - shift + (b & (VEC - 1));     // (negative: above V)
        const bool ok = hits != 0 && vi < ve && idx < (u32)V;
        const u64 key = ((u64)ord(ok ? E::load(xr, idx) : 0.0f) << 32) | (u32)~idx;
        const u64 mask = __ballot(ok && key > best.kth);
        hits &= hits - 1;
        if (mask) best.add(mask, key, lane);
      }
    }
    if (enter && G == 1) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!INSIDE && u >= nu) break;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float v = E::at(r[u], e);
          u64 mask = __ballot(!(v <= thr));
          if (mask) {
            const int vi = t0 + u * 64 + lane;
            const u32 idx = (u32)vi * VEC - shift + e;               // (negative: above V)
            const u64 key = ((u64)ord(v) << 32) | (u32)~idx;
            if (!INSIDE) mask &= __ballot(vi < ve && idx < (u32)V);
            if (best.kth) mask &= __ballot(key > best.kth);
            if (mask) best.add(mask, key, lane);
          }
        }
      }
    }
  }

  const float m_new = nan_max(s.m, tmax);
  const float delta = fmaxf((s.m - m_new) * c, D_MIN), a = exp2_(delta);
  const float mref = finite_or_0(m_new);
  s.s1 = a * (s.s1 + delta * s.s0);
  s.s0 = a * s.s0;
  s.m = m_new;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!INSIDE && u >= nu) break;
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

// one wave's share of a row: wave `w` of the `G` of a group, vectors [vb, ve) of the row.  s_max (64, zero):
// the group's lane maxima.
template <int DT, int G, bool TOP, bool ENT>
__device__ __forceinline__ Stat stream_row(const char *xr, int V, int vb, int ve, int w, float c, Best &best,
                                           u32 *s_max) {
  constexpr int VEC = Elem<DT>::VEC;
  const int shift = (int)(((uintptr_t)xr / Elem<DT>::ES) & (VEC - 1));   // vector i = elements i VEC - shift ..
  const int full = (int)(((long long)V + shift) / VEC);                    // whole vectors end here
  const int last = min(ve, full), begin = vb + w * 64 * U;
  Stat s = {-INFINITY, 0.0f, 0.0f};
  int t0 = begin;
  if (!(TOP && G > 1) && t0 >= ve) return s;                               // (else every wave gives its maxima)
  do {
    if ((t0 > 0 || shift == 0) && t0 + 64 * U <= last)
      stream_tile<DT, G, TOP, ENT, true>(xr, V, shift, t0, ve, c, t0 == begin, s, best, s_max);
    else
      stream_tile<DT, G, TOP, ENT, false>(xr, V, shift, t0, ve, c, t0 == begin, s, best, s_max);
    t0 += G * 64 * U;
  } while (t0 < ve);
  return wave_combine(s, c);
}

// ---- what is written for a row ---------------------------------------------------------------------------
// stats: {mref, s0, entropy, log2 s0} of scores, {mref, s0, max w, 1 / sum 2^((w - max w) c)} of distillation;
// s0 = 0 marks a row without gradient (else it is at least 1, for the largest logit), NaN one whose gradient is
// NaN.  Backward, p is formed as 2^d (1 / s0): d - log2 s0 would be rounded at its size, 10 to 25, and leave up to
// 11 roundings in p where this leaves one.
__device__ __forceinline__ float log2_sum(const Stat &s) {
  return s.s0 == 0.0f ? INFINITY : log2f(s.s0);        // (0: every logit is -inf)
}

// G waves of a workgroup share a row's stretch: waves per workgroup, groups per workgroup
template <int G> struct Shape {
  static constexpr int WAVES = G == 1 ? 4 : G, THREADS = 64 * WAVES, GROUPS = WAVES / G;
};

// the partial results of a row that several workgroups read
struct Split {
  int n;               // stretches per row, a power of two; 1: none
  Stat *part;          // (rows, n)
  u64 *keys;           // (rows, n, k)
};

// Statistics (and, TOP, the k best) of stretch `seg` of `segs` of a row, by the G waves of a group.
// Wave 0 of the group gets the result; its k best are in `lists[G > 1 ? G : 0]`, 0 after the last one.
// Every wave of the workgroup comes here together where G > 1.
template <int DT, int G, bool TOP, bool ENT>
__device__ __forceinline__ Stat group_stat(const char *xr, int V, int seg, int segs, int k, float c,
                                           u64 (*lists)[BUF], Stat *s_part, Shared *sh) {
  typedef Elem<DT> E;
  const int lane = lane_id(), w = G == 1 ? 0 : wave_id();
  const int shift = (int)(((uintptr_t)xr / E::ES) & (E::VEC - 1));
  const int nvec = (int)(((long long)V + shift + E::VEC - 1) / E::VEC);
  const int per = (nvec + segs - 1) / segs;
  const int vb = min(nvec, seg * per), ve = min(nvec, vb + per);
  Best best;
  if (TOP) best.init(lists[w], k);
  // (nobody counts before the barrier inside stream_row, nobody reads the last count after the one before this)
  if (TOP && G > 1 && w == 0 && lane == 0) sh->n = 0;
  Stat s = stream_row<DT, G, TOP, ENT>(xr, V, vb, ve, w, c, best, TOP && G > 1 ? sh->max : nullptr);
  if (G == 1) {
    if (TOP) best.cut(lane);
    return s;
  }
  if (TOP) {
    int at = 0;
    if (lane == 0) at = atomicAdd(&sh->n, best.cnt);
    at = __builtin_amdgcn_readfirstlane(at);
    if (at + best.cnt <= BUF)
      for (int i = lane; i < best.cnt; i += 64) lists[G][at + i] = lists[w][i];
  }
  if (lane == 0) s_part[w] = s;
  __syncthreads();
  const int n = TOP ? sh->n : 0;
  if (n > BUF) {                             // too many for one buffer: every wave's k best, sorted
    best.cut(lane);
    for (int j = best.cnt + lane; j < k; j += 64) lists[w][j] = 0;
    __syncthreads();
  }
  if (w == 0) {
    Stat o = {-INFINITY, 0.0f, 0.0f};
    if (lane < G) o = s_part[lane];
    s = wave_combine(o, c);
    if (TOP) {
      sh->max[lane] = 0;                     // (read by all, needed again after the workgroup's next barrier)
      Best all;
      all.init(lists[G], k);
      if (n > BUF) {
        merge_lists(all, G, lane, [&](int list, int pos) { return lists[list][pos]; });
      } else {
        all.cnt = n;
        all.cut(lane);
      }
      for (int j = all.cnt + lane; j < k; j += 64) lists[G][j] = 0;
      wave_lds_fence();
    }
  }
  return s;
}

// a wave joins the stretches of a row; the k best go to `list`
__device__ __forceinline__ Stat join_stretches(const Split &sp, int r, int k, float c, u64 *list, int lane) {
  Stat o = {-INFINITY, 0.0f, 0.0f};
  if (lane < sp.n) o = sp.part[(size_t)r * sp.n + lane];
  o = wave_combine(o, c);
  if (k) {
    Best all;
    all.init(list, k);
    const u64 *keys = sp.keys + (size_t)r * sp.n * k;
    merge_lists(all, sp.n, lane, [&](int l, int pos) { return keys[(size_t)l * k + pos]; });
  }
  return o;
}

__device__ __forceinline__ void write_part(const Split &sp, size_t unit, const Stat &s, const u64 *list, int k,
                                           int lane) {
  if (lane == 0) sp.part[unit] = s;
  if (lane < k) sp.keys[unit * k + lane] = list[lane];
}

__device__ __forceinline__ bool scores_dead(const s2c_token_scores_args &a, int r) {
  return a.has_ignore && a.token && a.token[r] == a.ignore;
}

__device__ __forceinline__ void scores_write_dead(const s2c_token_scores_args &a, int r, int lane) {
  if (lane == 0) {
    if (a.logp) a.logp[r] = 0.0f;
    a.entropy[r] = 0.0f;
    if (a.stats) *reinterpret_cast<float4 *>(a.stats + 4 * (size_t)r) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
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
    if (a.stats) *reinterpret_cast<float4 *>(a.stats + 4 * (size_t)r) =
        make_float4(mref, bad ? NAN : s.s0, h < 0.0f ? 0.0f : h, l2s);
  }
  if (lane < a.k) {
    const u64 key = top[lane];
    a.top_logp[(size_t)r * a.k + lane] = (unord((u32)(key >> 32)) - mref) * a.lg.inv_t - LN2 * sub;
    a.top_ids[(size_t)r * a.k + lane] = (long long)(u32)~(u32)key;
  }
}

template <int DT, int G, bool TOP>
__global__ __launch_bounds__(Shape<G>::THREADS) void scores_fwd_kernel(s2c_token_scores_args a, Split sp) {
  typedef Shape<G> Sh;
  __shared__ u64 s_lists[TOP ? Sh::WAVES + (G > 1) : 1][TOP ? BUF : 1];
  __shared__ Stat s_part[Sh::WAVES];
  __shared__ Shared s_shared;
  const int lane = lane_id(), w = wave_id();
  const int grp = G == 1 ? w : 0;
  const bool first = G == 1 || w == 0;
  if (TOP && G > 1) {
    if (w == 0) s_shared.max[lane] = 0;
    __syncthreads();
  }
  u64 (*lists)[BUF] = reinterpret_cast<u64 (*)[BUF]>(&s_lists[TOP ? grp : 0][0]);
  const float c = a.lg.inv_t * LOG2E;
  const long long units = (long long)a.lg.rows * sp.n;
  for (long long un = (long long)blockIdx.x * Sh::GROUPS + grp; un < units; un += (long long)gridDim.x * Sh::GROUPS) {
    int r, seg;
    row_and_stretch(un, sp.n, r, seg);
    if (scores_dead(a, r)) {
      if (first && sp.n == 1) scores_write_dead(a, r, lane);
      continue;
    }
    const char *xr = row_ptr(a.lg, Elem<DT>::ES, r);
    const Stat s = group_stat<DT, G, TOP, true>(xr, a.lg.V, seg, sp.n, a.k, c, lists, s_part, &s_shared);
    if (first) {
      const u64 *list = lists[G > 1 ? G : 0];
      if (sp.n == 1) scores_write<DT>(a, r, xr, s, list, lane);
      else write_part(sp, (size_t)un, s, list, a.k, lane);
    }
    if (G > 1) __syncthreads();
  }
}

template <int DT>
__global__ __launch_bounds__(256) void scores_join_kernel(s2c_token_scores_args a, Split sp) {
  __shared__ u64 s_list[4][BUF];
  const int lane = lane_id(), w = wave_id();
  const float c = a.lg.inv_t * LOG2E;
  for (long long r = (long long)blockIdx.x * 4 + w; r < a.lg.rows; r += (long long)gridDim.x * 4) {
    if (scores_dead(a, (int)r)) {
      scores_write_dead(a, (int)r, lane);
      continue;
    }
    const Stat s = join_stretches(sp, (int)r, a.k, c, s_list[w], lane);
    scores_write<DT>(a, (int)r, row_ptr(a.lg, Elem<DT>::ES, (int)r), s, s_list[w], lane);
  }
}

// ---- distillation --------------------------------------------------------------------------------------
// the teacher's softmax over a row's slots, slot j of lane l = l + 64 i: log q and q; id -1: an empty slot
struct Slots {
  long long id[SLOTS / 64];
  float lq[SLOTS / 64], q[SLOTS / 64];
  float wm, l2w, inv;     // log2 of the sum and its inverse; l2w = +inf: no slot is used
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
      if (w[i] == -INFINITY) s.id[i] = -1;
    }
    m = nan_max(m, w[i]);
  }
  s.wm = finite_or_0(wave_max(m));
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < SLOTS / 64; ++i) sum += exp2_((w[i] - s.wm) * c);
  sum = wave_sum(sum);
  s.l2w = sum == 0.0f ? INFINITY : log2f(sum);
  s.inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int i = 0; i < SLOTS / 64; ++i) {
    s.lq[i] = (w[i] - s.wm) * a.lg.inv_t - LN2 * s.l2w;
    s.q[i] = exp2_((w[i] - s.wm) * c) * s.inv;
  }
  return s;
}

__device__ __forceinline__ void distill_write_dead(const s2c_distill_args &a, int r, int lane) {
  if (lane == 0) {
    a.loss[r] = 0.0f;
    if (a.stats) *reinterpret_cast<float4 *>(a.stats + 4 * (size_t)r) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
}

// the student's logits at a lane's slots (asked for before the row is read)
template <int DT>
__device__ __forceinline__ void gather_slots(float (&at)[SLOTS / 64], const char *xr, int V, const Slots &t) {
#pragma unroll
  for (int i = 0; i < SLOTS / 64; ++i)
    at[i] = t.id[i] >= 0 && t.id[i] < V ? Elem<DT>::load(xr, t.id[i]) : 0.0f;
}

__device__ __forceinline__ void distill_write(const s2c_distill_args &a, int r, const float (&at)[SLOTS / 64],
                                              const Stat &s, const Slots &t, int lane) {
  const float mref = finite_or_0(s.m);
  const float l2s = log2_sum(s);
  const float sub = l2s == INFINITY ? 0.0f : l2s;
  float part = 0.0f;
  bool bad = t.l2w != t.l2w;                    // (a teacher's NaN or +inf)
#pragma unroll
  for (int i = 0; i < SLOTS / 64; ++i) {
    if (t.id[i] >= a.lg.V) bad = true;
    else if (t.q[i] != 0.0f)                    // (empty slots and vanishing ones add nothing)
      part += t.q[i] * (t.lq[i] - ((at[i] - mref) * a.lg.inv_t - LN2 * sub));
  }
  part = wave_sum(part);
  bad = __ballot(bad) != 0;
  if (lane == 0) {
    a.loss[r] = bad ? NAN : part;
    if (a.stats) *reinterpret_cast<float4 *>(a.stats + 4 * (size_t)r) =
        make_float4(mref, bad ? NAN : s.s0, t.wm, t.inv);
  }
}

template <int DT, int G>
__global__ __launch_bounds__(Shape<G>::THREADS) void distill_fwd_kernel(s2c_distill_args a, Split sp) {
  typedef Shape<G> Sh;
  __shared__ Stat s_part[Sh::WAVES];
  const int lane = lane_id(), w = wave_id();
  const int grp = G == 1 ? w : 0;
  const bool first = G == 1 || w == 0;
  const float c = a.lg.inv_t * LOG2E;
  const long long units = (long long)a.lg.rows * sp.n;
  for (long long un = (long long)blockIdx.x * Sh::GROUPS + grp; un < units; un += (long long)gridDim.x * Sh::GROUPS) {
    int r, seg;
    row_and_stretch(un, sp.n, r, seg);
    bool dead = a.mask && a.mask[r] == 0;
    const char *xr = row_ptr(a.lg, Elem<DT>::ES, r);
    Slots t;
    float at[SLOTS / 64];
    if (!dead && sp.n == 1) {
      t = load_slots(a, r, c, lane);
      dead = t.l2w == INFINITY;
      if (!dead) gather_slots<DT>(at, xr, a.lg.V, t);
    }
    if (dead) {
      if (first && sp.n == 1) distill_write_dead(a, r, lane);
      continue;
    }
    const Stat s = group_stat<DT, G, false, false>(xr, a.lg.V, seg, sp.n, 0, c, nullptr, s_part, nullptr);
    if (first) {
      if (sp.n == 1) distill_write(a, r, at, s, t, lane);
      else write_part(sp, (size_t)un, s, nullptr, 0, lane);
    }
    if (G > 1) __syncthreads();
  }
}

template <int DT>
__global__ __launch_bounds__(256) void distill_join_kernel(s2c_distill_args a, Split sp) {
  const int lane = lane_id(), w = wave_id();
  const float c = a.lg.inv_t * LOG2E;
  for (long long r = (long long)blockIdx.x * 4 + w; r < a.lg.rows; r += (long long)gridDim.x * 4) {
    bool dead = a.mask && a.mask[r] == 0;
    Slots t;
    if (!dead) {
      t = load_slots(a, (int)r, c, lane);
      dead = t.l2w == INFINITY;
    }
    if (dead) {
      distill_write_dead(a, (int)r, lane);
      continue;
    }
    float at[SLOTS / 64];
    gather_slots<DT>(at, row_ptr(a.lg, Elem<DT>::ES, (int)r), a.lg.V, t);
    distill_write(a, (int)r, at, join_stretches(sp, (int)r, 0, c, nullptr, lane), t, lane);
  }
}

// ---- gradients -------------------------------------------------------------------------------------------
// dx_v = 2^d_v (A + B max(d_v, D_MIN)) + the sparse entries of v, with i = inv_t / s0:
//   scores  A = -(g + sum g_top + g_H (H - ln 2 log2 s0)) i, B = -g_H ln 2 i, entries g inv_t at the token and
//           g_top_j inv_t at top_ids_j
//   distill A = g i, B = 0, entries -g q_j inv_t at id_j
// A group of G waves loads its stretch of the row (U vectors a lane).  While the loads are under way its
// first wave gathers the entries that lie in the stretch, in slot order, with their logits.  Then the dense
// part is written, and the first entry of every word writes its element once more with all entries of
// that word added in slot order (rounded once; no atomics).
struct GradArgs {
  s2c_logits lg;
  const float *stats;
  void *dx;
  int segs, span;        // stretches per row, of `span` vectors (64 G U at most)
  int past_cache;        // dx does not fit the cache: stored past it
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

template <int G>
__device__ __forceinline__ void group_sync() {
  if (G == 1) wave_lds_fence(); else __syncthreads();
}

template <int DT, int G, bool DISTILL>
__global__ __launch_bounds__(256) void vocab_bwd_kernel(GradArgs a) {
  typedef Elem<DT> E;
  constexpr int VEC = E::VEC, GROUPS = 4 / G, LANES = 64 * G;
  static_assert(SLOTS >= KMAX + 1, "entries of a row");
  struct Entries {
    int id[SLOTS];
    float val[SLOTS], x[SLOTS];
    int n;
    float sum;               // of all the row's entries (scores)
  };
  __shared__ Entries s_entries[GROUPS];
  const int lane = lane_id();
  const int grp = G == 1 ? wave_id() : 0, tid = G == 1 ? lane : (int)threadIdx.x;
  Entries &en = s_entries[grp];
  const float c = a.lg.inv_t * LOG2E, it = a.lg.inv_t;
  const int V = a.lg.V;
  const long long units = (long long)a.lg.rows * a.segs;
  for (long long un = (long long)blockIdx.x * GROUPS + grp; un < units; un += (long long)gridDim.x * GROUPS) {
    int r, seg;
    row_and_stretch(un, a.segs, r, seg);
    const char *xr = row_ptr(a.lg, E::ES, r);
    const long long o0 = (long long)r * V;
    const int shift = (int)((((uintptr_t)a.dx / E::ES) + o0) & (VEC - 1));       // of the stores
    const float4 st = *reinterpret_cast<const float4 *>(a.stats + 4 * (size_t)r);
    const float mref = st.x, inv = 1.0f / st.y;
    const bool dead = st.y == 0.0f;
    const long long b0 = (long long)seg * a.span * VEC - shift;                  // the stretch's elements
    const long long b1 = min((long long)V, b0 + (long long)a.span * VEC);
    Raw x[U];
    if (!dead) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long e0 = b0 + (long long)(u * LANES + tid) * VEC;
        if (e0 >= 0 && e0 + VEC <= b1) {
          x[u] = load16<DT>(xr, e0);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[u].w[i] = 0;
          if (e0 > -VEC && e0 < b1) {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
              if (e0 + e >= 0 && e0 + e < b1) E::put(x[u], e, E::bits(xr, e0 + e));
          }
        }
      }
    }
    float A = 0.0f, B = 0.0f;
    if (!dead) {
      int n;                                         // entries of the row
      float g;
      if (DISTILL) {
        n = a.K;
        g = a.g_loss[r] * it;
        A = g * inv;
      } else {
        const float ge = a.g_entropy ? a.g_entropy[r] : 0.0f;
        g = (a.g_logp && a.token) ? a.g_logp[r] * it : 0.0f;
        n = 1 + (a.g_top ? a.k : 0);
        A = -ge * (st.z - LN2 * st.w) * it;
        B = -ge * LN2 * it * inv;
      }
      if (tid < 64) {
        float sum = 0.0f;
        int found = 0;
        for (int j0 = 0; j0 < n; j0 += 64) {
          const int j = j0 + lane;
          long long id = -1;
          float val = 0.0f;
          if (j < n) {
            if (DISTILL) {
              id = a.ids[(size_t)r * n + j];
              if (id >= 0)
                val = -g * (exp2_((load_any(a.teacher, (long long)r * n + j, a.teacher_dtype) - st.z) * c) * st.w);
            } else if (j == 0) {
              id = a.token ? a.token[r] : -1;
              val = g;
            } else {
              id = a.top_ids[(size_t)r * (n - 1) + j - 1];
              val = a.g_top[(size_t)r * (n - 1) + j - 1] * it;
            }
          }
          sum += val;
          const bool here = id >= 0 && id >= b0 && id < b1;
          const u64 mask = __ballot(here);
          if (here) {
            const int to = found + mask_rank_below(mask);
            en.id[to] = (int)id;
            en.val[to] = val;
            en.x[to] = E::load(xr, id);
          }
          found += __popcll(mask);
        }
        if (!DISTILL) sum = wave_sum(sum);
        if (lane == 0) {
          en.n = found;
          en.sum = sum;
        }
      }
    }
    group_sync<G>();
    if (!DISTILL && !dead) A = (A - en.sum) * inv;
    auto grad = [&](float v) {
      const float d = (v - mref) * c;
      return exp2_(d) * (DISTILL ? A : __builtin_fmaf(B, fmaxf(d, D_MIN), A));
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long e0 = b0 + (long long)(u * LANES + tid) * VEC;
      float f[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = dead ? 0.0f : grad(E::at(x[u], e));
      if (e0 >= 0 && e0 + VEC <= b1) {
        if (a.past_cache) store16_past_cache(a.dx, (o0 + e0) * E::ES, E::pack(f));
        else store16<DT>(a.dx, o0 + e0, E::pack(f));
      } else if (e0 > -VEC && e0 < b1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (e0 + e >= 0 && e0 + e < b1) E::store(a.dx, o0 + e0 + e, f[e]);
      }
    }
    group_sync<G>();
    if (!dead && tid < 64) {
      const int n = en.n;
      for (int j = lane; j < n; j += 64) {
        const int id = en.id[j];
        float sum = 0.0f;
        bool first = true;
        for (int i = 0; i < n; ++i)
          if (en.id[i] == id) {
            sum += en.val[i];
            first = first && i >= j;
          }
        if (first) E::store(a.dx, o0 + id, grad(en.x[j]) + sum);
      }
    }
    group_sync<G>();
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

constexpr int MAX_GRID = 1 << 21;       // workgroups of up to 1024: below 2^32 work-items

int grid_of(long long units) { return (int)(units < MAX_GRID ? units : MAX_GRID); }

// fn<element type>(), by the run-time code
template <class F>
void by_type(int dtype, F f) {
  if (dtype == S2C_F32) f(std::integral_constant<int, S2C_F32>());
  else if (dtype == S2C_BF16) f(std::integral_constant<int, S2C_BF16>());
  else f(std::integral_constant<int, S2C_F16>());
}

long long vectors(int V, int dtype) {                  // of a row, at any alignment
  const int vec = dtype == S2C_F32 ? 4 : 8;
  return ((long long)V + 2 * vec - 2) / vec;
}

// How a row is shared out: `waves` of a workgroup to a stretch, `split` stretches to a row.
//  * many rows: a wave each -- no barrier, no merge, one threshold for the whole row (59392 rows of 3500
//    fp32 words, 5 alternatives: 151 us, 303 with 4 waves a row);
//  * rows that would leave most of the chip empty: 16 waves (32768 bf16 words, one row: 7.4 us, 8.6 with 4,
//    19.9 with 1), and stretches of at least one round of tiles, up to 256 workgroups, joined by a second
//    launch (64 rows of 131072 words, 20 alternatives: 14.9 us in 4 stretches, 17.2 in one; one row of 262144
//    fp32 words: 13 in 16, 25.5 in one);
//  * 4 waves between (512 rows of 32000 words: 13.4 us with 8 alternatives, 31.5 with 1, 17.7 with 16; without
//    alternatives 9.8, 18.0 and 12.2; the floor is 6.4) and for short rows (248 rows of 3500: 3.9 us, the same
//    with 16).
struct Plan { int waves, split; };

Plan forward_plan(int rows, int V, int dtype) {
  const long long nvec = vectors(V, dtype);
  Plan p = {4, 1};
  if (rows >= 2048) {
    p.waves = 1;
  } else if (rows < 256 && nvec > 1024) {
    p.waves = 16;
    while (p.split < MAX_SPLIT && 2LL * p.split * rows <= 256 && 2LL * p.split * (16 * 64 * 4) <= nvec) p.split *= 2;
  }
  return p;
}

template <class F>
void by_plan(const Plan &p, F f) {
  if (p.waves == 16) f(std::integral_constant<int, 16>());
  else if (p.waves == 4) f(std::integral_constant<int, 4>());
  else f(std::integral_constant<int, 1>());
}

long long split_bytes(int rows, int split, int k) {
  return split == 1 ? 0 : (long long)rows * split * (sizeof(Stat) + 8LL * k) + 8;
}

Split split_of(const Plan &p, int rows, int k, void *ws) {
  Split sp = {p.split, nullptr, nullptr};
  sp.keys = (u64 *)ws;
  sp.part = (Stat *)((char *)ws + 8LL * rows * p.split * k);
  return sp;
}

template <bool DISTILL>
int backward(GradArgs &a, const char *what, hipStream_t st) {
  const long long nvec = vectors(a.lg.V, a.lg.dtype);
  // waves of their own for short rows, whose stretches would leave most of a workgroup idle (59392 x 3500 bf16,
  // 439 vectors: 156 us, 252 with 4 waves; 8192 x 8000, 1001 vectors: 47 and 44 us), and further where a
  // stretch waits for its slots (the same with 32 slots: 51 and 55 us; 1000 x 10007, 33 slots: 13.0 and 16.7;
  // 4096 x 65536, 64 slots: 198 and 184)
  const int G = nvec <= (DISTILL ? 2048 : 512) ? 1 : 4;
  a.segs = (int)((nvec + 64 * G * U - 1) / (64 * G * U));
  a.span = (int)((nvec + a.segs - 1) / a.segs);
  // a gradient that the 256 MB cache cannot hold would leave it full of lines to be written back: the
  // next forward pass over 4096 x 50001 bf16 takes 118 us behind ordinary stores, 82 to 90 us behind these
  a.past_cache = (double)a.lg.rows * a.lg.V * (a.lg.dtype == S2C_F32 ? 4 : 2) >= 256.0 * (1 << 20);
  const long long units = (long long)a.lg.rows * a.segs;
  by_type(a.lg.dtype, [&](auto dt) {
    if (G == 1) hipLaunchKernelGGL((vocab_bwd_kernel<dt.value, 1, DISTILL>), dim3(grid_of((units + 3) / 4)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((vocab_bwd_kernel<dt.value, 4, DISTILL>), dim3(grid_of(units)), dim3(256), 0, st, a);
  });
  return launched(what);
}

// the gradient, and the statistics that are read 16 bytes at a time
bool bad_backward(const s2c_logits &l, const float *stats, const void *dx) {
  return !stats || ((uintptr_t)stats & 15) || !dx || ((uintptr_t)dx & (l.dtype == S2C_F32 ? 3 : 1));
}

bool bad_workspace(const void *ws) { return !ws || ((uintptr_t)ws & 7); }

bool bad_scores(const s2c_token_scores_args *a) {
  return !a || bad_logits(a->lg) || a->k < 0 || a->k > KMAX || a->k > a->lg.V || (a->k && !a->top_ids);
}

bool bad_distill(const s2c_distill_args *a) {
  return !a || bad_logits(a->lg) || a->K <= 0 || a->K > SLOTS || a->teacher_dtype < 0 ||
         a->teacher_dtype > 2 || !a->ids || !a->teacher;
}

}  // namespace

extern "C" long long s2c_words_args_sizeof(int which) {
  return which == 0 ? sizeof(s2c_logits) : which == 1 ? sizeof(s2c_token_scores_args)
         : which == 2 ? sizeof(s2c_distill_args) : 0;
}

extern "C" long long s2c_token_scores_workspace_bytes(int rows, int V, int dtype, int k) {
  return split_bytes(rows, forward_plan(rows, V, dtype).split, k);
}

extern "C" int s2c_token_scores_fwd(const s2c_token_scores_args *a, void *stream) {
  if (bad_scores(a) || !a->entropy || (a->token && !a->logp) || (a->k && !a->top_logp) ||
      ((uintptr_t)a->stats & 15))
    return S2C_EINVAL;
  const int rows = a->lg.rows;
  if (rows == 0) return 0;
  const Plan p = forward_plan(rows, a->lg.V, a->lg.dtype);
  if (p.split > 1 && bad_workspace(a->ws)) return S2C_EINVAL;
  const Split sp = split_of(p, rows, a->k, a->ws);
  const long long units = (long long)rows * p.split;
  hipStream_t st = (hipStream_t)stream;
  by_type(a->lg.dtype, [&](auto dt) {
    auto go = [&](auto g) {
      typedef Shape<g.value> Sh;
      const dim3 grid(grid_of((units + Sh::GROUPS - 1) / Sh::GROUPS)), block(Sh::THREADS);
      if (a->k) hipLaunchKernelGGL((scores_fwd_kernel<dt.value, g.value, true>), grid, block, 0, st, *a, sp);
      else hipLaunchKernelGGL((scores_fwd_kernel<dt.value, g.value, false>), grid, block, 0, st, *a, sp);
    };
    by_plan(p, go);
    if (p.split > 1)
      hipLaunchKernelGGL((scores_join_kernel<dt.value>), dim3(grid_of((rows + 3LL) / 4)), dim3(256), 0, st, *a, sp);
  });
  return launched("token_scores_fwd");
}

extern "C" int s2c_token_scores_bwd(const s2c_token_scores_args *a, const float *g_logp,
                                    const float *g_entropy, const float *g_top, void *dx, void *stream) {
  if (bad_scores(a) || bad_backward(a->lg, a->stats, dx)) return S2C_EINVAL;
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

extern "C" long long s2c_distill_workspace_bytes(int rows, int V, int dtype) {
  return split_bytes(rows, forward_plan(rows, V, dtype).split, 0);
}

extern "C" int s2c_distill_fwd(const s2c_distill_args *a, void *stream) {
  if (bad_distill(a) || !a->loss || ((uintptr_t)a->stats & 15)) return S2C_EINVAL;
  const int rows = a->lg.rows;
  if (rows == 0) return 0;
  const Plan p = forward_plan(rows, a->lg.V, a->lg.dtype);
  if (p.split > 1 && bad_workspace(a->ws)) return S2C_EINVAL;
  const Split sp = split_of(p, rows, 0, a->ws);
  const long long units = (long long)rows * p.split;
  hipStream_t st = (hipStream_t)stream;
  by_type(a->lg.dtype, [&](auto dt) {
    auto go = [&](auto g) {
      typedef Shape<g.value> Sh;
      hipLaunchKernelGGL((distill_fwd_kernel<dt.value, g.value>),
                         dim3(grid_of((units + Sh::GROUPS - 1) / Sh::GROUPS)), dim3(Sh::THREADS), 0, st, *a, sp);
    };
    by_plan(p, go);
    if (p.split > 1)
      hipLaunchKernelGGL((distill_join_kernel<dt.value>), dim3(grid_of((rows + 3LL) / 4)), dim3(256), 0, st, *a, sp);
  });
  return launched("distill_fwd");
}

extern "C" int s2c_distill_bwd(const s2c_distill_args *a, const float *g_loss, void *dx, void *stream) {
  if (bad_distill(a) || !g_loss || bad_backward(a->lg, a->stats, dx)) return S2C_EINVAL;
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
