// Log probability, rank, entropy and likeliest alternatives of tokens, from logits.
//
// For a row x of V logits, m = max x and r = sum over all but one largest element of exp(x_j - m):
//     log p_t = (x_t - m) - log1p(r)      entropy = log1p(r) - sum (x_j - m) exp(x_j - m) / (1 + r)
// (log1p keeps the digits of a token that is nearly certain: log p = -r there.)  The rank of t is 1 + the number of logits
// above x_t, equal ones with a lower index counted; alternatives come in that order too.  The sums are in 32 bits, over
// terms relative to a share's own maximum; shares are put together as
//     r = r* + sum_c w_c (1 + r_c),   E = E* + sum_c w_c (E_c + d_c (1 + r_c)),   d_c = m_c - m, w_c = exp(d_c)
// where * is the share that holds the row's maximum.
//
// Bound by memory: a row is read once, by 1 to 8 CTAs of a cluster, 16 bytes a lane and four such loads on their way.  Each
// warp carries its maximum and each lane its sums relative to it; a new maximum of a batch of four vectors a lane rescales
// them.  Elements that equal the maximum are counted, all others go into the sums.  CTAs write their results into the first
// one's shared memory, where they are put together: no scratch in global memory, no atomics whose order shows.
// The best tokens of a share: the top-th best of its threads' maxima bounds them from below, so no more threads than that
// (and a few) hold any; those threads' vectors are read again, from the L2 cache, and a candidate's rank is the number of
// its betters.  Where that leaves more candidates than there is room for, the best are taken one by one.
// 4662 x 50257 bf16 take 116 us, 4.0 TB/s, at 13 instructions a logit: issue slots bound it, three quarters of them taken.  Two
// floats an instruction, counting in pairs of 16 bits and vectors without edges brought it there from 362 us with a row's
// logits held in registers and every pass over them.
#include "common.cuh"
#include <type_traits>

namespace ronn {

constexpr int TL_TOP = 32;
constexpr int TL_CLUSTER = 8;
constexpr int TL_SLACK = 8;            // threads beyond `top` that may offer candidates
constexpr int TL_CAND = 1024;
constexpr float TL_LOG2E = 1.4426950408889634f;
constexpr int TL_BATCH = 4;            // vectors a lane has on their way
// A term's exponent is x log2 e - m log2 e in one operation, and what rounding m log2 e leaves over (m_lo) is made good once a
// row.  That is half a unit at most up to this magnitude; further out it would pass the range of an exponent.  A warp whose
// maximum lies there (nothing but masks of -1e9 so far, a token forced by 1e10) takes x - m first, element by element.
constexpr float TL_FAR = 8388608.f;

struct TlArgs {
  const void* logits;
  const void* tokens;
  float *logprob, *entropy, *top_logprobs;
  int *rank, *top_ids;
  long ld, token_stride, rows;
  int vocab, top, cluster, wide_tokens;
};

// Total order of the logits: larger first, then the lower index; NaN above everything, -0 equal to 0.
__device__ __forceinline__ uint32_t tl_key(float x) {
  const uint32_t b = __float_as_uint(x), mag = b & 0x7fffffffu;          // on the bits: float comparisons here take subnormals for 0
  if (mag > 0x7f800000u) return 0xffffffffu;
  return mag == 0 || !(b >> 31) ? mag | 0x80000000u : ~b;
}
__device__ __forceinline__ float tl_value(uint32_t key) {
  return __uint_as_float(key == 0xffffffffu ? 0x7fffffffu : key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// (key, index) as one number: larger is better.  0 is below every logit.
__device__ __forceinline__ unsigned long long tl_pair(uint32_t key, int idx) {
  return (static_cast<unsigned long long>(key) << 32) | uint32_t(~idx);
}
__device__ __forceinline__ float tl_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float tl_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float tl_exp(float d) { return tl_exp2(d * TL_LOG2E); }

template <class T> __device__ __forceinline__ uint32_t tl_max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <class T> __device__ __forceinline__ uint32_t tl_max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Two floats in one instruction.
__device__ __forceinline__ unsigned long long tl_two(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 tl_split(unsigned long long v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ unsigned long long tl_add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long tl_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// A 16-byte vector of logits as E = 4 or 8 floats.
template <class T> struct TlVec {
  static constexpr int E = 8;
  static __device__ __forceinline__ float largest(const uint4& v) {       // NaN if any is
    float lo, hi;
    Pair16<T>::unpack(tl_max2_nan<T>(tl_max2_nan<T>(v.x, v.y), tl_max2_nan<T>(v.z, v.w)), lo, hi);
    return tl_max_nan(lo, hi);
  }
  // With a maximum above LOW, -inf and the type's lowest value weigh the same: nothing.
  static constexpr float LOW = std::is_same<T, __half>::value ? -6e4f : -1e30f;
  static constexpr float FROM = std::is_same<T, __half>::value ? -6e4f : -TL_FAR;        // maxima from here to TL_FAR: the fast way
  static __device__ __forceinline__ uint4 finite(uint4 v) {
    const uint32_t low = std::is_same<T, __half>::value ? 0xfbfffbffu : 0xfe96fe96u;        // bf16: -1e38, whose product with log2 e is finite
    return make_uint4(tl_max2<T>(v.x, low), tl_max2<T>(v.y, low), tl_max2<T>(v.z, low), tl_max2<T>(v.w, low));
  }
  // How many of the eight pass x > t, or x >= t: two counters in a pair of the type, exact to 256 and more.
  using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  static constexpr uint32_t NONE = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;        // two of -inf
  struct Count {
    Pair t, n;
    __device__ __forceinline__ explicit Count(float th) {
      const uint32_t w = Pair16<T>::pack(th, th), z = 0u;
      t = *reinterpret_cast<const Pair*>(&w), n = *reinterpret_cast<const Pair*>(&z);
    }
    __device__ __forceinline__ void add(const uint4& v, bool or_equal) {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Pair x = *reinterpret_cast<const Pair*>(&w[i]);
        n = __hadd2(n, or_equal ? __hge2(x, t) : __hgt2(x, t));
      }
    }
    __device__ __forceinline__ int sum() const {
      float lo, hi;
      Pair16<T>::unpack(*reinterpret_cast<const uint32_t*>(&n), lo, hi);
      return int(lo + hi);
    }
  };
  static __device__ __forceinline__ uint32_t word(float x) { return Pair16<T>::pack(x, x); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    Pair16<T>::unpack(v.x, f[0], f[1]);
    Pair16<T>::unpack(v.y, f[2], f[3]);
    Pair16<T>::unpack(v.z, f[4], f[5]);
    Pair16<T>::unpack(v.w, f[6], f[7]);
  }
};
template <> struct TlVec<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ float largest(const uint4& v) {
    return tl_max_nan(tl_max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), tl_max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static constexpr float LOW = -1e30f, FROM = -TL_FAR;
  static __device__ __forceinline__ uint4 finite(uint4 v) {
    return make_uint4(__float_as_uint(fmaxf(__uint_as_float(v.x), -1e32f)), __float_as_uint(fmaxf(__uint_as_float(v.y), -1e32f)),
                      __float_as_uint(fmaxf(__uint_as_float(v.z), -1e32f)), __float_as_uint(fmaxf(__uint_as_float(v.w), -1e32f)));
  }
  static constexpr uint32_t NONE = 0xff800000u;
  struct Count {
    float t;
    int n = 0;
    __device__ __forceinline__ explicit Count(float th) : t(th) {}
    __device__ __forceinline__ void add(const uint4& v, bool or_equal) {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) n += (or_equal ? __uint_as_float(w[i]) >= t : __uint_as_float(w[i]) > t) ? 1 : 0;
    }
    __device__ __forceinline__ int sum() const { return n; }
  };
  static __device__ __forceinline__ uint32_t word(float x) { return __float_as_uint(x); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
};

struct TlShare {
  float m, r, e;
  int ahead;
};

__device__ __forceinline__ uint32_t tl_remote(const void* p, int cta) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(uint32_t(__cvta_generic_to_shared(p))), "r"(cta));
  return a;
}
__device__ __forceinline__ void tl_store(uint32_t a, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void tl_store(uint32_t a, unsigned long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }
__device__ __forceinline__ void tl_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void tl_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Shares of a row put together, in order.  One without a probability weighs nothing.
__device__ __forceinline__ TlShare tl_join(const TlShare* s, int n) {
  int best = 0;
  for (int c = 1; c < n; ++c)
    if (tl_key(s[c].m) > tl_key(s[best].m)) best = c;
  TlShare all = s[best];
  for (int c = 0; c < n; ++c) {
    if (c == best) continue;
    all.ahead += s[c].ahead;
    const float d = s[c].m - all.m, w = tl_exp(d);
    if (w != 0.f && s[c].m != -INFINITY) all.r += w * (1.f + s[c].r), all.e += w * (s[c].e + d * (1.f + s[c].r));
  }
  return all;
}

// Places a list of `top` best pairs holds above v: the list is sorted, best first, and ends in zeros.
__device__ __forceinline__ int tl_above(const unsigned long long* list, int top, unsigned long long v) {
  int lo = 0, hi = top;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (list[mid] > v) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// Vector v of a row of `end` elements from `base` on, the first `skip` of which are not the row's: elements outside are -inf,
// and a vector that holds some is read element by element.
template <class T>
__device__ __forceinline__ uint4 tl_load(const T* base, int v, int skip, int end) {
  constexpr int E = TlVec<T>::E;
  const int i0 = v * E, whole = skip ? 1 : 0;
  if (unsigned(v - whole) < unsigned(end / E - whole)) return *reinterpret_cast<const uint4*>(base + i0);
  alignas(16) T edge[E];
#pragma unroll
  for (int j = 0; j < E; ++j) edge[j] = i0 + j >= skip && i0 + j < end ? base[i0 + j] : Cvt<T>::from_f(-INFINITY);
  return *reinterpret_cast<const uint4*>(edge);
}

template <class T, int TL_THREADS>
__global__ void __launch_bounds__(TL_THREADS, 1024 / TL_THREADS) token_logprobs_kernel(TlArgs a) {
  constexpr int TL_WARPS = TL_THREADS / 32;
  using V = TlVec<T>;
  constexpr int E = V::E;
  __shared__ TlShare s_share[TL_CLUSTER];                                // of the first CTA: one of each CTA
  __shared__ unsigned long long s_list[TL_CLUSTER][TL_TOP];
  __shared__ unsigned long long s_mine[TL_TOP], s_merged[TL_TOP], s_cand[TL_CAND], s_best[TL_WARPS];
  __shared__ uint32_t s_key[TL_THREADS], s_low[TL_THREADS];
  __shared__ TlShare s_warp[TL_WARPS];
  __shared__ int s_sel[TL_TOP + TL_SLACK], s_selected, s_count, s_have, s_bound;
  __shared__ uint32_t s_tau;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cl = a.cluster;
  const int cta = cl > 1 ? int(blockIdx.x) % cl : 0;
  const long row = blockIdx.x / cl;
  pdl_wait();
  pdl_trigger();
  if (cl > 1) tl_arrive();                                               // met before the first CTA's memory is written to
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const int skip = int(reinterpret_cast<uintptr_t>(x) & 15) / int(sizeof(T));
  const T* base = x - skip;                                              // aligned; element i of the row is base[skip + i]
  const int end = a.vocab + skip, vectors = (end + E - 1) / E;
  const int v_lo = int(long(vectors) * cta / cl), v_hi = int(long(vectors) * (cta + 1) / cl);
  const int left = v_lo + tid < v_hi ? (v_hi - v_lo - tid + TL_THREADS - 1) / TL_THREADS : 0;        // this thread's vectors
  const int rounds = (v_hi - v_lo + TL_THREADS - 1) / TL_THREADS;
  const float none = -INFINITY;
  // of those, the ones whole in the row: all but the row's first and last vector
  const int whole = v_lo + tid < end / E ? min(left, (end / E - v_lo - tid + TL_THREADS - 1) / TL_THREADS) : 0;
  const uint4 nothing = make_uint4(V::NONE, V::NONE, V::NONE, V::NONE);
  const uint4* from = reinterpret_cast<const uint4*>(base) + v_lo + tid;
  uint4 next[TL_BATCH];
#pragma unroll
  for (int k = 0; k < TL_BATCH; ++k) next[k] = k < left ? tl_load(base, v_lo + tid + k * TL_THREADS, skip, end) : nothing;
  long wide = -1;
  if (a.tokens) wide = a.wide_tokens ? static_cast<const long*>(a.tokens)[row * a.token_stride] : static_cast<const int*>(a.tokens)[row * a.token_stride];
  const bool given = wide >= 0 && wide < a.vocab;
  const int t = given ? int(wide) + skip : -1;                           // places count from base
  const float xt = given ? Cvt<T>::to_f(base[t]) : 0.f;
  const uint32_t kt = tl_key(xt);
  // comparisons of floats are those of keys where the token's logit is a normal number that `finite` keeps
  const bool plain = fabsf(xt) >= 1.17549435e-38f && xt > V::LOW && xt < INFINITY;
  const int vt = plain ? t / E : -1;                                     // the token's vector: before it x >= xt counts, from it on x > xt
  const float above = plain ? tl_value(kt - 1) : INFINITY;               // x > above is x >= xt

  float m = none, m_hi = 0.f, m_lo = 0.f;                                // the warp's
  float mine = none, r = 0.f, e = 0.f;                                   // the lane's; e in units of ln 2, both without 2^-m_lo
  uint32_t mk = tl_key(none);
  int equal = 0, ahead = 0;
  if (tid == 0) s_selected = 0, s_count = 0, s_bound = 0x7fffffff, s_have = 0;
  for (int k0 = 0; k0 < rounds; k0 += TL_BATCH) {
    uint4 raw[TL_BATCH];
    float vm[TL_BATCH], top = none;
#pragma unroll
    for (int k = 0; k < TL_BATCH; ++k) {
      raw[k] = next[k];
      vm[k] = V::largest(raw[k]);
      top = tl_max_nan(top, vm[k]);
    }
    from += TL_BATCH * TL_THREADS;
#pragma unroll
    for (int k = 0; k < TL_BATCH; ++k) {
      const int kn = k0 + TL_BATCH + k;
      next[k] = nothing;
      if (kn < whole) next[k] = from[k * TL_THREADS];
      else if (kn < left) next[k] = tl_load(base, v_lo + tid + kn * TL_THREADS, skip, end);
    }
    mine = tl_max_nan(mine, top);
    const uint32_t bk = __reduce_max_sync(0xffffffffu, tl_key(top));
    if (bk > mk) {
      const float up = tl_value(bk);
      if (m != none) {                                                   // what is held is relative to a lower maximum
        const float d = (m - up) * TL_LOG2E, w = tl_exp2(d), fix = tl_exp2(-m_lo), n = fmaf(r, fix, float(equal));
        e = w != 0.f ? ((e - m_lo * r) * fix + d * n) * w : 0.f;
        r = n * w;
        equal = 0;
      }
      m_hi = up * TL_LOG2E;                                              // m log2 e in two parts
      m_lo = up > V::FROM && up < TL_FAR ? fmaf(up, TL_LOG2E, -m_hi) : 0.f;        // only terms of the branch below lack 2^-m_lo
      m = up, mk = bk;
    }
    if (m > V::FROM && m < TL_FAR) {
      const unsigned long long minus = tl_two(-m_hi, -m_hi), log2e = tl_two(TL_LOG2E, TL_LOG2E);
      unsigned long long r2 = 0, e2 = 0;
      if (top > above) {                                                 // logits before the token's
        typename V::Count count(xt);
#pragma unroll
        for (int k = 0; k < TL_BATCH; ++k) {
          if (v_lo + tid + (k0 + k) * TL_THREADS < vt) count.add(raw[k], true);
          else count.add(raw[k], false);
        }
        ahead += count.sum();
      }
#pragma unroll
      for (int k = 0; k < TL_BATCH; ++k) {
        if (k0 + k >= rounds) break;                                     // the same for the whole CTA
        float f[E];
        V::unpack(V::finite(raw[k]), f);
        if (vm[k] == m) {
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (f[j] == m) ++equal, f[j] = -1e32f;
        }
#pragma unroll
        for (int j = 0; j < E; j += 2) {
          const unsigned long long d = tl_fma2(tl_two(f[j], f[j + 1]), log2e, minus);
          const float2 u = tl_split(d);
          const unsigned long long p = tl_two(tl_exp2(u.x), tl_exp2(u.y));
          r2 = tl_add2(r2, p), e2 = tl_fma2(d, p, e2);
        }
      }
      const float2 rs = tl_split(r2), es = tl_split(e2);
      r += rs.x + rs.y, e += es.x + es.y;
    } else {                                                             // nothing seen yet, or a maximum far out: differences first
      const uint32_t word = V::word(m);                                  // a mask's vectors, all maximum, are counted whole
      uint32_t mixed = 0;
#pragma unroll
      for (int k = 0; k < TL_BATCH; ++k)
        if (raw[k].x != word || raw[k].y != word || raw[k].z != word || raw[k].w != word) mixed |= 1u << k;
      for (int k = 0; k < TL_BATCH && k0 + k < left; ++k) {
        const float th = v_lo + tid + (k0 + k) * TL_THREADS < vt ? above : xt;
        if (!(mixed >> k & 1)) {
          if (m != none) equal += E, ahead += m > th ? E : 0;
          continue;
        }
        float f[E];
        V::unpack(tl_load(base, v_lo + tid + (k0 + k) * TL_THREADS, skip, end), f);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          ahead += f[j] > th ? 1 : 0;
          if (m == none) continue;
          const float d = fmaxf(f[j] - m, -1e30f) * TL_LOG2E, p = tl_exp2(d);        // -inf: weight 0, not 0 * inf
          if (f[j] == m) ++equal;
          else r += p, e += d * p;
        }
      }
    }
  }
  if (given && plain) {                                                  // equal logits in the token's own vector, in front of it
    if (v_lo <= vt && vt < v_hi && (vt - v_lo) % TL_THREADS == tid) {
      float f[E];
      V::unpack(tl_load(base, vt, skip, end), f);
#pragma unroll
      for (int j = 0; j < E; ++j) ahead += f[j] == xt && vt * E + j < t ? 1 : 0;
    }
  }
  if (given && (!plain || m != m)) {                                     // by keys
    ahead = 0;
    for (int k = 0; k < left; ++k) {
      const int v = v_lo + tid + k * TL_THREADS;
      float f[E];
      V::unpack(tl_load(base, v, skip, end), f);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const uint32_t key = tl_key(f[j]);
        ahead += v * E + j >= skip && v * E + j < end && (key > kt || (key == kt && v * E + j < t)) ? 1 : 0;
      }
    }
  }
  e = (e - m_lo * r) * tl_exp2(-m_lo) * 0.6931471805599453f;
  r *= tl_exp2(-m_lo);
  if (m != m) r = m;                                                     // NaN: the row's figures are NaN
  r = warp_sum(r), e = warp_sum(e);
  equal = __reduce_add_sync(0xffffffffu, equal);
  ahead = __reduce_add_sync(0xffffffffu, ahead);
  // one of the elements that equal the maximum stays out of the sum
  if (lane == 0) s_warp[warp] = TlShare{m, equal > 1 ? r + float(equal - 1) : r, e, ahead};
  s_key[tid] = left > 0 ? tl_key(mine) : 0u;
  if (tid < TL_TOP) s_mine[tid] = 0;
  __syncthreads();

  // ---- this share's best, sorted
  if (a.top > 0) {
    // a bound: the largest key that at least `top` threads reach
    if (warp == TL_WARPS - 1) {
      uint32_t tau = 0;
      int have = TL_THREADS;
      for (int bit = 31; bit >= 0 && have > a.top; --bit) {
        const uint32_t probe = tau | (1u << bit);
        int n = 0;
#pragma unroll
        for (int w = 0; w < TL_WARPS; ++w) n += s_key[w * 32 + lane] >= probe ? 1 : 0;
        n = __reduce_add_sync(0xffffffffu, n);
        if (n >= a.top) tau = probe, have = n;
      }
      if (lane == 0) s_tau = tau, s_have = have;
    }
    __syncthreads();
    const uint32_t tau = s_tau, key = s_key[tid];
    if (s_have > a.top + TL_SLACK) {
      // many threads share the bound's value: of those, the ones with the lowest places
      uint32_t low = 0x7fffffffu;
      if (key == tau && key != 0u) {
        for (int k = left - 1; k >= 0; --k) {
          const int v = v_lo + tid + k * TL_THREADS;
          float f[E];
          V::unpack(tl_load(base, v, skip, end), f);
#pragma unroll
          for (int j = E - 1; j >= 0; --j)
            if (tl_key(f[j]) == tau && v * E + j >= skip && v * E + j < end) low = uint32_t(v * E + j);
        }
      }
      s_low[tid] = low;
      __syncthreads();
      if (warp == 0) {
        int over = 0;
#pragma unroll
        for (int w = 0; w < TL_WARPS; ++w) over += s_key[w * 32 + lane] > tau ? 1 : 0;
        const int want = a.top - __reduce_add_sync(0xffffffffu, over);             // 1 or more of the ties
        uint32_t bound = 0x7fffffffu;                                            // the least that `want` places reach
        for (int bit = 30; bit >= 0; --bit) {
          const uint32_t probe = bound & ~(1u << bit);
          int n = 0;
#pragma unroll
          for (int w = 0; w < TL_WARPS; ++w) n += s_low[w * 32 + lane] <= probe ? 1 : 0;
          if (__reduce_add_sync(0xffffffffu, n) >= want) bound = probe;
        }
        if (lane == 0) s_bound = int(bound);
      }
      __syncthreads();
      if (key > tau || (key == tau && low <= uint32_t(s_bound) && low != 0x7fffffffu)) {
        const int n = atomicAdd(&s_selected, 1);
        if (n < TL_TOP + TL_SLACK) s_sel[n] = tid;
      }
    } else if (key >= tau && key != 0u) {
      s_sel[atomicAdd(&s_selected, 1)] = tid;
    }
    __syncthreads();
    const int selected = min(s_selected, TL_TOP + TL_SLACK), bound = s_bound;
    // a warp reads a selected thread's vectors again, one a lane
    for (int i = warp; i < selected; i += TL_WARPS) {
      const int who = s_sel[i];
      for (int v = v_lo + who + lane * TL_THREADS; v < v_hi; v += 32 * TL_THREADS) {
        const uint4 raw = tl_load(base, v, skip, end);
        if (tl_key(V::largest(raw)) < tau) continue;
        float f[E];
        V::unpack(raw, f);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const uint32_t fk = tl_key(f[j]);
          const int at = v * E + j;
          if ((fk > tau || (fk == tau && at <= bound)) && at >= skip && at < end) {
            const int n = atomicAdd(&s_count, 1);
            if (n < TL_CAND) s_cand[n] = tl_pair(fk, at - skip);
          }
        }
      }
    }
    __syncthreads();
    const int count = s_count;
    if (count <= TL_CAND) {
      for (int i = tid; i < count; i += TL_THREADS) {
        const unsigned long long v = s_cand[i];
        int better = 0;
        for (int j = 0; j < count; ++j) better += s_cand[j] > v ? 1 : 0;
        if (better < a.top) s_mine[better] = v;
      }
    } else {
      unsigned long long last = ~0ull;
      for (int k = 0; k < a.top; ++k) {
        unsigned long long best = 0;
        for (int q = 0; q < left; ++q) {
          const int v = v_lo + tid + q * TL_THREADS;
          float f[E];
          V::unpack(tl_load(base, v, skip, end), f);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const int at = v * E + j;
            const unsigned long long c = tl_pair(tl_key(f[j]), at - skip);
            if (at >= skip && at < end && c < last && c > best) best = c;
          }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const unsigned long long c = __shfl_xor_sync(0xffffffffu, best, o);
          best = c > best ? c : best;
        }
        if (lane == 0) s_best[warp] = best;
        __syncthreads();
        for (int w = 0; w < TL_WARPS; ++w) best = s_best[w] > best ? s_best[w] : best;
        if (tid == 0) s_mine[k] = best;
        last = best;
        __syncthreads();
      }
    }
    __syncthreads();
  }

  // ---- into the first CTA
  if (cl > 1) tl_wait();
  if (tid < a.top) {
    if (cl > 1) tl_store(tl_remote(&s_list[cta][tid], 0), s_mine[tid]);
    else s_merged[tid] = s_mine[tid];
  }
  if (tid == 0) {
    const TlShare s = tl_join(s_warp, TL_WARPS);
    if (cl > 1) {
      const uint32_t to = tl_remote(&s_share[cta], 0);
      tl_store(to, __float_as_uint(s.m));
      tl_store(to + 4, __float_as_uint(s.r));
      tl_store(to + 8, __float_as_uint(s.e));
      tl_store(to + 12, uint32_t(s.ahead));
    } else {
      s_share[0] = s;
    }
  }
  if (cl > 1) {
    tl_arrive();
    tl_wait();
    if (cta != 0) return;
    for (int i = tid; i < cl * a.top; i += TL_THREADS) {
      const int c = i / a.top;
      const unsigned long long v = s_list[c][i - c * a.top];
      int better = i - c * a.top;
      for (int o = 0; o < cl; ++o)
        if (o != c) better += tl_above(s_list[o], a.top, v);
      if (v != 0 && better < a.top) s_merged[better] = v;
    }
  }
  __syncthreads();
  if (warp != 0) return;
  const TlShare all = tl_join(s_share, cl);
  const bool empty = all.m == none;                                      // no token has a probability
  const float lz = empty ? 0.f : log1pf(all.r) + (all.m - all.m);        // NaN where the maximum is none or infinite
  if (tid == 0) {
    a.logprob[row] = given ? (empty ? none : (xt - all.m) - lz) : 0.f;
    a.rank[row] = given ? all.ahead + 1 : 0;
    a.entropy[row] = empty ? 0.f : lz - all.e / (1.f + all.r);
  }
  if (tid < a.top) {
    const unsigned long long v = s_merged[tid];
    a.top_ids[row * a.top + tid] = int(~uint32_t(v));
    a.top_logprobs[row * a.top + tid] = empty ? none : (tl_value(uint32_t(v >> 32)) - all.m) - lz;
  }
}

}  // namespace ronn

using namespace ronn;

template <class T, int TL_THREADS>
static int launch_token_logprobs(const TlArgs& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.rows * a.cluster));
  cfg.blockDim = dim3(TL_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(a.cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, TL_THREADS>, a) == cudaSuccess ? 0 : -100;
}

// One call.  logits: [rows, ld], dtype 0 bf16, 1 fp16, 2 fp32; tokens: int32 (wide_tokens: int64) every token_stride values, or
// null (a token outside [0, vocab) is not given: log probability 0, rank 0); top_ids, top_logprobs: [rows, top], top <= min(vocab, 32).
struct TokenLogprobsCall {
  const void *logits, *tokens;
  float *logprob, *entropy, *top_logprobs;
  int *rank, *top_ids;
  long ld, rows, token_stride;
  int vocab, wide_tokens, top, dtype;
};

extern "C" int ronn_token_logprobs(const TokenLogprobsCall* call, cudaStream_t stream) {
  const auto& [logits, tokens, logprob, entropy, top_logprobs, rank, top_ids, ld, rows, token_stride, vocab, wide_tokens, top, dtype] = *call;
  if (rows <= 0) return 0;
  if (vocab <= 0 || vocab > (1 << 30) || top < 0 || top > TL_TOP || top > vocab || rows > 2147483647L / TL_CLUSTER) return -2;
  if (dtype < 0 || dtype > 2) return -1;
  // CTAs of a row: more while there are fewer than SMs and each thread still has a batch of vectors.  256 x 50257 fp32 with five
  // alternatives took 24.6 us with 1 or 2, 31 with 4, 49 with 8 (now 22.5 with 2); 1 x 50257 took 20, 15.8, 13.8 and 13.8.
  const long vectors = vocab / (dtype == 2 ? 4 : 8);
  int cl = 1;
  while (cl < TL_CLUSTER && rows * cl < device_sm_count() && vectors >= 2L * cl * 256 * TL_BATCH) cl *= 2;
  const TlArgs a{logits, tokens, logprob, entropy, top_logprobs, rank, top_ids, ld, token_stride, rows, vocab, top, cl, wide_tokens};
  // Many short rows: CTAs of 64 threads, 16 to an SM.  Microseconds with 256 and with 64 threads, five alternatives: 4800 x 1000
  // bf16 66 and 41, 2400 x 4728 41 and 33, 600 x 12000 22.6 and 18.4; but 4800 x 32000 124 and 127, 300 x 12000 14.3 and 18.4.
  const bool narrow = cl == 1 && rows >= 4L * device_sm_count() && vectors <= 1500;
#define RONN_TL(T) return narrow ? launch_token_logprobs<T, 64>(a, stream) : launch_token_logprobs<T, 256>(a, stream)
  if (dtype == 0) RONN_TL(__nv_bfloat16);
  if (dtype == 1) RONN_TL(__half);
  RONN_TL(float);
#undef RONN_TL
}
