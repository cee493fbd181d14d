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
// Bound by memory: each logit is read once and stays in registers, up to 8 16-byte vectors a thread.  A row is shared by a
// cluster of 1 to 8 CTAs; each finds its maximum, its sums and its own best `top` tokens, and writes them into the first
// CTA's shared memory, where they are put together.  No scratch in global memory, no atomics whose order shows.
// The best tokens of a share: the top-th best of its threads' maxima bounds them from below, so at most that many threads
// (and a few more) hold candidates, at most 64 each; a rank among the candidates is their number of betters.
// Vocabularies beyond 8 CTAs go by in tiles, with the result so far as one more share.
#include "common.cuh"

namespace ronn {

constexpr int TL_THREADS = 512;
constexpr int TL_WARPS = TL_THREADS / 32;
constexpr int TL_TOP = 32;
constexpr int TL_CLUSTER = 8;
constexpr int TL_SLACK = 8;            // threads beyond `top` that may offer candidates
constexpr int TL_CAND = (TL_TOP + TL_SLACK) * 64;

struct TlArgs {
  const void* logits;
  const void* tokens;
  float *logprob, *entropy, *top_logprobs;
  int *rank, *top_ids;
  long ld, token_stride, rows;
  int vocab, top, cluster, tiles, wide_tokens;
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
__device__ __forceinline__ float tl_exp(float d) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * 1.4426950408889634f));
  return y;
}

// A 16-byte vector of logits as E = 4 or 8 floats.
template <class T> struct TlVec {
  static constexpr int E = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    Pair16<T>::unpack(v.x, f[0], f[1]);
    Pair16<T>::unpack(v.y, f[2], f[3]);
    Pair16<T>::unpack(v.z, f[4], f[5]);
    Pair16<T>::unpack(v.w, f[6], f[7]);
  }
};
template <> struct TlVec<float> {
  static constexpr int E = 4;
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

template <class T, int NV>
__global__ void __launch_bounds__(TL_THREADS, 2) token_logprobs_kernel(TlArgs a) {
  using V = TlVec<T>;
  constexpr int E = V::E;
  __shared__ TlShare s_share[TL_CLUSTER + 1];                            // of the first CTA: one of each CTA, and the row so far
  __shared__ unsigned long long s_list[TL_CLUSTER + 1][TL_TOP];
  __shared__ unsigned long long s_mine[TL_TOP], s_cand[TL_CAND], s_merged[TL_TOP];
  __shared__ uint32_t s_key[TL_THREADS];
  __shared__ float s_m[TL_WARPS], s_r[TL_WARPS], s_e[TL_WARPS];
  __shared__ int s_ahead[TL_WARPS], s_owner, s_count, s_bound;
  __shared__ uint32_t s_tau;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cl = a.cluster;
  const int cta = cl > 1 ? int(blockIdx.x) % cl : 0;
  const long row = blockIdx.x / cl;
  pdl_wait();
  pdl_trigger();
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const uintptr_t at = reinterpret_cast<uintptr_t>(x);
  const int skip = int(at & 15) / int(sizeof(T));                        // elements before the row in its first vector
  const T* base = x - skip;
  long wide = -1;
  if (a.tokens) wide = a.wide_tokens ? static_cast<const long*>(a.tokens)[row * a.token_stride] : static_cast<const int*>(a.tokens)[row * a.token_stride];
  const bool given = wide >= 0 && wide < a.vocab;
  const int t = given ? int(wide) : -1;
  const float xt = given ? Cvt<T>::to_f(x[t]) : 0.f;
  const float none = -INFINITY;

  for (int tile = 0; tile < a.tiles; ++tile) {
    const int v0 = (tile * cl + cta) * (NV * TL_THREADS) + tid;   // this thread's vectors: v0 + k * TL_THREADS
    uint4 raw[NV];
    // ---- read; vectors that hold elements outside the row come element by element
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i0 = (v0 + k * TL_THREADS) * E - skip;
      if (i0 >= 0 && i0 + E <= a.vocab) {
        raw[k] = *reinterpret_cast<const uint4*>(base + i0 + skip);
      } else {
        alignas(16) T edge[E];
#pragma unroll
        for (int j = 0; j < E; ++j) edge[j] = i0 + j >= 0 && i0 + j < a.vocab ? x[i0 + j] : Cvt<T>::from_f(none);
        raw[k] = *reinterpret_cast<const uint4*>(edge);
      }
    }
    float mine = none;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[E];
      V::unpack(raw[k], f);
#pragma unroll
      for (int j = 0; j < E; ++j) mine = tl_max_nan(mine, f[j]);
    }
    float m = mine;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = tl_max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s_m[warp] = m;
    if (tid == 0) s_owner = TL_THREADS, s_count = 0, s_bound = 0x7fffffff;
    s_key[tid] = tl_key(mine);
    if (tid < TL_TOP) s_mine[tid] = 0;
    __syncthreads();
    m = s_m[0];
#pragma unroll
    for (int w = 1; w < TL_WARPS; ++w) m = tl_max_nan(m, s_m[w]);
    if (mine == m) atomicMin(&s_owner, tid);
    // ---- a bound for the best: the largest key that at least `top` threads reach
    if (a.top > 0 && warp == 0) {
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
      if (lane == 0) s_tau = tau, s_count = have;
    }
    __syncthreads();
    // ---- sums relative to this share's maximum, without one element that equals it
    const bool owner = s_owner == tid;
    float r0 = 0.f, r1 = 0.f, e0 = 0.f, e1 = 0.f;
    if (m != none) {
      bool leave = owner;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float f[E];
        V::unpack(raw[k], f);
        if (!leave) {
#pragma unroll
          for (int j = 0; j < E; j += 2) {
            const float da = fmaxf(f[j] - m, -1e30f), db = fmaxf(f[j + 1] - m, -1e30f);      // -inf: weight 0, not 0 * inf
            const float pa = tl_exp(da), pb = tl_exp(db);
            r0 += pa, r1 += pb, e0 += da * pa, e1 += db * pb;
          }
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const float d = fmaxf(f[j] - m, -1e30f), p = tl_exp(d);
            if (leave && f[j] == m) leave = false;
            else r0 += p, e0 += d * p;
          }
        }
      }
      if (m != m) r0 = m;                                               // NaN: the row's figures are NaN
    }
    // ---- logits before the token's
    int ahead = 0;
    if (given) {
      // comparisons of floats are those of keys where the token's logit is a normal number
      const bool plain = fabsf(xt) >= 1.17549435e-38f && xt != none && mine == mine;
      const uint32_t kt = tl_key(xt);
      if (plain && mine >= xt) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int i0 = (v0 + k * TL_THREADS) * E - skip;
          float f[E];
          V::unpack(raw[k], f);
          if (i0 > t) {
#pragma unroll
            for (int j = 0; j < E; ++j) ahead += f[j] > xt ? 1 : 0;
          } else if (i0 + E <= t) {
#pragma unroll
            for (int j = 0; j < E; ++j) ahead += f[j] >= xt ? 1 : 0;
          } else {
#pragma unroll
            for (int j = 0; j < E; ++j) ahead += f[j] > xt || (f[j] == xt && i0 + j < t) ? 1 : 0;
          }
        }
      } else if (!plain) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int i0 = (v0 + k * TL_THREADS) * E - skip;
          float f[E];
          V::unpack(raw[k], f);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const uint32_t key = tl_key(f[j]);
            ahead += i0 + j >= 0 && i0 + j < a.vocab && (key > kt || (key == kt && i0 + j < t)) ? 1 : 0;
          }
        }
      }
    }
    const float r = warp_sum(r0 + r1), e = warp_sum(e0 + e1);
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    if (lane == 0) s_r[warp] = r, s_e[warp] = e, s_ahead[warp] = ahead;
    // ---- this share's best, sorted
    if (a.top > 0) {
      const uint32_t tau = s_tau, mk = s_key[tid];
      const int have = s_count;
      __syncthreads();
      if (tid == 0) s_count = 0;
      // many threads may share the bound's value: of those, the ones with the lowest indices
      if (have > a.top + TL_SLACK) {
        int low = 0x7fffffff;
        if (mk == tau) {
#pragma unroll
          for (int k = NV - 1; k >= 0; --k) {
            const int i0 = (v0 + k * TL_THREADS) * E - skip;
            float f[E];
            V::unpack(raw[k], f);
#pragma unroll
            for (int j = E - 1; j >= 0; --j)
              if (tl_key(f[j]) == tau && i0 + j >= 0 && i0 + j < a.vocab) low = i0 + j;
          }
        }
        // s_cand is free until the barrier after this
        int* s_low = reinterpret_cast<int*>(s_cand);
        s_low[tid] = mk == tau ? low : 0x7fffffff;
        __syncthreads();
        if (warp == 0) {
          int over = 0;
#pragma unroll
          for (int w = 0; w < TL_WARPS; ++w) over += s_key[w * 32 + lane] > tau ? 1 : 0;
          const int want = a.top - __reduce_add_sync(0xffffffffu, over);           // 1 or more of the ties
          int bound = 0x7fffffff;                                                // the least bound that `want` indices reach
#pragma unroll 1
          for (int bit = 30; bit >= 0; --bit) {
            const int probe = bound & ~(1 << bit);
            int n = 0;
#pragma unroll
            for (int w = 0; w < TL_WARPS; ++w) n += s_low[w * 32 + lane] <= probe ? 1 : 0;
            if (__reduce_add_sync(0xffffffffu, n) >= want) bound = probe;
          }
          if (lane == 0) s_bound = bound;
        }
      }
      __syncthreads();
      const int bound = s_bound;
      if (mk >= tau) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int i0 = (v0 + k * TL_THREADS) * E - skip;
          float f[E];
          V::unpack(raw[k], f);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const uint32_t key = tl_key(f[j]);
            const int i = i0 + j;
            if ((key > tau || (key == tau && i <= bound)) && i >= 0 && i < a.vocab) {
              const int n = atomicAdd(&s_count, 1);
              if (n < TL_CAND) s_cand[n] = tl_pair(key, i);
            }
          }
        }
      }
      __syncthreads();
      const int count = min(s_count, TL_CAND);
      for (int i = tid; i < count; i += TL_THREADS) {
        const unsigned long long v = s_cand[i];
        int better = 0;
        for (int j = 0; j < count; ++j) better += s_cand[j] > v ? 1 : 0;
        if (better < a.top) s_mine[better] = v;
      }
    }
    __syncthreads();
    // ---- into the first CTA
    if (cl > 1) tl_arrive();                                             // the first CTA has started, and has read the last tile's
    if (cl > 1) tl_wait();
    if (tid < a.top) {
      if (cl > 1) tl_store(tl_remote(&s_list[cta][tid], 0), s_mine[tid]);
      else s_list[0][tid] = s_mine[tid];
    }
    if (tid == 0) {
      float sr = 0.f, se = 0.f;
      int sa = 0;
      for (int w = 0; w < TL_WARPS; ++w) sr += s_r[w], se += s_e[w], sa += s_ahead[w];
      if (cl > 1) {
        const uint32_t to = tl_remote(&s_share[cta], 0);
        tl_store(to, __float_as_uint(m));
        tl_store(to + 4, __float_as_uint(sr));
        tl_store(to + 8, __float_as_uint(se));
        tl_store(to + 12, uint32_t(sa));
      } else {
        s_share[0] = TlShare{m, sr, se, sa};
      }
    }
    if (cl > 1) {
      tl_arrive();
      tl_wait();
    } else {
      __syncthreads();
    }
    if (cta != 0) continue;
    // ---- put together, with the row so far at place cl
    const int shares = cl + (tile > 0 ? 1 : 0);
    int best = 0;
    for (int c = 1; c < shares; ++c)
      if (tl_key(s_share[c].m) > tl_key(s_share[best].m)) best = c;
    TlShare all = s_share[best];
    for (int c = 0; c < shares; ++c) {
      if (c == best) continue;
      const TlShare s = s_share[c];
      all.ahead += s.ahead;
      const float d = s.m - all.m, w = tl_exp(d);
      if (w != 0.f) all.r += w * (1.f + s.r), all.e += w * (s.e + d * (1.f + s.r));
    }
    if (shares > 1) {
      for (int i = tid; i < shares * a.top; i += TL_THREADS) {
        const int c = i / a.top;
        const unsigned long long v = s_list[c][i - c * a.top];
        int better = i - c * a.top;
        for (int o = 0; o < shares; ++o)
          if (o != c) better += tl_above(s_list[o], a.top, v);
        if (v != 0 && better < a.top) s_merged[better] = v;
      }
    } else if (tid < a.top) {
      s_merged[tid] = s_list[0][tid];
    }
    __syncthreads();
    if (tile + 1 < a.tiles) {
      if (tid < a.top) s_list[cl][tid] = s_merged[tid];
      if (tid == 0) s_share[cl] = all;
      continue;
    }
    const bool empty = all.m == none;                                    // no token has a probability
    const float lz = empty ? 0.f : log1pf(all.r) + (all.m - all.m);      // NaN where the maximum is none or infinite
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
}

}  // namespace ronn

using namespace ronn;

template <class T, int NV>
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
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, NV>, a) == cudaSuccess ? 0 : -100;
}

// logits: [rows, ld], dtype 0 bf16, 1 fp16, 2 fp32; tokens: int32 (wide_tokens: int64) every token_stride values, or null (a
// token outside [0, vocab) is not given: log probability 0, rank 0); top_ids, top_logprobs: [rows, top], top <= min(vocab, 32).
extern "C" int ronn_token_logprobs(const void* logits, long ld, int vocab, long rows, const void* tokens, long token_stride,
                                   int wide_tokens, float* logprob, int* rank, float* entropy, int* top_ids, float* top_logprobs,
                                   int top, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (vocab <= 0 || vocab > (1 << 30) || top < 0 || top > TL_TOP || top > vocab || rows > 2147483647L / TL_CLUSTER) return -2;
  if (dtype < 0 || dtype > 2) return -1;
  const int per = dtype == 2 ? 4 : 8;
  const long vectors = (long(vocab) + 2 * per - 2) / per;                // the row may start and end inside one
  // One CTA reads up to 8 vectors a thread.  More CTAs where the row is longer, and while there are fewer than SMs.
  int cl = 1;
  while (cl < TL_CLUSTER && (cl * 8L * TL_THREADS < vectors || (rows * cl < device_sm_count() && cl * long(TL_THREADS) < vectors))) cl *= 2;
  const long each = (vectors + cl * long(TL_THREADS) - 1) / (cl * long(TL_THREADS));          // vectors a thread
  const int nv = each <= 1 ? 1 : each <= 2 ? 2 : each <= 4 ? 4 : 8;
  TlArgs a{logits, tokens, logprob, entropy, top_logprobs, rank, top_ids, ld, token_stride, rows, vocab, top, cl, int((each + nv - 1) / nv),
           wide_tokens};
#define RONN_TL(T) \
  return nv == 1 ? launch_token_logprobs<T, 1>(a, stream) : nv == 2 ? launch_token_logprobs<T, 2>(a, stream) \
       : nv == 4 ? launch_token_logprobs<T, 4>(a, stream) : launch_token_logprobs<T, 8>(a, stream)
  if (dtype == 0) RONN_TL(__nv_bfloat16);
  if (dtype == 1) RONN_TL(__half);
  RONN_TL(float);
#undef RONN_TL
}
