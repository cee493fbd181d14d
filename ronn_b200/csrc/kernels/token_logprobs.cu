// Log probability, rank, entropy and likeliest alternatives of tokens, from logits.
//
// For a row x of V logits, m = max x and r = sum over all but one largest element of exp(x_j - m):
//     log p_t = (x_t - m) - log1p(r)      entropy = log1p(r) - sum (x_j - m) exp(x_j - m) / (1 + r)
// (log1p keeps the digits of a token that is nearly certain: log p = -r there.)  The rank of t is 1 + the number of logits
// above x_t, equal ones with a lower index counted; alternatives come in that order too.
//
// First form: one CTA per row reads it once for the maximum, once for the sums and the rank, and once per alternative.
#include "common.cuh"

namespace ronn {

constexpr int TL_THREADS = 256;

// Total order of the logits: larger first, then the lower index; NaN above everything, -0 equal to 0.
__device__ __forceinline__ uint32_t tl_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct TlPair {
  uint32_t key;
  int idx;
};
__device__ __forceinline__ TlPair tl_better(TlPair a, TlPair b) {
  return b.key > a.key || (b.key == a.key && b.idx < a.idx) ? b : a;
}
__device__ __forceinline__ TlPair tl_block_best(TlPair v, TlPair* scratch) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v = tl_better(v, TlPair{__shfl_xor_sync(0xffffffffu, v.key, o), __shfl_xor_sync(0xffffffffu, v.idx, o)});
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
  for (int w = 1; w < TL_THREADS / 32; ++w) v = tl_better(v, scratch[w]);
  return v;
}

template <class T>
__global__ void __launch_bounds__(TL_THREADS)
token_logprobs_kernel(const T* __restrict__ logits, long ld, int vocab, const int* __restrict__ tokens, float* __restrict__ logprob,
                      int* __restrict__ rank, float* __restrict__ entropy, int* __restrict__ top_ids,
                      float* __restrict__ top_logprobs, int top) {
  __shared__ TlPair s_best[TL_THREADS / 32];
  __shared__ float red[32];
  pdl_wait();
  pdl_trigger();
  const long row = blockIdx.x;
  const T* x = logits + row * ld;
  TlPair best{0u, 0x7fffffff};
  for (int j = threadIdx.x; j < vocab; j += TL_THREADS) best = tl_better(best, TlPair{tl_key(Cvt<T>::to_f(x[j])), j});
  best = tl_block_best(best, s_best);
  const float m = Cvt<T>::to_f(x[best.idx]);
  const int t = tokens ? tokens[row] : -1;
  const bool given = t >= 0 && t < vocab;
  const float xt = given ? Cvt<T>::to_f(x[t]) : 0.f;
  const uint32_t kt = tl_key(xt);
  float r = 0.f, e = 0.f, ahead = 0.f;
  for (int j = threadIdx.x; j < vocab; j += TL_THREADS) {
    const float xv = Cvt<T>::to_f(x[j]);
    if (given) {
      const uint32_t k = tl_key(xv);
      ahead += k > kt || (k == kt && j < t) ? 1.f : 0.f;
    }
    if (j == best.idx) continue;
    const float d = xv - m;
    const float p = expf(d);
    r += p;
    if (p != 0.f) e += d * p;
  }
  r = block_sum(r, red);
  e = block_sum(e, red);
  ahead = block_sum(ahead, red);
  const bool empty = m == -INFINITY;             // no token has a probability
  const float lz = empty ? 0.f : log1pf(r) + (m - m);
  if (threadIdx.x == 0) {
    logprob[row] = given ? (empty ? -INFINITY : (xt - m) - lz) : 0.f;
    rank[row] = given ? int(ahead) + 1 : 0;
    entropy[row] = empty ? 0.f : lz - e / (1.f + r);
  }
  TlPair last{0xffffffffu, -1};
  for (int k = 0; k < top; ++k) {
    TlPair v{0u, 0x7fffffff};
    for (int j = threadIdx.x; j < vocab; j += TL_THREADS) {
      const uint32_t key = tl_key(Cvt<T>::to_f(x[j]));
      if (key < last.key || (key == last.key && j > last.idx)) v = tl_better(v, TlPair{key, j});
    }
    v = tl_block_best(v, s_best);
    if (threadIdx.x == 0) {
      top_ids[row * top + k] = v.idx;
      const float xv = Cvt<T>::to_f(x[v.idx]);
      top_logprobs[row * top + k] = empty ? -INFINITY : (xv - m) - lz;
    }
    last = v;
  }
}

}  // namespace ronn

using namespace ronn;

// logits: [rows, ld], dtype 0 bf16, 1 fp16, 2 fp32; tokens: int32 [rows] or null (a token outside [0, vocab) is not given:
// log probability 0, rank 0); top_ids, top_logprobs: [rows, top], top <= min(vocab, 32).
extern "C" int ronn_token_logprobs(const void* logits, long ld, int vocab, long rows, const int* tokens, float* logprob, int* rank,
                                   float* entropy, int* top_ids, float* top_logprobs, int top, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (rows > 2147483647L || vocab <= 0 || top < 0 || top > 32 || top > vocab) return -2;
#define RONN_TL(T) launch(token_logprobs_kernel<T>, dim3(unsigned(rows)), dim3(TL_THREADS), 0, stream, (const T*)logits, ld, vocab, \
                          tokens, logprob, rank, entropy, top_ids, top_logprobs, top)
  if (dtype == 0) RONN_TL(__nv_bfloat16);
  else if (dtype == 1) RONN_TL(__half);
  else if (dtype == 2) RONN_TL(float);
  else return -1;
#undef RONN_TL
  return cudaGetLastError() == cudaSuccess ? 0 : -100;
}
