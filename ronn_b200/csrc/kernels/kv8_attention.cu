// Attention over the 8-bit paged KV cache (kv8.cuh): o = softmax(scale q k^T) v with k and v as the cache holds them.
//
//   ronn_kv8_attention : query rows grouped by sequence.  Sequence s has q_len[s] queries from row seq_start[s] on (without
//                        these two: row s, one query) and attends to the kv_len[s] keys its block-table row lists; with
//                        `causal` its queries are the last positions of that context.  Queries without keys give zeros.
//
// First form: one warp per (query, head), one token at a time, statistics and sums in 32 bits.
#include "kv8.cuh"

namespace ronn {

struct Kv8AttnArgs {
  const void* q;
  void* out;
  const uint8_t* kcodes;
  const uint8_t* vcodes;
  const float* kscale;
  const float* vscale;
  const int* tables;
  const int* kv_len;
  const int* bt_row;
  const int* seq_start;
  const int* q_len;
  uint32_t* status;
  long ld_q, ld_o, num_blocks, rows, table_ld;
  int table_rows, max_blocks, heads, kv_heads, causal;
  float scale_log2;
};

template <class T, int D, int CODE>
__global__ void __launch_bounds__(32) kv8_attention_kernel(Kv8AttnArgs a) {
  constexpr int PER = D / 32;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x;
  const int seq = blockIdx.x, head = blockIdx.y, qi = blockIdx.z;
  const int n = a.q_len ? a.q_len[seq] : 1;
  if (qi >= n) return;
  const long row = a.seq_start ? long(a.seq_start[seq]) + qi : seq;
  int table = a.bt_row ? a.bt_row[seq] : seq;
  int len = min(a.kv_len[seq], a.max_blocks * KV8_BLOCK);
  if (row < 0 || row >= a.rows) {
    if (lane == 0) kv8_report(a.status);
    return;
  }
  if (table < 0 || table >= a.table_rows) {
    if (lane == 0) kv8_report(a.status);
    len = 0;
  }
  if (a.causal) len -= n - 1 - qi;
  const int kvh = head / (a.heads / a.kv_heads);
  const T* q = static_cast<const T*>(a.q) + row * a.ld_q + long(head) * D + lane * PER;
  float qf[PER], acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) qf[i] = Cvt<T>::to_f(q[i]) * a.scale_log2, acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int t = 0; t < len; ++t) {
    const int blk = a.tables[long(table) * a.table_ld + t / KV8_BLOCK];
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0) kv8_report(a.status);
      continue;
    }
    const long unit = long(blk) * a.kv_heads + kvh;
    const long at = (unit * KV8_BLOCK + t % KV8_BLOCK) * D + lane * PER;
    float s = 0.f, kf[PER], vf[PER];
#pragma unroll
    for (int i = 0; i < PER; i += 2) {
      const float2 k = kv8_unpack2<CODE>(*reinterpret_cast<const uint16_t*>(a.kcodes + at + i));
      const float2 v = kv8_unpack2<CODE>(*reinterpret_cast<const uint16_t*>(a.vcodes + at + i));
      kf[i] = k.x, kf[i + 1] = k.y, vf[i] = v.x, vf[i + 1] = v.y;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) s += qf[i] * kf[i];
    s = warp_sum(s) * a.kscale[unit];
    const float vs = a.vscale[unit];
    const float mn = fmaxf(m, s);
    const float c = exp2f(m - mn), p = exp2f(s - mn);
    l = l * c + p;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = acc[i] * c + p * (vf[i] * vs);
    m = mn;
  }
  T* o = static_cast<T*>(a.out) + row * a.ld_o + long(head) * D + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; ++i) o[i] = Cvt<T>::from_f(len > 0 ? acc[i] / l : 0.f);
}

}  // namespace ronn

using namespace ronn;

// q, out: 16-bit [rows, ld]; dtype 0 bf16, 1 fp16; code 0 int8, 1 e4m3; head_dim 64 or 128.  max_q_len bounds q_len.
extern "C" int ronn_kv8_attention(const void* q, long ld_q, long rows, const void* kcodes, const void* vcodes, const float* kscale,
                                  const float* vscale, long num_blocks, const int* tables, long table_ld, int table_rows, int max_blocks,
                                  const int* bt_row, const int* seq_start, const int* q_len, const int* kv_len, void* out,
                                  long ld_o, int n_seq, int max_q_len, int heads, int kv_heads, int head_dim, int causal,
                                  float scale, int dtype, int code, uint32_t* status, cudaStream_t stream) {
  if (n_seq <= 0 || max_q_len <= 0) return 0;
  if (heads <= 0 || heads > 65535 || kv_heads <= 0 || heads % kv_heads || max_q_len > 65535 || (ld_q & 7) || (ld_o & 7)) return -2;
  if ((seq_start == nullptr) != (q_len == nullptr)) return -2;
  Kv8AttnArgs a{q, out, (const uint8_t*)kcodes, (const uint8_t*)vcodes, kscale, vscale, tables, kv_len, bt_row, seq_start, q_len,
                status, ld_q, ld_o, num_blocks, rows, table_ld, table_rows, max_blocks, heads, kv_heads, causal, scale * 1.4426950408889634f};
  const dim3 grid{unsigned(n_seq), unsigned(heads), unsigned(max_q_len)};
#define RONN_KV8T(T, D, C) launch(kv8_attention_kernel<T, D, C>, grid, dim3(32), 0, stream, a)
#define RONN_KV8T_(T) \
  do { \
    if (head_dim == 64 && code == 0) RONN_KV8T(T, 64, 0); \
    else if (head_dim == 64 && code == 1) RONN_KV8T(T, 64, 1); \
    else if (head_dim == 128 && code == 0) RONN_KV8T(T, 128, 0); \
    else if (head_dim == 128 && code == 1) RONN_KV8T(T, 128, 1); \
    else return -1; \
  } while (0)
  if (dtype == 0) RONN_KV8T_(__nv_bfloat16);
  else if (dtype == 1) RONN_KV8T_(__half);
  else return -1;
#undef RONN_KV8T
#undef RONN_KV8T_
  return cudaGetLastError() == cudaSuccess ? 0 : -100;
}
