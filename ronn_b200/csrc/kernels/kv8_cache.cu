// Writing to and reading from the 8-bit paged KV cache (kv8.cuh has the layout and the mathematics).
//
//   ronn_kv8_append : the K and V columns of a fused QKV activation into their cache slots, optionally after rotary
//                     embedding of Q and K.
//   ronn_kv8_read   : whole cache blocks as 16-bit values.
//
// Both are bound by memory: append reads 2 bytes and writes 1 for every value (with rotary embedding it also reads and
// writes Q and writes K), read reads 1 and writes 2.  4384 tokens of 16 heads of 64 go in at 6.8 us, 3.9 TB/s; with rotary
// embedding 2000 tokens of 32 / 8 heads of 128 take 22 us: the pairs of floats of a rotated value, 17 operations, fill 68 % of
// the issue slots.
#include "kv8.cuh"

namespace ronn {

struct Kv8AppendArgs {
  const void* qkv;
  void* rotated;               // where rotated q and k go, columns as in qkv (may be qkv itself)
  const int* slots;            // [tokens], -1: not cached
  const int* positions;        // null: no rotary
  uint8_t* kcodes;
  uint8_t* vcodes;
  float* kscale;
  float* vscale;
  uint32_t* status;
  long ld, ld_rot, tokens, num_slots;
  int k_off, v_off, heads, kv_heads, per_cta, window;
};

// Tokens of one cache block stand in consecutive rows with rising slots; such a run (1 to 16 tokens) is one unit of work
// for each head, and a warp holds the head's part of it in registers: 16 tokens x 64 or 128 values, 16 or 32 registers.
// The block's largest magnitude, its scale, the codes and, where the scale grew, the older codes are the warp's own
// affair, without shared memory.  A CTA looks at the rows of its window, 16 or 1, for the first rows of runs (grid.x), and at
// a share of the heads (grid.y).
constexpr int KV8_AP_WARPS = 8;

template <class T, int D, int CODE, bool ROPE>
__global__ void __launch_bounds__(KV8_AP_WARPS * 32, ROPE ? 3 : 4)
kv8_append_kernel(Kv8AppendArgs a, Kv8Turns turns) {
  constexpr int CH = D / 8;                 // 16-byte chunks (lanes) per token
  constexpr int TPW = 32 / CH;              // tokens per warp pass
  constexpr int PASSES = KV8_BLOCK / TPW;
  constexpr int HALF = D / 2;
  extern __shared__ float4 s_cs[];          // [16][HALF], with rotary embedding
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / CH, chunk = lane % CH;
  // the window's rows and at least 15 behind them, one per lane
  const long w0 = long(blockIdx.x) * a.window;
  const long row = w0 + lane;
  int slot = row < a.tokens ? max(a.slots[row], -1) : -2;      // -2: past the end
  if (slot >= a.num_slots) {
    if (lane < a.window) kv8_report(a.status);
    slot = -1;
  }
  int before = __shfl_up_sync(0xffffffffu, slot, 1);
  if (lane == 0) {
    before = w0 > 0 ? max(a.slots[w0 - 1], -1) : -2;
    if (before >= a.num_slots) before = -1;
  }
  // a row goes on with the run of the row before it: next slot of the same block, or another row without a slot (those
  // only pass through the rotary embedding, in groups of at most 16)
  const bool goes_on = slot >= 0 ? before == slot - 1 && (slot & (KV8_BLOCK - 1)) != 0
                                 : slot == -1 && before == -1 && (row & (KV8_BLOCK - 1)) != 0;
  const uint32_t starts = __ballot_sync(0xffffffffu, !goes_on);          // rows past the end count as starts
  const uint32_t live = __ballot_sync(0xffffffffu, slot != -2);
  const int q_units = ROPE ? a.heads : 0;
  const int units = q_units + 2 * a.kv_heads;
  const int u0 = blockIdx.y * a.per_cta, u1 = min(units, u0 + a.per_cta);
  const T* qkv = static_cast<const T*>(a.qkv);

  for (uint32_t todo = starts & live & ((1u << a.window) - 1u); todo; todo &= todo - 1) {
    const int first = __ffs(todo) - 1;
    const uint32_t later = first < 31 ? starts >> (first + 1) : 0u;
    const int n = min(later ? __ffs(later) : 32 - first, KV8_BLOCK);     // rows of the run (a block's end ends it)
    const int slot0 = __shfl_sync(0xffffffffu, slot, first);
    const long t0 = w0 + first;
    if constexpr (ROPE) {
      __syncthreads();                       // the table of the run before has been read
      for (int i = threadIdx.x; i < n * HALF; i += KV8_AP_WARPS * 32)
        s_cs[i / HALF * HALF + kv8_angle_at<D>(i % HALF)] = kv8_cos_sin(turns.t[i % HALF], a.positions[t0 + i / HALF]);
      __syncthreads();
    }
    for (int u = u0 + warp; u < u1; u += KV8_AP_WARPS) {
      const bool is_q = u < q_units;
      const int kvu = u - q_units;
      const bool is_v = !is_q && kvu >= a.kv_heads;
      const int h = is_q ? u : is_v ? kvu - a.kv_heads : kvu;
      const long col = (is_q ? 0 : is_v ? a.v_off : a.k_off) + long(h) * D + chunk * 8;
      if (!is_q && slot0 < 0 && (is_v || !ROPE)) continue;
      Vec8 x[PASSES];
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int t = p * TPW + sub;
        if (t < n) x[p] = *reinterpret_cast<const Vec8*>(qkv + (t0 + t) * a.ld + col);
        else x[p] = Vec8{{0u, 0u, 0u, 0u}};
      }
      if (ROPE && !is_v) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          const int t = p * TPW + sub;
          Vec8 oth;
#pragma unroll
          for (int i = 0; i < 4; ++i) oth.w[i] = __shfl_xor_sync(0xffffffffu, x[p].w[i], CH / 2);
          if (t < n) {
            x[p] = kv8_rotate8<T, CH / 2>(x[p], oth, chunk < CH / 2, s_cs + t * HALF + chunk % (CH / 2));
            *reinterpret_cast<Vec8*>(static_cast<T*>(a.rotated) + (t0 + t) * a.ld_rot + col) = x[p];
          }
        }
      }
      if (is_q || slot0 < 0) continue;
      const long unit = long(slot0 / KV8_BLOCK) * a.kv_heads + h;
      kv8_store_run<T, D, CODE, PASSES>(x, chunk, sub, n, slot0 % KV8_BLOCK, (is_v ? a.vscale : a.kscale) + unit,
                                        (is_v ? a.vcodes : a.kcodes) + unit * (KV8_BLOCK * D));
    }
  }
}

// One warp for each (block, head, K or V): 16 x D codes -> 16 x D values, 16 bytes of codes a lane and pass.
template <class T, int D, int CODE>
__global__ void __launch_bounds__(256)
kv8_read_kernel(const uint8_t* __restrict__ kcodes, const uint8_t* __restrict__ vcodes, const float* __restrict__ kscale,
                const float* __restrict__ vscale, const int* __restrict__ blocks, T* __restrict__ kout, T* __restrict__ vout,
                long n, long num_blocks, int kv_heads, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long unit = (long(blockIdx.x) * 8 + (threadIdx.x >> 5));
  const long items = n * kv_heads;
  if (unit >= 2 * items) return;
  const bool is_v = unit >= items;
  const long item = is_v ? unit - items : unit;
  const long i = item / kv_heads;
  const int h = int(item - i * kv_heads);
  const int blk = blocks[i];
  const bool ok = blk >= 0 && blk < num_blocks;
  if (!ok && lane == 0) kv8_report(status);
  const long src = (long(ok ? blk : 0) * kv_heads + h);
  const uint4* codes = reinterpret_cast<const uint4*>((is_v ? vcodes : kcodes) + src * (KV8_BLOCK * D));
  const float s = ok ? (is_v ? vscale : kscale)[src] : 0.f;
  T* out = (is_v ? vout : kout) + item * (KV8_BLOCK * D);
  constexpr int PASSES = KV8_BLOCK * D / 512;
  uint4 c[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) c[p] = codes[p * 32 + lane];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const uint32_t w[4] = {c[p].x, c[p].y, c[p].z, c[p].w};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float f[8], g[4];
      kv8_unpack4<CODE>(w[2 * k], g);
      f[0] = g[0] * s, f[1] = g[1] * s, f[2] = g[2] * s, f[3] = g[3] * s;
      kv8_unpack4<CODE>(w[2 * k + 1], g);
      f[4] = g[0] * s, f[5] = g[1] * s, f[6] = g[2] * s, f[7] = g[3] * s;
      *reinterpret_cast<Vec8*>(out + (p * 32 + lane) * 16 + k * 8) = ok ? pack8<T>(f) : Vec8{{0u, 0u, 0u, 0u}};
    }
  }
}

}  // namespace ronn

using namespace ronn;

static int launch_status() { return cudaGetLastError() == cudaSuccess ? 0 : -100; }

// turns: head_dim / 2 fractions of a turn per position (kv8.cuh) or null without rotary embedding; positions null likewise.
// dtype 0 bf16, 1 fp16; code 0 int8, 1 e4m3; head_dim 64 or 128.
struct Kv8AppendCall {
  const void* qkv;
  void* rotated;
  const int *slots, *positions;
  const unsigned long long* turns;
  void *kcodes, *vcodes;
  float *kscale, *vscale;
  uint32_t* status;
  long ld, ld_rot, num_blocks, tokens;
  int k_off, v_off, heads, kv_heads, head_dim, dtype, code, pad;
};

extern "C" int ronn_kv8_append(const Kv8AppendCall* call, cudaStream_t stream) {
  const auto& [qkv, rotated, slots, positions, turns, kcodes, vcodes, kscale, vscale, status, ld, ld_rot, num_blocks, tokens, k_off, v_off,
               heads, kv_heads, head_dim, dtype, code, pad] = *call;
  if (tokens <= 0) return 0;
  if ((ld & 7) || (ld_rot & 7) || (k_off & 7) || (v_off & 7) || kv_heads <= 0 || heads < 0 || num_blocks < 0) return -2;
  if (positions && (!turns || !rotated)) return -2;
  Kv8Turns tn = {};
  if (positions)
    for (int j = 0; j < head_dim / 2 && j < KV8_MAX_HALF; ++j) tn.t[j] = turns[j];
  const int units = (positions ? heads : 0) + 2 * kv_heads;
  // Windows of 16 rows and, with rotary embedding, two units a warp (its table of angles serves more heads) where that gives two
  // CTAs an SM; else of one row and one unit a warp.  Microseconds with 16 rows and with one: 64 single tokens, 16 heads of 64,
  // 12.5 and 2.7 (with rotary 46 and 4.5: 16 rows put them one after the other), 20 prompts of 30 tokens with rotary 9.8 and
  // 6.6, one prompt of 300 tokens 2.7 and 3.7; but 16 prompts, 4384 tokens, 6.8 and 22.7.
  const long coarse = (tokens + KV8_BLOCK - 1) / KV8_BLOCK * ((units + 2 * KV8_AP_WARPS - 1) / (2 * KV8_AP_WARPS));
  const bool few = coarse < 2L * device_sm_count();
  const int window = few ? 1 : KV8_BLOCK, per_cta = positions && !few ? 2 * KV8_AP_WARPS : KV8_AP_WARPS;
  const long windows = (tokens + window - 1) / window;
  const int ys = (units + per_cta - 1) / per_cta;
  if (windows > 2147483647L || ys > 65535) return -2;
  Kv8AppendArgs a{qkv, rotated, slots, positions, (uint8_t*)kcodes, (uint8_t*)vcodes, kscale, vscale, status, ld, ld_rot, tokens,
                  num_blocks * KV8_BLOCK, k_off, v_off, heads, kv_heads, per_cta, window};
  const dim3 grid{unsigned(windows), unsigned(ys), 1u};
  const size_t smem = positions ? size_t(KV8_BLOCK) * (head_dim / 2) * sizeof(float4) : 0;
#define RONN_KV8A(T, D, C) \
  (positions ? launch(kv8_append_kernel<T, D, C, true>, grid, dim3(KV8_AP_WARPS * 32), smem, stream, a, tn) \
             : launch(kv8_append_kernel<T, D, C, false>, grid, dim3(KV8_AP_WARPS * 32), smem, stream, a, tn))
#define RONN_KV8A_(T) \
  do { \
    if (head_dim == 64 && code == 0) RONN_KV8A(T, 64, 0); \
    else if (head_dim == 64 && code == 1) RONN_KV8A(T, 64, 1); \
    else if (head_dim == 128 && code == 0) RONN_KV8A(T, 128, 0); \
    else if (head_dim == 128 && code == 1) RONN_KV8A(T, 128, 1); \
    else return -1; \
  } while (0)
  if (dtype == 0) RONN_KV8A_(__nv_bfloat16);
  else if (dtype == 1) RONN_KV8A_(__half);
  else return -1;
#undef RONN_KV8A
#undef RONN_KV8A_
  return launch_status();
}

// blocks: [n] cache blocks; kout, vout: [n, kv_heads, 16, head_dim].  A block outside the cache gives zeros and a status code.
struct Kv8ReadCall {
  const void *kcodes, *vcodes;
  const float *kscale, *vscale;
  const int* blocks;
  void *kout, *vout;
  uint32_t* status;
  long n, num_blocks;
  int kv_heads, head_dim, dtype, code;
};

extern "C" int ronn_kv8_read(const Kv8ReadCall* call, cudaStream_t stream) {
  const auto& [kcodes, vcodes, kscale, vscale, blocks, kout, vout, status, n, num_blocks, kv_heads, head_dim, dtype, code] = *call;
  if (n <= 0) return 0;
  if (kv_heads <= 0 || num_blocks <= 0) return -2;
  const long ctas = (2 * n * kv_heads + 7) / 8;
  if (ctas > 2147483647L) return -2;
#define RONN_KV8R(T, D, C) launch(kv8_read_kernel<T, D, C>, dim3(unsigned(ctas)), dim3(256), 0, stream, (const uint8_t*)kcodes, \
                                  (const uint8_t*)vcodes, kscale, vscale, blocks, (T*)kout, (T*)vout, n, num_blocks, kv_heads, status)
#define RONN_KV8R_(T) \
  do { \
    if (head_dim == 64 && code == 0) RONN_KV8R(T, 64, 0); \
    else if (head_dim == 64 && code == 1) RONN_KV8R(T, 64, 1); \
    else if (head_dim == 128 && code == 0) RONN_KV8R(T, 128, 0); \
    else if (head_dim == 128 && code == 1) RONN_KV8R(T, 128, 1); \
    else return -1; \
  } while (0)
  if (dtype == 0) RONN_KV8R_(__nv_bfloat16);
  else if (dtype == 1) RONN_KV8R_(__half);
  else return -1;
#undef RONN_KV8R
#undef RONN_KV8R_
  return launch_status();
}
