// Attention over the 8-bit paged KV cache (kv8.cuh): o = softmax(scale q k^T) v with k and v as the cache holds them.
//
//   ronn_kv8_attention : query rows grouped by sequence.  Sequence s has q_len[s] queries from row seq_start[s] on (without
//                        these two: row s, one query) and attends to the kv_len[s] keys its block-table row lists; with
//                        `causal` its queries are the last positions of that context.  Queries without keys give zeros.
//                        With append slots (one query per sequence, up to 16 heads to a KV head) the row's new K and V join
//                        the cache first.
//
// Bound by memory: every code is read once for all the queries that share it.  A warp takes cache blocks of 16 tokens one
// after the other, by asynchronous 16-byte copies into a ring of its own in shared memory and from there into the fragments
// of mma.sync m16n8k16:
//   S^T = K Q^T   A = 16 tokens, B = 8 query rows (heads of the group, queries of a chunk); the head dimension is the sum's
//                 index, so its order is free: lane (g, c) of the fragment takes 16 consecutive bytes of a token, and Q is laid
//                 out to match.
//   O^T = V^T P^T A = 16 channels, B = P^T: the accumulator of S^T, (token g, two rows), turned around by movmatrix.  V's
//                 channels are in free order too: lane (g, c) takes 8 or 16 consecutive bytes of c's four tokens and
//                 interleaves the bytes of two.
// Queries as B waste nothing on a decode step's missing rows: 8 products a block of 64 channels, not 12.
// The 16-byte pieces of a row stand in the ring in an order that depends on the row (Kv8Ring), so that neither read meets a
// bank twice.  With the blocks in registers (48 of them, and not enough left) or the ring and 80 registers a thread, 256 rows of 64
// to 768 keys, 16 heads of 64 in int8, took a quarter longer than with the ring and 128: 16 warps an SM without spills beat 24
// with.  They take 53 us, 4.2 TB/s of codes, and nothing is full: issue slots 58 %, ALU 50 %, DRAM 53 %, with 3.6 warps a scheduler
// to hide what each waits for.  An SM is idle for 12 % of the time on average, as the longest rows are alone at the end.  A block
// takes about 180 instructions (a third of them turn int8 into f16; e4m3 takes one for two codes), and a warp 1100 around its
// blocks.  Long contexts of e4m3 go by at 5 TB/s.
// Codes become f16 exactly.  Q in bf16 is scaled by a power of two for each row, so that it fits f16 (its 8 significant bits
// do; what is 2^-34 of the row's largest is lost).  Softmax statistics, sums and O are in 32 bits; P is rounded to f16 as
// 2^15 p, by at most 2^-11 of it or 2^-40.  The scale of a K block multiplies its scores, that of a V block its P,
// relative to the largest V scale of the 32 blocks that the warp looks up together.
#include "kv8.cuh"

#include <type_traits>

namespace ronn {

constexpr int KV8_NW = 4;        // warps of an attention CTA

struct Kv8AttnArgs {
  const void* q;
  void* out;
  uint8_t* kcodes;
  uint8_t* vcodes;
  float* kscale;
  float* vscale;
  const int* tables;
  const int* kv_len;
  const int* bt_row;
  const int* seq_start;
  const int* q_len;
  const int* slots;           // append: cache slot of each row's new token, or null
  const int* positions;       // rotary embedding of q and the new k, or null
  float* part;                // splits > 1: [item][split][rows][D + 2] partial results
  uint32_t* status;
  long ld_q, ld_o, num_blocks, rows, table_ld;
  int group, items_x, table_rows, max_blocks, heads, kv_heads, causal, splits, share, part_rows, max_q, max_keys, k_off, v_off;
  float scale_log2;
};

// A sequence's table row, the keys that it lists, and whether it has fewer than the sequence has keys: the others are left out.
struct Kv8Keys {
  int table, len;
  bool cut;
};
__device__ __forceinline__ Kv8Keys kv8_keys(const Kv8AttnArgs& a, int seq) {
  const int table = a.bt_row ? a.bt_row[seq] : seq, keys = a.kv_len[seq];
  const bool listed = table >= 0 && table < a.table_rows;
  const int len = listed ? min(keys, a.max_blocks * KV8_BLOCK) : 0;
  return {listed ? table : 0, len, !listed || len < keys};
}
// False for a sequence of a chunk whose rows or lengths pass the call's bounds: it is left out, and its rows stay as they are.
__device__ __forceinline__ bool kv8_takes_part(const Kv8AttnArgs& a, long row0, int n, int len) {
  return row0 >= 0 && n >= 0 && row0 + n <= a.rows && (!a.q_len || (n <= a.max_q && len <= a.max_keys));
}

__device__ __forceinline__ void kv8_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float kv8_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t kv8_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Weight of a partial result with maximum m and sum l beside others whose maximum is mx: none without keys, NaN for NaN.
__device__ __forceinline__ float kv8_weight(float m, float l, float mx) { return l == 0.f ? 0.f : l != l ? l : kv8_exp2(m - mx); }

__device__ __forceinline__ uint32_t kv8_turn(uint32_t a) {      // an 8 x 8 matrix of 16-bit values, transposed
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

// Four codes in a word -> two f16 pairs.  int8: x + 128 as the low byte of a half with exponent 2^10 is 1024 + 128 + x.
template <int CODE>
__device__ __forceinline__ void kv8_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CODE == KV8_INT8) {
    w ^= 0x80808080u;
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    asm("sub.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
  } else {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(uint16_t(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(uint16_t(w >> 16)));
  }
}

// Places in a block of codes in shared memory: row t's 16-byte pieces are permuted by an exclusive or with `turn(t)`.  A token
// of fragment column n is `token(n)`: for rows of 64 bytes, two rows to a line of banks, c's tokens are 2c and 2c + 1 in an order
// that gives the four c of one load rows of both parities.
template <int D> struct Kv8Ring {
  static constexpr int PIECES = D / 16;                                  // of a row
  static __device__ __forceinline__ int turn(int t) { return D == 64 ? ((t >> 2) & 1) * 2 : (((t >> 1) & 3) * 2) ^ ((t & 1) * 4); }
  static __device__ __forceinline__ int token(int n) { return D == 64 ? n ^ ((n >> 1) & 1) : n; }
  static __device__ __forceinline__ int at(int t, int piece) { return t * D + ((piece ^ turn(t)) << 4); }
};
template <int OFF>
__device__ __forceinline__ uint4 kv8_shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at), "n"(OFF) : "memory");
  return v;
}
template <int OFF>
__device__ __forceinline__ uint2 kv8_shared8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2 + %3];" : "=r"(v.x), "=r"(v.y) : "r"(at), "n"(OFF) : "memory");
  return v;
}
template <int TO, int FROM>
__device__ __forceinline__ void kv8_copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(to), "l"(from), "n"(TO), "n"(FROM) : "memory");
}

// The new K and V of one row into its slot, by one warp: kv8_append for a run of one token, K in lanes 0 to 15 and V in the
// others.  `ks` and `vs` become the block's scales.
template <class T, int D, int CODE>
__device__ __forceinline__ void kv8_append_one(const Kv8AttnArgs& a, long row, int slot, int kvh, const float4* cs, float& ks, float& vs) {
  constexpr int CH = D / 8;
  const int lane = threadIdx.x & 31, chunk = lane % CH;
  const bool is_v = lane >= 16;
  const T* src = static_cast<const T*>(a.q) + row * a.ld_q + (is_v ? a.v_off : a.k_off) + long(kvh) * D;
  Vec8 x = *reinterpret_cast<const Vec8*>(src + chunk * 8);
  const long unit = long(slot / KV8_BLOCK) * a.kv_heads + kvh;
  const int off = slot % KV8_BLOCK;
  float* scale = (is_v ? a.vscale : a.kscale) + unit;
  const float old = off > 0 ? *scale : 0.f;
  if (a.positions) {
    Vec8 oth;
#pragma unroll
    for (int i = 0; i < 4; ++i) oth.w[i] = __shfl_xor_sync(0xffffffffu, x.w[i], CH / 2);
    const Vec8 turned = kv8_rotate8<T, CH / 2>(x, oth, chunk < CH / 2, cs + chunk % (CH / 2));
    if (!is_v) x = turned;
  }
  uint32_t m = kv8_absmax(0u, x);
#pragma unroll
  for (int o = 8; o; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));       // over each half of the warp
  m = max(m & 0xffffu, m >> 16);
  float lo, hi;
  Pair16<T>::unpack(m, lo, hi);
  const float s = kv8_new_scale<CODE>(__float_as_uint(lo), old), inv = kv8_inverse(s);
  uint8_t* codes = (is_v ? a.vcodes : a.kcodes) + unit * (KV8_BLOCK * D);
  if (off > 0 && s != old) kv8_round_again<CODE>(codes, off * (D / 4), lane & 15, 16, old, inv);
  if ((lane & 15) == 0 && (off == 0 || s != old)) *scale = s;
  if ((lane & 15) < CH) *reinterpret_cast<uint2*>(codes + off * D + chunk * 8) = kv8_pack8<T, CODE>(x, inv);
  ks = __shfl_sync(0xffffffffu, s, 0), vs = __shfl_sync(0xffffffffu, s, 16);
}

// Barrier of the warps that share an item.
template <int WPI>
__device__ __forceinline__ void kv8_item_sync(int item) {
  if constexpr (WPI == KV8_NW) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(item + 1), "n"(WPI * 32) : "memory");
}

// An item is a tile of up to 16 query rows of one (sequence, KV head), and one of `splits` shares of its blocks; WPI of the
// CTA's warps work on it.  NT = 1: at most 8 rows.  U: blocks a warp works on at a time; ST: blocks in its ring, U at work and the others on their way.
// A warp's first loads start before q is fetched: the chain length -> page -> codes is the longer one.
template <class T, int D, int CODE, int NT, int WPI, int U, int ST>
__global__ void __launch_bounds__(KV8_NW * 32, D == 64 ? (NT == 1 ? 4 : 3) : (NT == 1 ? 4 : 2)) kv8_attention_kernel(Kv8AttnArgs a, Kv8Turns turns) {
  constexpr int KW = D / 64;                  // 16-byte loads of K a lane and 8 tokens
  constexpr int VB = D / 8;                   // bytes of V a lane and token
  constexpr int VW = VB / 4;
  constexpr int MT = D / 16;                  // channel tiles of O^T, k steps of S
  constexpr int R = 8 * NT;
  constexpr int IPC = KV8_NW / WPI;           // items of a CTA
  constexpr int CH = D / 8;
  __shared__ alignas(16) __half s_q_all[IPC][R][D];
  __shared__ float s_qs_all[IPC][R];
  __shared__ float4 s_cs_all[IPC][D / 2];
  __shared__ float s_m_all[KV8_NW][R], s_l_all[KV8_NW][R];
  constexpr int STAGE = 2 * KV8_BLOCK * D;    // bytes of a block: keys, values
  extern __shared__ __align__(128) uint8_t s_ring_all[];           // [KV8_NW][ST][STAGE], later [KV8_NW][R][D] floats
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int in_cta = warp / WPI, iw = warp % WPI, it = iw * 32 + lane;        // item of the CTA, warp and thread of the item
  const int x_item = int(blockIdx.x) * IPC + in_cta;
  if (x_item >= a.items_x) return;
  auto& s_q = s_q_all[in_cta];
  auto& s_qs = s_qs_all[in_cta];
  auto& s_cs = s_cs_all[in_cta];
  auto* s_m = s_m_all + in_cta * WPI;
  auto* s_l = s_l_all + in_cta * WPI;
  const uint32_t ring_at = uint32_t(__cvta_generic_to_shared(s_ring_all)) + warp * (ST * STAGE);
  // this lane's results start its warp's part of the ring
  static_assert(R * D * 4 <= ST * STAGE, "a warp's results fit its ring");
  auto s_o = [&](int w, int r) { return reinterpret_cast<float*>(s_ring_all + (in_cta * WPI + w) * (ST * STAGE)) + r * D; };
  const int seq = a.kv_heads == 1 ? x_item : x_item / a.kv_heads, kvh = x_item - seq * a.kv_heads;
  const int group = a.group;
  const int n = a.q_len ? a.q_len[seq] : 1;
  const int r0 = blockIdx.y * 16;
  const int live = min(min(16, a.part_rows), n * group - r0);   // rows of this tile
  const long row0 = a.seq_start ? long(a.seq_start[seq]) : seq;
  const Kv8Keys keys = kv8_keys(a, seq);
  const int len = keys.len, table = keys.table;
  const bool takes_part = kv8_takes_part(a, row0, n, len);
  if ((!takes_part || keys.cut) && it == 0) kv8_report(a.status);
  if (!takes_part || live <= 0) return;
  const int slot = a.slots ? a.slots[seq] : -1;
  const int pos = a.positions ? a.positions[seq] : 0;
  // keys that the tile's last query sees, this share's blocks, this warp's
  auto query_of = [&](int r) { return n == 1 ? 0 : r / group; };          // of row r: a decode step has one
  const int seen = a.causal ? len - (n - 1 - query_of(r0 + live - 1)) : len;
  const int nblk = seen > 0 ? (seen + KV8_BLOCK - 1) / KV8_BLOCK : 0;
  const int b_lo = min(nblk, int(blockIdx.z) * a.share), b_hi = blockIdx.z + 1 == a.splits ? nblk : min(nblk, b_lo + a.share);
  const int w_lo = b_lo + int(long(b_hi - b_lo) * iw / WPI), w_hi = b_lo + int(long(b_hi - b_lo) * (iw + 1) / WPI);
  const int cnt = w_hi - w_lo;
  const int* bt = a.tables + long(table) * a.table_ld + w_lo;
  const bool appends = slot >= 0 && cnt > 0 && w_hi == nblk;    // the warp that reads the last block writes the new token

  using Ring = Kv8Ring<D>;
  // this lane's pieces of a block: piece lane + 32 i, for keys and for values; for 128 channels the pieces of odd i, four rows
  // further, are turned differently
  constexpr int BYTES = KV8_BLOCK * D;
  const uint8_t* const k_from = a.kcodes + long(kvh) * BYTES + lane * 16;
  const uint8_t* const v_from = a.vcodes + long(kvh) * BYTES + lane * 16;
  const uint32_t to_even = ring_at + Ring::at(lane / Ring::PIECES, lane % Ring::PIECES);
  const uint32_t to_odd = ring_at + Ring::at(lane / Ring::PIECES + 32 / Ring::PIECES, lane % Ring::PIECES) - 512;
  const uint32_t page_bytes = uint32_t(a.kv_heads) * BYTES;
  auto load = [&](int at, int p) {              // the block of page p to byte `at` of the ring
    const unsigned long long off = static_cast<unsigned long long>(uint32_t(p)) * page_bytes;
    const uint8_t *kp = k_from + off, *vp = v_from + off;
    kv8_copy16<0, 0>(to_even + at, kp);
    kv8_copy16<BYTES, 0>(to_even + at, vp);
    kv8_copy16<512, 512>(to_odd + at, kp);
    kv8_copy16<BYTES + 512, 512>(to_odd + at, vp);
    if constexpr (D == 128) {
      kv8_copy16<1024, 1024>(to_even + at, kp);
      kv8_copy16<BYTES + 1024, 1024>(to_even + at, vp);
      kv8_copy16<1536, 1536>(to_odd + at, kp);
      kv8_copy16<BYTES + 1536, 1536>(to_odd + at, vp);
    }
  };
  auto commit = [&] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  // pages and scales are looked up for 32 blocks at a time, one a lane: pages two such groups ahead, scales one
  auto page_of = [&](int b) {                   // -1: none
    int p = b < cnt ? bt[b] : -1;
    if (b < cnt && (p < 0 || p >= a.num_blocks)) kv8_report(a.status), p = -1;
    return p;
  };
  auto scale_of = [&](const float* s, int p) { return p >= 0 ? s[long(p) * a.kv_heads + kvh] : 0.f; };
  int page = page_of(lane), page1 = cnt > 32 ? page_of(32 + lane) : -1, page2 = -1;
  float kf = scale_of(a.kscale, page), vf = scale_of(a.vscale, page), kf1 = 0.f, vf1 = 0.f;
  uint32_t gone_of = __ballot_sync(0xffffffffu, page < 0);        // of the 32 blocks at hand
  page = max(page, 0);                          // what is loaded for a block without a page is not used
  constexpr int AHEAD = ST - U;                // blocks on their way, a group of U at a time
  static_assert(ST % U == 0 && AHEAD > 0, "whole groups");
  const int early = appends ? min(cnt - 1, AHEAD) : min(cnt, AHEAD);          // the last block waits for its new token
  const int held = appends && early < AHEAD ? early / U : AHEAD;             // and with it its group
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) {
    if (s < early) load(s * STAGE, __shfl_sync(0xffffffffu, page, s));
    if (s % U == U - 1 && s / U < held) commit();
  }

  // ---- q to shared memory: rotated, scaled to f16
  if (a.positions) {
    for (int j = it; j < D / 2; j += WPI * 32) s_cs[kv8_angle_at<D>(j)] = kv8_cos_sin(turns.t[j], pos);
    kv8_item_sync<WPI>(in_cta);
  }
  for (int r = iw; r < live; r += WPI) {
    const int chunk = lane % CH;
    uint4 h;
    float down;
    {
      const int t = query_of(r0 + r), head = kvh * group + r0 + r - t * group;
      Vec8 x = *reinterpret_cast<const Vec8*>(static_cast<const T*>(a.q) + (row0 + t) * a.ld_q + long(head) * D + chunk * 8);
      if (a.positions) {
        Vec8 oth;
#pragma unroll
        for (int i = 0; i < 4; ++i) oth.w[i] = __shfl_xor_sync(0xffffffffu, x.w[i], CH / 2);
        x = kv8_rotate8<T, CH / 2>(x, oth, chunk < CH / 2, s_cs + chunk % (CH / 2));
      }
      float up = 1.f;
      down = 1.f;
      if constexpr (!std::is_same<T, __half>::value) {
        const uint32_t m = kv8_warp_amax<T>(kv8_absmax(0u, x)) >> 23;           // exponent of the largest
        if (m > 0 && m < 255) {
          const int e = max(int(m) - 127 - 10, -100);                          // largest to [2^10, 2^11)
          up = __uint_as_float(uint32_t(127 - e) << 23);
          down = __uint_as_float(uint32_t(127 + e) << 23);
        }
      }
      float f[8];
      unpack8<T>(x, f);
      h.x = kv8_half2(f[0] * up, f[1] * up), h.y = kv8_half2(f[2] * up, f[3] * up);
      h.z = kv8_half2(f[4] * up, f[5] * up), h.w = kv8_half2(f[6] * up, f[7] * up);
    }
    if (lane < CH) *reinterpret_cast<uint4*>(&s_q[r][chunk * 8]) = h;
    if (lane == 0) s_qs[r] = down * a.scale_log2;
  }
  if (appends) {
    if (slot >= a.num_blocks * KV8_BLOCK) {
      if (lane == 0) kv8_report(a.status);
    } else {
      float ks, vs;
      kv8_append_one<T, D, CODE>(a, row0, slot, kvh, s_cs, ks, vs);
      __syncwarp();
      if (lane == cnt - 1 && page == slot / KV8_BLOCK) kf = ks, vf = vs;
    }
    if (early < AHEAD) {
      load(early * STAGE, __shfl_sync(0xffffffffu, page, early));
      for (int s = held; s < AHEAD / U; ++s) commit();
    }
  }
  if (vf != vf) kf = vf, vf = 0.f;              // seeing the block's keys is seeing its values: NaN through the scores
  kv8_item_sync<WPI>(in_cta);
  // Q fragments: k step j of lane c is bytes 4 (j % 4) .. + 3 of its 16 in chunk j / 4 of 64 channels
  uint32_t qa[MT][2 * NT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int ch = (j / 4) * 64 + c * 16 + (j % 4) * 4;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint2 w = g + 8 * t < live ? *reinterpret_cast<const uint2*>(&s_q[g + 8 * t][ch]) : make_uint2(0u, 0u);
      qa[j][t] = w.x;
      qa[j][NT + t] = w.y;
    }
  }
  float qs[NT][2];                             // of rows 2c and 2c + 1, and 8 t further
  int lim[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = 2 * c + k + 8 * t;
      qs[t][k] = r < live ? s_qs[r] : 0.f;
      lim[t][k] = r < live ? (a.causal ? len - (n - 1 - query_of(r0 + r)) : len) : 0;
    }
  const int first_lim = a.causal ? len - (n - 1 - query_of(r0)) : len;        // the fewest keys of a live row

  float o[MT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t][0] = m[t][1] = -INFINITY, l[t][0] = l[t][1] = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[i][t][k] = 0.f;
  }
  float vref = 0.f;                            // o is in units of vref * 2^-15
  // where this lane reads: keys of tokens token(g) and 8 further, values of c's tokens
  uint32_t k_at[KW], v_at[2];
#pragma unroll
  for (int i = 0; i < KW; ++i) k_at[i] = ring_at + Ring::at(Ring::token(g), i * 4 + c);
  int tok_of[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    tok_of[k] = Ring::token(2 * c + k);
    v_at[k] = ring_at + KV8_BLOCK * D + Ring::at(tok_of[k], g * VB / 16) + (g * VB) % 16;
  }
  for (int b = 0, into = AHEAD * STAGE, from = 0; b < cnt; b += U) {
    if ((b & 31) == 0) {
      if (b > 0) {
        gone_of = __ballot_sync(0xffffffffu, page1 < 0);
        page = max(page1, 0), page1 = page2, kf = kf1, vf = vf1;
        if (vf != vf) kf = vf, vf = 0.f;
      }
      if (cnt > b + 32) {
        kf1 = scale_of(a.kscale, page1), vf1 = scale_of(a.vscale, page1);
        page2 = cnt > b + 64 ? page_of(b + 64 + lane) : -1;
      }
      const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vf)));
      if (top > vref) {
        const float down = vref * kv8_inverse(top);          // 0 the first time
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[i][t][k] *= down;
        vref = top;
      }
      vf *= kv8_inverse(vref) * 32768.f;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD / U - 1) : "memory");
    __syncwarp();                             // blocks b .. have landed, and every lane is done with those before
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int nb = b + AHEAD + u;
      if (nb < cnt) load(into + u * STAGE, max(__shfl_sync(0xffffffffu, ((nb ^ b) & 32) ? page1 : page, nb & 31), 0));
    }
    commit();
    const int place = from;
    into = from, from = from + U * STAGE == ST * STAGE ? 0 : from + U * STAGE;
    // ---- scores: (tokens token(g) and 8 further; rows 2c and 2c + 1)
    float x[U][NT][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t) x[u][t][0] = x[u][t][1] = x[u][t][2] = x[u][t][3] = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        const uint32_t at = k_at[i] + place;
        const uint4 w0 = kv8_shared16<0>(at + u * STAGE), w1 = kv8_shared16<8 * D>(at + u * STAGE);
        const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a0, a1, a2, a3;
          kv8_halves<CODE>(u0[j], a0, a2);
          kv8_halves<CODE>(u1[j], a1, a3);
#pragma unroll
          for (int t = 0; t < NT; ++t) kv8_mma(x[u][t], a0, a1, a2, a3, qa[4 * i + j][t], qa[4 * i + j][NT + t]);
        }
      }
    float vfac[U];
    bool rise = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float kfac = __shfl_sync(0xffffffffu, kf, (b + u) & 31);
      vfac[u] = __shfl_sync(0xffffffffu, vf, (b + u) & 31);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float f0 = kfac * qs[t][0], f1 = kfac * qs[t][1];
        x[u][t][0] *= f0, x[u][t][1] *= f1, x[u][t][2] *= f0, x[u][t][3] *= f1;
      }
    }
    const uint32_t gone = (gone_of >> (b & 31)) & ((1u << U) - 1u);          // blocks without a page, or behind the warp's last
    const int t0 = (w_lo + b) * KV8_BLOCK;
    const bool edge = gone || t0 + U * KV8_BLOCK > first_lim;
    if (edge) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int mine = (gone >> u) & 1 ? 0x7fffffff - 8 : t0 + u * KV8_BLOCK + Ring::token(g);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (mine + 8 * (k >> 1) >= lim[t][k & 1]) x[u][t][k] = -INFINITY;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t) rise |= fmaxf(x[u][t][0], x[u][t][2]) > m[t][0] || fmaxf(x[u][t][1], x[u][t][3]) > m[t][1];
    if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float alpha[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float mx = m[t][k];
#pragma unroll
          for (int u = 0; u < U; ++u) mx = fmaxf(mx, fmaxf(x[u][t][k], x[u][t][k + 2]));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          alpha[k] = mx == -INFINITY ? 1.f : kv8_exp2(m[t][k] - mx);
          l[t][k] *= alpha[k];
          m[t][k] = mx;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) o[i][t][0] *= alpha[0], o[i][t][1] *= alpha[1], o[i][t][2] *= alpha[0], o[i][t][3] *= alpha[1];
      }
    }
    uint32_t p[U][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float m0 = m[t][0] == -INFINITY ? 0.f : m[t][0], m1 = m[t][1] == -INFINITY ? 0.f : m[t][1];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e0 = kv8_exp2(x[u][t][0] - m0), e1 = kv8_exp2(x[u][t][1] - m1), e2 = kv8_exp2(x[u][t][2] - m0), e3 = kv8_exp2(x[u][t][3] - m1);
        l[t][0] += e0 + e2, l[t][1] += e1 + e3;
        p[u][t][0] = kv8_turn(kv8_half2(e0 * vfac[u], e1 * vfac[u]));
        p[u][t][1] = kv8_turn(kv8_half2(e2 * vfac[u], e3 * vfac[u]));
      }
    }
    // ---- values: channel tile i has channels 2 i and 2 i + 1 of the lane's
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t vb[4][VW];                     // c's tokens tok_of[0], tok_of[1], and 8 further
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t src = v_at[k & 1] + place + u * STAGE;
        if constexpr (VW == 2) {
          const uint2 w = k < 2 ? kv8_shared8<0>(src) : kv8_shared8<8 * D>(src);
          vb[k][0] = w.x, vb[k][1] = w.y;
        } else {
          const uint4 w = k < 2 ? kv8_shared16<0>(src) : kv8_shared16<8 * D>(src);
          vb[k][0] = w.x, vb[k][1] = w.y, vb[k][2] = w.z, vb[k][3] = w.w;
        }
      }
      if (edge) {                             // bytes behind the context are no codes
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (((gone >> u) & 1) || t0 + u * KV8_BLOCK + tok_of[k & 1] + 8 * (k >> 1) >= len) {
#pragma unroll
            for (int i = 0; i < VW; ++i) vb[k][i] = 0u;
          }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int w = i / 2;
        const uint32_t sel = (i & 1) ? 0x7362 : 0x5140;
        uint32_t a0, a1, a2, a3;
        kv8_halves<CODE>(__byte_perm(vb[0][w], vb[1][w], sel), a0, a1);
        kv8_halves<CODE>(__byte_perm(vb[2][w], vb[3][w], sel), a2, a3);
#pragma unroll
        for (int t = 0; t < NT; ++t) kv8_mma(o[i][t], a0, a1, a2, a3, p[u][t][0], p[u][t][1]);
      }
    }
  }

  // ---- the warps' results together
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[t][k] += __shfl_xor_sync(0xffffffffu, l[t][k], d);
      if (g == 0) s_m[iw][2 * c + k + 8 * t] = m[t][k], s_l[iw][2 * c + k + 8 * t] = l[t][k];
    }
  const float unit = vref * (1.f / 32768.f);
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();                               // the ring is done with
  // o[i][t][k]: channel g * VB + 2 i + (k >> 1), row 2c + (k & 1) + 8 t
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = 2 * c + k + 8 * t;
      if (r < live) {
        float* dst = s_o(iw, r) + g * VB;
#pragma unroll
        for (int i = 0; i < MT; ++i) *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(o[i][t][k] * unit, o[i][t][k + 2] * unit);
      }
    }
  kv8_item_sync<WPI>(in_cta);
  const long share = (long(blockIdx.y) * a.items_x + x_item) * a.splits + blockIdx.z;
  for (int i = it; i < live * (D / 2); i += WPI * 32) {
    const int r = i / (D / 2), ch = (i % (D / 2)) * 2;
    float mx = s_m[0][r];
#pragma unroll
    for (int w = 1; w < WPI; ++w) mx = fmaxf(mx, s_m[w][r]);
    float s0 = 0.f, s1 = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WPI; ++w) {
      const float f = kv8_weight(s_m[w][r], s_l[w][r], mx);
      const float2 v = *reinterpret_cast<const float2*>(s_o(w, r) + ch);
      if (f != 0.f) s0 += f * v.x, s1 += f * v.y, sum += f * s_l[w][r];
    }
    if (a.splits > 1) {
      float* dst = a.part + (share * a.part_rows + r) * (D + 2);
      *reinterpret_cast<float2*>(dst + ch) = make_float2(s0, s1);
      if (ch == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(mx, sum);
    } else {
      const int t = query_of(r0 + r), h = kvh * group + r0 + r - t * group;
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      T* dst = static_cast<T*>(a.out) + (row0 + t) * a.ld_o + long(h) * D + ch;
      *reinterpret_cast<uint32_t*>(dst) = Pair16<T>::pack(s0 * inv, s1 * inv);
    }
  }
}

// The shares of a row together: one CTA of CW warps for each row of each tile.  A warp weighs 32 shares at a time, one a lane,
// and adds those of its own number; the warps' sums meet in shared memory, in order.  37 shares of 96 rows take 6 us with four
// warps and 11 with one, 3 shares of 3456 rows are faster with one (chunks of 1 to 24 queries: 24.6 against 26.4 us in all).
template <class T, int D, int KV8_CW>
__global__ void __launch_bounds__(KV8_CW * 32) kv8_combine_kernel(Kv8AttnArgs a) {
  constexpr int PER = D / 32;
  __shared__ float s_acc[KV8_CW][D];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tile = int(blockIdx.x / a.part_rows), r = int(blockIdx.x) - tile * a.part_rows;
  const int x = tile % a.items_x, r0 = tile / a.items_x * 16;
  const int seq = x / a.kv_heads, kvh = x - seq * a.kv_heads, group = a.group;
  const int n = a.q_len ? a.q_len[seq] : 1;
  if (r0 + r >= n * group || r >= 16) return;
  const long row0 = a.seq_start ? long(a.seq_start[seq]) : seq;
  if (!kv8_takes_part(a, row0, n, a.q_len ? kv8_keys(a, seq).len : 0)) return;
  const float* src = a.part + (long(tile) * a.splits * a.part_rows + r) * (D + 2);
  const long step = long(a.part_rows) * (D + 2);
  auto share = [&](int z) { return z < a.splits ? *reinterpret_cast<const float2*>(src + z * step + D) : make_float2(-INFINITY, 0.f); };
  float mx = -INFINITY;                                      // the row's maximum and sum, the same in every warp
  for (int z0 = 0; z0 < a.splits; z0 += 32) mx = fmaxf(mx, share(z0 + lane).x);
  mx = warp_max(mx);
  float acc[PER], sum = 0.f;
#pragma unroll
  for (int k = 0; k < PER; ++k) acc[k] = 0.f;
  for (int z0 = 0; z0 < a.splits; z0 += 32) {
    const float2 ml = share(z0 + lane);
    const float w = kv8_weight(ml.x, ml.y, mx);
    sum += w != 0.f ? w * ml.y : 0.f;
    const int here = min(32, a.splits - z0);
#pragma unroll 4
    for (int i = warp; i < here; i += KV8_CW) {
      const float f = __shfl_sync(0xffffffffu, w, i);
      const float* v = src + (z0 + i) * step + lane * PER;
      float part[PER];
#pragma unroll
      for (int k = 0; k < PER; k += 2) {
        const float2 t = *reinterpret_cast<const float2*>(v + k);
        part[k] = t.x, part[k + 1] = t.y;
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) acc[k] += f != 0.f ? f * part[k] : 0.f;
    }
  }
  sum = warp_sum(sum);
#pragma unroll
  for (int k = 0; k < PER; ++k) s_acc[warp][lane * PER + k] = acc[k];
  __syncthreads();
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  for (int i = threadIdx.x; i < D / 2; i += KV8_CW * 32) {
    float v0 = 0.f, v1 = 0.f;
#pragma unroll
    for (int w = 0; w < KV8_CW; ++w) v0 += s_acc[w][2 * i], v1 += s_acc[w][2 * i + 1];
    T* dst = static_cast<T*>(a.out) + (row0 + (n == 1 ? 0 : (r0 + r) / group)) * a.ld_o;
    dst += long(kvh * group + (n == 1 ? r0 + r : (r0 + r) % group)) * D + 2 * i;
    *reinterpret_cast<uint32_t*>(dst) = Pair16<T>::pack(v0 * inv, v1 * inv);
  }
}

}  // namespace ronn

using namespace ronn;

constexpr int KV8_SHARE = 32;
struct Kv8Plan {
  int wpi, splits, share;      // warps of an item, CTAs along a context, cache blocks each of them takes
};

// Warps of an item: two where that gives every SM's schedulers at least two rounds of warps, else four.  256 rows of 64 to 768
// keys, 16 heads of 64, took 72, 65.5 and 72 us with one, two and four; 128 rows of 41 to 577 keys, 20 heads of 128: 72, 65.5 and
// 65.5.  A context is cut into equal shares, whatever its row's length, so that long rows give more CTAs and not longer ones;
// shares are taken for about six CTAs an SM at the longest context, of KV8_SHARE blocks at least (chunks of 1 to 24 queries over
// 200 to 1500 keys: 28.7, 26.4 and 28.6 us with at least 16, 32 and 64).
static Kv8Plan kv8_plan(long tiles, int max_ctx) {
  const int sms = device_sm_count(), nblk = (max_ctx + KV8_BLOCK - 1) / KV8_BLOCK;
  Kv8Plan p{tiles >= 8L * sms ? 2 : 4, 1, nblk > 0 ? nblk : 1};
  const long want = tiles > 0 ? 6L * sms / tiles : 1;
  if (want > 1 && nblk > KV8_SHARE) {
    const long share = (nblk + want - 1) / want;
    p.share = int(share < KV8_SHARE ? KV8_SHARE : share);
    p.splits = (nblk + p.share - 1) / p.share;
    if (p.splits > 1) p.wpi = 4;
  }
  return p;
}

// Bytes of scratch that ronn_kv8_attention needs for these sizes; 0 where one CTA takes a whole tile.
extern "C" long ronn_kv8_attention_scratch(int n_seq, int max_q_len, int max_ctx, int heads, int kv_heads, int head_dim) {
  if (n_seq <= 0 || max_q_len <= 0 || kv_heads <= 0 || heads % kv_heads) return 0;
  const long rows = long(max_q_len) * (heads / kv_heads), tiles = (rows + 15) / 16 * n_seq * kv_heads;
  const int s = kv8_plan(tiles, max_ctx).splits;
  return s <= 1 ? 0 : tiles * s * (rows < 16 ? rows : 16) * (head_dim + 2) * long(sizeof(float));
}

extern "C" int ronn_kv8_attention(const Kv8AttnCall* call, cudaStream_t stream) {
  const auto& [q, kcodes, vcodes, kscale, vscale, tables, bt_row, seq_start, q_len, kv_len, out, slots, positions, turns, scratch, status,
               ld_q, rows, num_blocks, table_ld, ld_o, scratch_bytes, table_rows, max_blocks, n_seq, max_q_len, max_ctx, heads, kv_heads,
               head_dim, causal, dtype, code, k_off, v_off, scale] = *call;
  if (n_seq <= 0 || max_q_len <= 0) return 0;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || (ld_q & 7) || (ld_o & 7) || max_ctx < 0) return -2;
  if ((seq_start == nullptr) != (q_len == nullptr)) return -2;
  if ((slots || positions) && seq_start) return -2;
  if (positions && (!turns || !slots)) return -2;
  if (slots && heads / kv_heads > 16) return -2;               // several tiles would append the same token
  if (head_dim != 64 && head_dim != 128) return -1;
  const long group_rows = long(max_q_len) * (heads / kv_heads), mtiles = (group_rows + 15) / 16, xs = long(n_seq) * kv_heads;
  if (xs > 2147483647L || mtiles > 65535 || xs * mtiles * 16 > 2147483647L) return -2;
  const Kv8Plan plan = kv8_plan(xs * mtiles, max_ctx);
  const int splits = plan.splits, wpi = plan.wpi;
  const int part_rows = int(group_rows < 16 ? group_rows : 16);
  const long need = ronn_kv8_attention_scratch(n_seq, max_q_len, max_ctx, heads, kv_heads, head_dim);
  if (splits > 65535 || (splits > 1 && (scratch == nullptr || scratch_bytes < need))) return -4;
  Kv8Turns tn = {};
  if (positions)
    for (int j = 0; j < head_dim / 2; ++j) tn.t[j] = turns[j];
  Kv8AttnArgs a{q, out, (uint8_t*)kcodes, (uint8_t*)vcodes, kscale, vscale, tables, kv_len, bt_row, seq_start, q_len, slots, positions,
                (float*)scratch, status, ld_q, ld_o, num_blocks, rows, table_ld, heads / kv_heads, int(xs), table_rows, max_blocks, heads, kv_heads, causal,
                plan.splits, plan.share, part_rows, max_q_len, int((long(max_ctx) + KV8_BLOCK - 1) / KV8_BLOCK * KV8_BLOCK), k_off, v_off, scale * 1.4426950408889634f};
  const long per_cta = KV8_NW / wpi;
  const dim3 grid{unsigned((xs + per_cta - 1) / per_cta), unsigned(mtiles), unsigned(splits)};
  const bool small = group_rows <= 8;
#define RONN_KV8T(T, D, C, NT) \
  do { \
    if (wpi == 2) RONN_KV8W(T, D, C, NT, 2); \
    else RONN_KV8W(T, D, C, NT, 4); \
  } while (0)
#define RONN_KV8W(T, D, C, NT, W) \
  do { \
    constexpr int u = D == 64 ? 2 : 1, st = D == 64 ? 6 : 3, smem = KV8_NW * st * 32 * D; \
    auto* kern = kv8_attention_kernel<T, D, C, NT, W, u, st>; \
    static bool seen[MAX_DEVICES] = {false}; \
    if (first_use_on_device(seen) && \
        (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess || \
         cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100) != cudaSuccess)) return -3; \
    launch(kern, grid, dim3(KV8_NW * 32), smem, stream, a, tn); \
  } while (0)
#define RONN_KV8T_(T, D) \
  do { \
    if (code == 0 && small) RONN_KV8T(T, D, 0, 1); \
    else if (code == 0) RONN_KV8T(T, D, 0, 2); \
    else if (code == 1 && small) RONN_KV8T(T, D, 1, 1); \
    else if (code == 1) RONN_KV8T(T, D, 1, 2); \
    else return -1; \
    if (splits > 1) { \
      const long units = xs * mtiles * part_rows; \
      if (splits > 8) launch(kv8_combine_kernel<T, D, 4>, dim3(unsigned(units)), dim3(128), 0, stream, a); \
      else launch(kv8_combine_kernel<T, D, 1>, dim3(unsigned(units)), dim3(32), 0, stream, a); \
    } \
  } while (0)
  if (dtype == 0 && head_dim == 64) RONN_KV8T_(__nv_bfloat16, 64);
  else if (dtype == 0) RONN_KV8T_(__nv_bfloat16, 128);
  else if (dtype == 1 && head_dim == 64) RONN_KV8T_(__half, 64);
  else if (dtype == 1) RONN_KV8T_(__half, 128);
  else return -1;
#undef RONN_KV8T
#undef RONN_KV8W
#undef RONN_KV8T_
  return cudaGetLastError() == cudaSuccess ? 0 : -100;
}
