// Attention of long query chunks over the 8-bit paged KV cache: the contexts' pages become 16-bit values in scratch, in order
// (kv8_expand_kernel), and o = softmax(scale q k^T) v goes over those on the tensor cores (kv8_chunk_kernel).
//
// A CTA takes two tiles of 128 queries that see the same keys: two heads of a group where groups are even, else two
// neighbouring tiles of one head.  Their tensor work alternates, so that one tile's products run while the other is in its softmax:
//   warp 0      TMA: both tiles of Q, then for each 128 keys K and V, two buffers of each.
//   warp 1      tcgen05: S = Q K^T (128 x 128), then O += P V with P taken from tensor memory.  Of its 512 columns S has 128 for
//               each tile, whose first 64 become P (16-bit pairs), and O has D.  S of the next keys waits for that product.
//   warps 2-9   four a tile, one query row a thread: the row of S in registers, maximum, exponentials, sum, P back.  O stays in
//               tensor memory and is rescaled only when a row's maximum has grown by more than 2^8.
// Statistics and O are in 32 bits.  P is rounded to the activations' type, by half a step: both operands of a product have one type,
// and bf16 holds any value of the cache where fp16 would not.  That adds a quarter to the error of bf16 results (0.0021 of the
// result's norm against 0.0017 with P in 32 bits, three chunks of 763 to 1024 queries over 1793 to 5024 keys).
// A step of 128 keys is a chain of softmax (1800 cycles, 1024 of them a warp's exponentials), P V and the next Q K^T (750 each);
// two tiles overlap theirs, so that neither the tensor pipe (46 % of a causal chunk) nor the exponentials are full.  2 x 4096
// queries over 4096 keys, 32 / 8 heads of 128, without a mask: 514 us, 1069 TFLOP/s.  674 us with instructions issued from a lane
// of its own; an issuer that looked for whichever tile could go on was slower still (3 chunks of 763 to 1024 queries: 230 us
// against 191 for taking the tiles in turn).
#include "kv8.cuh"
#include "ptx_sm100.cuh"
#include "tma_desc.cuh"

#include <type_traits>

namespace ronn {

constexpr int KC_THREADS = 320;
constexpr int KC_TILE = 128;             // queries of a tile, keys of a step
constexpr int KC_PAGES = KC_TILE / KV8_BLOCK;

struct Kv8ChunkArgs {
  const uint8_t *kcodes, *vcodes;
  const float *kscale, *vscale;
  const int *tables, *bt_row, *seq_start, *q_len, *kv_len;
  void *k, *v, *out;
  uint32_t* status;
  long table_ld, num_blocks, rows, ld_o;
  int table_rows, max_blocks, nb, padded, kv_heads, heads, max_q, causal, pair_heads, sorted;      // padded: blocks of a (sequence, head) in scratch
  float scale_log2, slack;      // slack: a growth of the maximum by 2^8, in scores before their scale
};
struct Kv8Chunk {
  int row0, n, len, table;
  bool cut;                                                 // keys that no table row lists are left out
};
// A sequence's place and lengths; false where they pass a bound: it is left out, and its rows stay as they are.
__device__ __forceinline__ bool kv8_chunk_of(const Kv8ChunkArgs& a, int seq, Kv8Chunk& s) {
  s.row0 = a.seq_start[seq], s.n = a.q_len[seq], s.table = a.bt_row ? a.bt_row[seq] : seq;
  const int keys = max(a.kv_len[seq], 0);
  const bool listed = s.table >= 0 && s.table < a.table_rows;
  s.len = listed ? min(keys, a.max_blocks * KV8_BLOCK) : 0;
  s.cut = !listed || s.len < keys;
  if (!listed) s.table = 0;
  return s.row0 >= 0 && s.n >= 0 && s.n <= a.max_q && long(s.row0) + s.n <= a.rows && s.len <= a.nb * KV8_BLOCK;
}

// Place `at` in the order of all sequences' items (128 or 256 queries, `unit`), those that see the most keys first: item i of a
// sequence stands at i + (keys in front of its first query) / unit.  For up to 64 sequences, two a lane; by a whole warp.  False
// behind the last.
constexpr int KC_SORTED = 64;
__device__ __forceinline__ bool kv8_chunk_item(const Kv8ChunkArgs& a, int n_seq, int unit, int at, int& seq, int& item) {
  const int lane = threadIdx.x & 31;
  int lo[2], end[2];                                        // [lo, end): the places that a sequence's items have
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    Kv8Chunk s;
    lo[k] = end[k] = 0;
    if (lane + 32 * k < n_seq && kv8_chunk_of(a, lane + 32 * k, s)) {
      const int shift = s.len - s.n;
      lo[k] = shift >= 0 ? shift / unit : -((unit - 1 - shift) / unit);
      end[k] = lo[k] + (s.n + unit - 1) / unit;
    }
  }
  auto from = [&](int v) {                                  // items at place v or above
    return __reduce_add_sync(0xffffffffu, max(0, end[0] - max(lo[0], v)) + max(0, end[1] - max(lo[1], v)));
  };
  int low = __reduce_min_sync(0xffffffffu, min(lo[0], lo[1])), high = __reduce_max_sync(0xffffffffu, max(end[0], end[1]));
  if (at >= from(low)) return false;
  while (high - low > 1) {                                  // the highest place that leaves `at` among its items
    const int mid = low + (high - low) / 2;
    if (from(mid) > at) low = mid;
    else high = mid;
  }
  int rank = at - from(low + 1);
  const uint32_t here0 = __ballot_sync(0xffffffffu, lo[0] <= low && low < end[0]), here1 = __ballot_sync(0xffffffffu, lo[1] <= low && low < end[1]);
  const bool second = rank >= __popc(here0);
  if (second) rank -= __popc(here0);
  uint32_t left = second ? here1 : here0;
  for (; rank > 0; --rank) left &= left - 1;
  const int owner = __ffs(left) - 1;
  seq = owner + (second ? 32 : 0);
  item = low - __shfl_sync(0xffffffffu, second ? lo[1] : lo[0], owner);
  return true;
}

// The pages of the sequences' contexts as values in order: [sequence][kv_head][padded * 16][D] of K and of V, one warp for each
// (block, head, K or V).  A value is exact in bf16; in fp16 it is kept within the type's range.  Slots behind the context, to the
// end of the last 128 keys, and blocks whose page lies outside the cache are zeros, which the attention leaves out.  A poisoned block
// has NaN keys and zero values, so that only those who see it read NaN.
template <class T, int D, int CODE>
__global__ void __launch_bounds__(256) kv8_expand_kernel(Kv8ChunkArgs a) {
  pdl_wait();
  pdl_trigger();
  const int seq = blockIdx.y, lane = threadIdx.x & 31, unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  Kv8Chunk s;
  const bool takes_part = kv8_chunk_of(a, seq, s);
  if ((!takes_part || s.cut) && unit == 0 && lane == 0) kv8_report(a.status);
  if (!takes_part) return;
  const int len = s.len, per = 2 * a.kv_heads, b = unit / per, rest = unit - b * per;
  if (b >= (len + KC_TILE - 1) / KC_TILE * KC_PAGES) return;
  const bool is_v = rest >= a.kv_heads;
  const int h = is_v ? rest - a.kv_heads : rest;
  const bool used = b * KV8_BLOCK < len;
  const int page = used ? a.tables[long(s.table) * a.table_ld + b] : -1;
  const bool there = page >= 0 && page < a.num_blocks;
  if (used && !there && lane == 0) kv8_report(a.status);
  const long src = long(there ? page : 0) * a.kv_heads + h;
  const float ks = there ? a.kscale[src] : 0.f, vs = there ? a.vscale[src] : 0.f;
  const bool poisoned = ks != ks || vs != vs;
  const float sc_all = is_v ? (poisoned ? 0.f : vs) : (poisoned ? __uint_as_float(0x7fc00000u) : ks);
  const uint4* codes = reinterpret_cast<const uint4*>((is_v ? a.vcodes : a.kcodes) + src * (KV8_BLOCK * D));
  T* out = static_cast<T*>(is_v ? a.v : a.k) + ((long(seq) * a.kv_heads + h) * a.padded + b) * (KV8_BLOCK * D);
  constexpr int PASSES = KV8_BLOCK * D / 512;
  constexpr float MOST = std::is_same<T, __half>::value ? 65504.f : 3.3e38f;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int at = (p * 32 + lane) * 16;                    // 16 channels of one token
    const bool live = there && b * KV8_BLOCK + at / D < len;
    uint4 c = codes[p * 32 + lane];
    if (!live) c = make_uint4(0u, 0u, 0u, 0u);
    const float sc = live ? sc_all : 0.f;
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float f[8], g[4];
      kv8_unpack4<CODE>(w[2 * k], g);
      f[0] = g[0] * sc, f[1] = g[1] * sc, f[2] = g[2] * sc, f[3] = g[3] * sc;
      kv8_unpack4<CODE>(w[2 * k + 1], g);
      f[4] = g[0] * sc, f[5] = g[1] * sc, f[6] = g[2] * sc, f[7] = g[3] * sc;
      if (!poisoned) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = fminf(fmaxf(f[j], -MOST), MOST);
      }
      *reinterpret_cast<Vec8*>(out + at + k * 8) = pack8<T>(f);
    }
  }
}

template <int D>
struct KcSmem {
  static constexpr int TILE = KC_TILE * D * 2;              // bytes of a tile of Q, K or V
  static constexpr int BYTES = 6 * TILE;
  // more than half of an SM's, also for D = 64: a CTA takes all of its tensor memory
  static constexpr int DYN = (BYTES + 256 + 1024) > 120 * 1024 ? BYTES + 256 + 1024 : 120 * 1024;
};

__device__ __forceinline__ float kc_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned long long kc_two(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 kc_split(unsigned long long v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ unsigned long long kc_add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long kc_mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float kc_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// One lane of a warp that is together, the same each time.
__device__ __forceinline__ bool kc_elect() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
// Registers to 32 lanes x 16 columns of tensor memory.
__device__ __forceinline__ void kc_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void kc_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] B[smem], A as 16-bit pairs in 32-bit columns.  Issued by one thread.
__device__ __forceinline__ void kc_mma_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Descriptor of V as it is stored, rows of 128 bytes for each key: groups of 8 keys 1024 bytes apart, the second 64 channels
// one tile of such rows further.
__device__ __forceinline__ uint64_t kc_desc_v(uint32_t smem_addr) {
  return uint64_t((smem_addr & 0x3FFFF) >> 4) | uint64_t((KC_TILE * 128) >> 4) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 |
         uint64_t(2) << 61;
}

template <class T, int D>
__global__ void __launch_bounds__(KC_THREADS, 1)
kv8_chunk_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 Kv8ChunkArgs a, uint32_t idesc_s, uint32_t idesc_pv) {
  using L = KcSmem<D>;
  constexpr int ATOMS = D / 64;
  extern __shared__ uint8_t kc_smem[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kc_smem) + 1023) & ~uintptr_t(1023));
  uint8_t *sq = base, *sk = base + 2 * L::TILE, *sv = base + 4 * L::TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::BYTES);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 7;         // two of each but q
  uint64_t *s_full = bars + 9, *p_full = bars + 11, *o_full = bars + 13;                                             // one a tile
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
  volatile uint32_t* abort = tmem_slot + 1;
  const int* volatile* s_pages = reinterpret_cast<const int* volatile*>(bars + 16);                   // the context's pages, and its last block
  volatile int* s_last = reinterpret_cast<volatile int*>(bars + 17);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  // With a causal mask the items differ in their keys: the longest first.  Three sequences of 763 to 1024 queries over 1793 to
  // 5024 keys, 336 CTAs of 9 to 40 steps, take 174 us, and 185 in the order of the grid.
  int seq = blockIdx.y, z = int(gridDim.z) - 1 - int(blockIdx.z);
  if (a.sorted && !kv8_chunk_item(a, a.sorted, a.pair_heads ? KC_TILE : 2 * KC_TILE, blockIdx.y, seq, z)) return;
  Kv8Chunk s;
  if (!kv8_chunk_of(a, seq, s)) return;
  const int head0 = a.pair_heads ? 2 * int(blockIdx.x) : int(blockIdx.x), tile0 = a.pair_heads ? z : 2 * z;
  if (tile0 * KC_TILE >= s.n) return;                       // the same for the whole CTA
  const int kvh = head0 / (a.heads / a.kv_heads), shift = s.len - s.n;
  int steps[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int tile = a.pair_heads ? tile0 : tile0 + u;
    const int seen = a.causal ? min(s.len, min((tile + 1) * KC_TILE, s.n) + shift) : s.len;         // keys of its last query
    steps[u] = tile * KC_TILE < s.n && seen > 0 ? (seen + KC_TILE - 1) / KC_TILE : 0;
  }
  const int all = max(steps[0], steps[1]);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1), mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 4), mbar_init(&o_full[i], 1);
    }
    *abort = 0;
    *s_pages = a.tables + long(s.table) * a.table_ld, *s_last = (s.len - 1) / KV8_BLOCK;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;                         // S of tile u at 128 u, O at 256 + 128 u
  // Only now may the next kernel start: one that takes tensor memory and then waits for this grid would keep a CTA that has
  // none yet waiting for good.
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0 && all > 0) {
      mbar_expect_tx(q_full, 2 * L::TILE);
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int at = 0; at < ATOMS; ++at)
          tma_load_2d(sq + u * L::TILE + at * (KC_TILE * 128), &map_q, q_full, (a.pair_heads ? head0 + u : head0) * D + at * 64,
                      s.row0 + (a.pair_heads ? tile0 : tile0 + u) * KC_TILE);
      const int row = (seq * a.kv_heads + kvh) * a.padded * KV8_BLOCK;
      for (int j = 0; j < all; ++j) {
        const int b = j & 1;
        const uint32_t parity = ((j >> 1) & 1) ^ 1;
        if (!mbar_wait(&k_empty[b], parity, abort, a.status, STATUS_WAIT_SLOT)) break;
        mbar_expect_tx(&k_full[b], L::TILE);
#pragma unroll
        for (int at = 0; at < ATOMS; ++at)
          tma_load_2d(sk + b * L::TILE + at * (KC_TILE * 128), &map_k, &k_full[b], at * 64, row + j * KC_TILE);
        if (!mbar_wait(&v_empty[b], parity, abort, a.status, STATUS_WAIT_SLOT)) break;
        mbar_expect_tx(&v_full[b], L::TILE);
#pragma unroll
        for (int at = 0; at < ATOMS; ++at)
          tma_load_2d(sv + b * L::TILE + at * (KC_TILE * 128), &map_v, &v_full[b], at * 64, row + j * KC_TILE);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // The warp stays together and one lane of it issues, so that descriptors are uniform: 30 cycles less an instruction.
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, a.status, code)) != 0;
    };
    auto last = [&](int j) { return j < steps[1] ? 1 : 0; };             // the last tile that takes part in step j
    const uint64_t dq = umma_desc_k128(smem_u32(sq)), dk = umma_desc_k128(smem_u32(sk)), dv = kc_desc_v(smem_u32(sv));
    auto scores = [&](int u, int j) -> bool {
      if (!wait(&k_full[j & 1], (j >> 1) & 1, STATUS_WAIT_TMA)) return false;
      tc_fence_after_sync();
      const uint64_t q = dq + uint64_t(u) * (L::TILE >> 4), k0 = dk + uint64_t(j & 1) * (L::TILE >> 4);
      if (kc_elect()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t off = (uint32_t(k / 4) * (KC_TILE * 128) + uint32_t(k % 4) * 32) >> 4;
          umma_f16(tmem + u * 128, q + off, k0 + off, idesc_s, k != 0);
        }
        umma_commit(&s_full[u]);
        if (u == last(j)) umma_commit(&k_empty[j & 1]);
      }
      __syncwarp();
      return true;
    };
    bool ok = all > 0 && wait(q_full, 0, STATUS_WAIT_TMA);
    for (int u = 0; u < 2; ++u)
      if (ok && steps[u] > 0) ok = scores(u, 0);
    for (int j = 0; j < all && ok; ++j) {
      for (int u = 0; u < 2 && ok; ++u) {
        if (j >= steps[u]) continue;
        ok = wait(&p_full[u], j & 1, STATUS_WAIT_EPI) && wait(&v_full[j & 1], (j >> 1) & 1, STATUS_WAIT_TMA);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t v0 = dv + uint64_t(j & 1) * (L::TILE >> 4);
        if (kc_elect()) {
#pragma unroll
          for (int k = 0; k < KC_TILE / 16; ++k)
            kc_mma_tmem(tmem + 256 + u * 128, tmem + u * 128 + k * 8, v0 + uint64_t(k * 16 * 128 >> 4), idesc_pv, j > 0 || k > 0);
          umma_commit(&o_full[u]);
          if (u == last(j)) umma_commit(&v_empty[j & 1]);
        }
        __syncwarp();
        if (j + 1 < steps[u]) ok = wait(&o_full[u], j & 1, STATUS_WAIT_ACCUM) && scores(u, j + 1);          // S takes P's place once the product has read it
      }
    }
    __syncwarp();
  } else {
    // A wait that gives up does not leave the loop: the warp runs every step, and `ok` gates the stores.
    const int u = (warp - 2) >> 2, quarter = warp & 3;
    const int mine = u == 0 ? steps[0] : steps[1];
    const int head = a.pair_heads ? head0 + u : head0, tile = a.pair_heads ? tile0 : tile0 + u;
    const int qi = tile * KC_TILE + quarter * 32 + lane;                 // this thread's query
    int limit = a.causal ? max(min(s.len, qi + shift + 1), 0) : s.len;   // the keys it sees
    const uint32_t at = tmem + (uint32_t(quarter * 32) << 16), s_at = at + u * 128, o_at = at + 256 + u * 128;
    const unsigned long long scale2 = kc_two(a.scale_log2, a.scale_log2);
    float m = -INFINITY;                                    // of the scores before their scale, which is positive
    unsigned long long l2[2] = {0ull, 0ull};
    bool ok = true;
    // Pages outside the cache: looked for while the first scores are on their way, and again in each step only where there are some:
    // `limit` is then its complement, below 0 in every lane, and all steps count as edges.  Anything more that lives through the
    // loop is spilled and took 1.4 % of a chunk, as did looking at one page after the other.
    auto absent = [&](int page) { return uint32_t(page) >= uint32_t(a.num_blocks); };
    bool lacks = false;
    {
      const int* const pages = *s_pages;
      const int last = *s_last;
#pragma unroll 8
      for (int b = lane; b < mine * KC_PAGES; b += 32) lacks |= absent(pages[min(b, last)]);
    }
    if (__any_sync(0xffffffffu, lacks)) limit = ~limit;
    for (int j = 0; j < mine; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[u], j & 1, abort, a.status, STATUS_WAIT_ACCUM)) && ok;
      tc_fence_after_sync();
      uint32_t x[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_at + c * 32, x[c]);
      tmem_ld_wait();
      const int key0 = j * KC_TILE;
      if (!__all_sync(0xffffffffu, key0 + KC_TILE <= limit)) {
        const int seen = (limit < 0 ? ~limit : limit) - key0;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i >= seen) x[c][i] = 0xff800000u;               // -inf
        if (limit < 0) {                                    // keys that are not there are left out
          const uint32_t gone = __ballot_sync(0xffffffffu, lane < KC_PAGES && absent((*s_pages)[min(j * KC_PAGES + lane, *s_last)]));
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (gone >> (2 * c + i / KV8_BLOCK) & 1) x[c][i] = 0xff800000u;
        }
      }
      float top[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        top[c] = fmaxf(__uint_as_float(x[c][0]), __uint_as_float(x[c][1]));
#pragma unroll
        for (int i = 2; i < 32; i += 2) top[c] = kc_max3(top[c], __uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1]));
      }
      const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      const float m_new = mx > m + a.slack ? mx : m;
      const float back = m_new == -INFINITY ? 0.f : -m_new;              // without a key all exponents are -inf, from 0 too
      if (__any_sync(0xffffffffu, m_new != m)) {
        const float alpha = kc_exp2((m + back) * a.scale_log2);
        if (j > 0) {                                        // the products so far are complete: S of this step came after them
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld_32x16(o_at + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            kc_tmem_st16(o_at + c, o);
          }
        }
        const float2 e = kc_split(l2[0]), f = kc_split(l2[1]);
        l2[0] = kc_two(e.x * alpha, e.y * alpha), l2[1] = kc_two(f.x * alpha, f.y * alpha);
        m = m_new;
      }
      // The difference first, then the scale: x scale - m scale in one operation leaves over what rounding m scale lost, which passes
      // an exponent's range where scores are far out (from 2^31 on; fp16 queries and keys can reach 2^35).  One operation more for two
      // scores: 514 us against 510 at 2 x 4096 queries with heads of 128, 260 against 252 with 16 heads of 64.
      const unsigned long long minus = kc_two(back, back);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 d = kc_split(kc_mul2(kc_add2(kc_two(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1])), minus), scale2));
          const float p0 = kc_exp2(d.x), p1 = kc_exp2(d.y);
          l2[i & 1] = kc_add2(l2[i & 1], kc_two(p0, p1));
          p[i] = Pair16<T>::pack(p0, p1);
        }
        kc_tmem_st16(s_at + c * 16, p);
      }
      kc_tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[u]);
    }
    float inv = 0.f;
    if (mine > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(&o_full[u], (mine - 1) & 1, abort, a.status, STATUS_WAIT_ACCUM)) && ok;
      tc_fence_after_sync();
      const float2 e = kc_split(kc_add2(l2[0], l2[1]));
      const float l = e.x + e.y;
      inv = l != 0.f ? 1.f / l : 0.f;
    }
    T* row = static_cast<T*>(a.out) + long(s.row0 + qi) * a.ld_o + long(head) * D;
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      uint32_t o[32];
      if (mine > 0) {
        tmem_ld_32x32(o_at + c, o);
        tmem_ld_wait();
      }
      if (qi < s.n && ok) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          float f[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = mine > 0 ? __uint_as_float(o[i + k]) * inv : 0.f;
          *reinterpret_cast<Vec8*>(row + c + i) = pack8<T>(f);
        }
      }
    }
  }
  if (*abort) {
    // copies and products still on their way land before shared and tensor memory go
    const long long t0 = clock64();
    while (clock64() - t0 < 400000ll) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

template <class T, int D>
static int kv8_chunk_tiles(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Kv8ChunkArgs& a, int n_seq, cudaStream_t stream) {
  using L = KcSmem<D>;
  auto* kern = kv8_chunk_kernel<T, D>;
  static bool seen[MAX_DEVICES] = {false};
  if (first_use_on_device(seen) && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::DYN) != cudaSuccess) return -3;
  const int tiles = (a.max_q + KC_TILE - 1) / KC_TILE;
  const int items = a.pair_heads ? tiles : (tiles + 1) / 2;
  const dim3 grid{unsigned(a.pair_heads ? a.heads / 2 : a.heads), unsigned(a.sorted ? n_seq * items : n_seq), unsigned(a.sorted ? 1 : items)};
  const uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
  const uint32_t idesc_pv = umma_idesc(KC_TILE, D, fmt, 1u) | (1u << 16);          // V's channels are contiguous, its keys are not
  launch(kern, grid, dim3(KC_THREADS), size_t(L::DYN), stream, mq, mk, mv, a, umma_idesc(KC_TILE, KC_TILE, fmt, 1u), idesc_pv);
  return cudaGetLastError() == cudaSuccess ? 0 : -100;
}

}  // namespace ronn

using namespace ronn;

static int kv8_chunk_padded(int max_kv) { return int((long(max_kv) + KC_TILE - 1) / KC_TILE * KC_PAGES); }
// Sequences that ronn_kv8_chunk_attention expands at a time: what fits 256 MiB, one at least.
static int kv8_chunk_group(int n_seq, int max_kv, int kv_heads, int head_dim) {
  const long per = 2L * kv8_chunk_padded(max_kv) * kv_heads * KV8_BLOCK * head_dim * 2;
  const long g = per > 0 ? (256L << 20) / per : n_seq;
  return int(g < 1 ? 1 : g > n_seq ? n_seq : g > 32768 ? 32768 : g);
}
extern "C" long ronn_kv8_chunk_scratch(int n_seq, int max_kv, int kv_heads, int head_dim) {
  if (n_seq <= 0 || max_kv <= 0) return 0;
  const long g = kv8_chunk_group(n_seq, max_kv, kv_heads, head_dim);
  return 2 * g * kv8_chunk_padded(max_kv) * kv_heads * KV8_BLOCK * head_dim * 2;
}

// Whether chunks of these sizes are faster that way (1) or straight from the codes (0), by what both cost in microseconds.
// Expanded: 128 keys after the other for each pair of tiles, 1.5 us a step (1.8 for heads of 128) while the SMs have no more than
// two thirds of a CTA each, and the values, 2 (1.6) TB/s.  Direct: 0.5 ns (0.9) for each 16 query rows and 16 keys.  Over 240
// sizes (1 to 16 sequences, contexts of 300 to 4000, 16 to 512 queries, four head layouts) the rule costs 0.5 % (1.0 %) against
// the faster form of each on average and 13 % (25 %, 4 us) at worst; 16 x 128 queries over 4000 keys, 32 / 8 heads of 128: 225 us
// against 711 direct; 4 x 32 queries over 4000 keys, 16 heads of 64: 78 against 37.
extern "C" int ronn_kv8_chunk_form(int n_seq, int max_q, int max_ctx, int heads, int kv_heads, int head_dim) {
  if (n_seq <= 0 || max_q <= 0 || max_ctx <= 0 || kv_heads <= 0) return 0;
  const bool wide = head_dim > 64, pairs = heads / kv_heads % 2 == 0;
  const double ctas = double(n_seq) * (pairs ? heads / 2 * ((max_q + 127L) / 128) : heads * ((max_q + 255L) / 256)) / device_sm_count() * 1.5;
  const double expanded = (wide ? 15 : 13) + (max_ctx + 127L) / 128 * (wide ? 1.8 : 1.53) * (ctas > 1 ? ctas : 1) +
                          double(n_seq) * max_ctx * kv_heads * head_dim * 2 * (wide ? 6.1e-7 : 5.1e-7);
  const double tiles = double(n_seq) * kv_heads * ((long(max_q) * (heads / kv_heads) + 15) / 16);
  return expanded < (wide ? 19.5 : 15) + tiles * ((max_ctx + 15L) / 16) * (wide ? 0.9e-3 : 0.49e-3);
}

// The same call as ronn_kv8_attention with queries grouped by sequence, no append, and scale > 0.
extern "C" int ronn_kv8_chunk_attention(const Kv8AttnCall* c, cudaStream_t stream) {
  if (c->n_seq <= 0 || c->max_q_len <= 0) return 0;
  if (c->heads <= 0 || c->kv_heads <= 0 || c->heads % c->kv_heads || (c->ld_q & 7) || (c->ld_o & 7) || !c->seq_start || !c->q_len || c->slots ||
      c->positions || !(c->scale > 0.f) || c->max_ctx <= 0 || c->max_blocks <= 0 || c->max_blocks > (1 << 26))
    return -2;
  if (c->head_dim != 64 && c->head_dim != 128) return -1;
  if (c->max_q_len > 65535 * KC_TILE || c->rows > 2147483647L) return -2;
  const int nb = (c->max_ctx + KV8_BLOCK - 1) / KV8_BLOCK, padded = kv8_chunk_padded(c->max_ctx);
  const int group = kv8_chunk_group(c->n_seq, c->max_ctx, c->kv_heads, c->head_dim);
  const long elems = long(group) * padded * c->kv_heads * KV8_BLOCK * c->head_dim, units = 2L * padded * c->kv_heads;
  if (!c->scratch || c->scratch_bytes < 4 * elems) return -4;
  const long rows = elems / c->head_dim;
  if (rows > 2147483647L || (units + 7) / 8 > 2147483647L) return -2;
  uint16_t *k = static_cast<uint16_t*>(c->scratch), *v = k + elems;
  const float scale_log2 = c->scale * 1.4426950408889634f;
  CUtensorMap mq, mk, mv;
  int rc = make_tmap_2d(&mq, c->q, uint64_t(c->rows), uint64_t(c->heads) * c->head_dim, uint64_t(c->ld_q), KC_TILE, 64, 2);
  if (rc) return rc - 20;
  rc = make_tmap_2d(&mk, k, uint64_t(rows), uint64_t(c->head_dim), uint64_t(c->head_dim), KC_TILE, 64, 2);
  if (rc) return rc - 30;
  rc = make_tmap_2d(&mv, v, uint64_t(rows), uint64_t(c->head_dim), uint64_t(c->head_dim), KC_TILE, 64, 2);
  if (rc) return rc - 40;
  for (int s0 = 0; s0 < c->n_seq; s0 += group) {
    const int n = c->n_seq - s0 < group ? c->n_seq - s0 : group;
    // without bt_row the sequence is its own table row
    Kv8ChunkArgs a{static_cast<const uint8_t*>(c->kcodes), static_cast<const uint8_t*>(c->vcodes), c->kscale, c->vscale,
                   c->bt_row ? c->tables : c->tables + s0 * c->table_ld, c->bt_row ? c->bt_row + s0 : nullptr, c->seq_start + s0, c->q_len + s0,
                   c->kv_len + s0, k, v, c->out, c->status, c->table_ld, c->num_blocks, c->rows, c->ld_o,
                   c->bt_row ? c->table_rows : c->table_rows - s0, c->max_blocks, nb, padded, c->kv_heads, c->heads, c->max_q_len, c->causal,
                   c->heads / c->kv_heads % 2 == 0, c->causal && n <= KC_SORTED && long(n) * ((c->max_q_len + KC_TILE - 1) / KC_TILE) <= 65535 ? n : 0,
                   scale_log2, fminf(8.f / scale_log2, 1e30f)};
    const dim3 grid{unsigned((units + 7) / 8), unsigned(n), 1u};
#define RONN_KV8X(T, D, C) \
  do { \
    launch(kv8_expand_kernel<T, D, C>, grid, dim3(256), 0, stream, a); \
    if (cudaGetLastError() != cudaSuccess) return -100; \
    rc = kv8_chunk_tiles<T, D>(mq, mk, mv, a, n, stream); \
  } while (0)
#define RONN_KV8X_(T) \
  do { \
    if (c->head_dim == 64 && c->code == 0) RONN_KV8X(T, 64, 0); \
    else if (c->head_dim == 64 && c->code == 1) RONN_KV8X(T, 64, 1); \
    else if (c->code == 0) RONN_KV8X(T, 128, 0); \
    else if (c->code == 1) RONN_KV8X(T, 128, 1); \
    else return -1; \
  } while (0)
    if (c->dtype == 0) RONN_KV8X_(__nv_bfloat16);
    else if (c->dtype == 1) RONN_KV8X_(__half);
    else return -1;
#undef RONN_KV8X
#undef RONN_KV8X_
    if (rc) return rc;
  }
  return 0;
}
