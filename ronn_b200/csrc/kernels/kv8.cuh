// 8-bit paged KV cache: codes, scales and their conversions.
//
// Codes of K and of V: [num_blocks, kv_heads, 16, head_dim] bytes, int8 (-127 .. 127) or e4m3; one fp32 scale for each
// (block, kv_head), K and V apart, always a power of two:
//     s = 2^e,  e the least integer >= -100 with amax * 2^-e <= 127 (int8) or 448 (e4m3);   value = code * s.
// A power of two costs at most one bit of int8 (none of e4m3, which carries its own exponent) and makes every step but the
// one rounding exact: x / s, code * s, and the change of scale when a larger token joins a block.  The codes are then a
// function of the block's tokens and not of the order of arithmetic, the same whether a prompt came in one call or many,
// as long as the scale does not change under a token (then that token is rounded once more, to the coarser step).
//   * Writing slot 0 begins a block: its scale starts from that call's tokens alone.  Otherwise s = max(old, new), and the
//     codes of the slots below the call's first one are rounded again when s grew.  Slots above its last one keep their bytes.
//   * A token with a value that is not finite makes the scale NaN until the block begins again: a query that sees any token
//     of that block and head reads NaN.  Codes themselves are always finite, so masked slots never spread one.
#pragma once
#include "common.cuh"

namespace ronn {

constexpr int KV8_BLOCK = 16;
constexpr uint32_t STATUS_KV8_PAGE = 0x5801;    // a block table, slot or table-row index outside the cache: not accessed

enum Kv8Code { KV8_INT8 = 0, KV8_E4M3 = 1 };

__device__ __forceinline__ void kv8_report(uint32_t* status) {
  if (status) atomicCAS(status, 0u, STATUS_KV8_PAGE);
}

// Scale of a block whose largest magnitude has the bits `amax` (of a finite float >= 0).
template <int CODE>
__device__ __forceinline__ float kv8_least_scale(uint32_t amax) {
  // 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8: one more when the significand is above the limit's
  const int top = CODE == KV8_INT8 ? 6 : 8;
  const uint32_t frac = CODE == KV8_INT8 ? 0x7E0000u : 0x600000u;
  int e = int(amax >> 23) - 127 - top + ((amax & 0x7fffffu) > frac ? 1 : 0);
  e = max(e, -100);
  return __uint_as_float(uint32_t(e + 127) << 23);
}

// 1 / s, exact for a scale made above; 0 for 0 (a block never written) and for NaN.  Scales that another quantiser left in a
// cache need not be powers of two.
__device__ __forceinline__ float kv8_inverse(float s) { return s > 0.f && s < 8.5e37f ? __frcp_rn(s) : 0.f; }

// Four values (already divided by the scale) to four codes, round to nearest even.
template <int CODE>
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d) {
  if constexpr (CODE == KV8_INT8) {
    // |x| <= 127: adding 1.5 * 2^23 rounds to an integer that stands in the low bits
    const float magic = 12582912.f;
    const uint32_t x = __float_as_uint(a + magic), y = __float_as_uint(b + magic);
    const uint32_t z = __float_as_uint(c + magic), w = __float_as_uint(d + magic);
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
  } else {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return uint32_t(lo) | (uint32_t(hi) << 16);
  }
}

// Two codes in the low 16 bits of w -> two floats.
template <int CODE>
__device__ __forceinline__ float2 kv8_unpack2(uint32_t w) {
  if constexpr (CODE == KV8_INT8) {
    return make_float2(float(int(int8_t(w & 0xff))), float(int(int8_t((w >> 8) & 0xff))));
  } else {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(w)));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
  }
}
template <int CODE>
__device__ __forceinline__ void kv8_unpack4(uint32_t w, float (&f)[4]) {
  const float2 a = kv8_unpack2<CODE>(w), b = kv8_unpack2<CODE>(w >> 16);
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}

// Rotary embedding: the angle of pair j at position p is p * base^(-2j/d).  `turns[j]` is base^(-2j/d) / (2 pi) as the nearest
// 64-bit binary fraction, so p * turns[j] modulo 2^64 is the angle's fraction of a turn, right to 2^-45 at p = 2^20 (a 32-bit
// angle is off by 0.004 rad at p = 65536).  Sine and cosine are taken in 64 bits and the rotated value is formed to 44, then
// rounded to 32 bits and to the activations' type, as a 64-bit tensor is converted: but for values within some 2^-40 of a
// rounding border the result is the one that 64-bit arithmetic gives.
constexpr int KV8_MAX_HALF = 64;
struct Kv8Turns {
  unsigned long long t[KV8_MAX_HALF];
};
// Cosine and sine, each as a float and the float that it leaves over: 48 bits.
__device__ __forceinline__ float4 kv8_cos_sin(unsigned long long turn, int pos) {
  const unsigned long long f = turn * (unsigned long long)(long long)pos;
  double s, c;
  sincospi(double((long long)f) * 1.0842021724855044e-19, &s, &c);       // 2^-63: half turns in [-1, 1)
  const float ch = __double2float_rn(c), sh = __double2float_rn(s);
  return make_float4(ch, __double2float_rn(c - double(ch)), sh, __double2float_rn(s - double(sh)));
}

// a c + b s rounded to 32 bits as if its products and their sum were exact to 2^-44: the products of 16-bit values with the
// upper parts are a float and the float left over, so is their sum.  (Conversions to and from 64 bits cost four times this:
// they run at a quarter of a multiplication's rate at best.)
__device__ __forceinline__ float kv8_turned(float a, float ch, float cl, float b, float sh, float sl) {
  const float p = __fmul_rn(a, ch), pe = __fmaf_rn(a, ch, -p), q = __fmul_rn(b, sh), qe = __fmaf_rn(b, sh, -q);
  const float r = __fadd_rn(p, q), z = __fadd_rn(r, -p), e = __fadd_rn(__fadd_rn(p, -__fadd_rn(r, -z)), __fadd_rn(q, -z));
  return __fadd_rn(r, __fadd_rn(e, __fadd_rn(__fadd_rn(pe, qe), __fmaf_rn(a, cl, __fmul_rn(b, sl)))));
}

// Eight rotated values: `own` the chunk, `oth` the chunk half a head away, `low` whether own is in the first half.  cs: the
// pair's angle, the eight of a chunk STEP apart, so that the lanes of a token read neighbouring places.
template <class T, int STEP>
__device__ __forceinline__ Vec8 kv8_rotate8(const Vec8& own, const Vec8& oth, bool low, const float4* cs) {
  float a[8], b[8];
  unpack8<T>(own, a);
  unpack8<T>(oth, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 k = cs[i * STEP];
    a[i] = kv8_turned(a[i], k.x, k.y, b[i], low ? -k.z : k.z, low ? -k.w : k.w);
  }
  return pack8<T>(a);
}
// Place of pair j of a head of D channels in a table of angles.
template <int D>
__device__ __forceinline__ int kv8_angle_at(int j) { return (j % 8) * (D / 16) + j / 8; }

// Largest magnitude of eight 16-bit values as 16-bit patterns, two running maxima in one word.
__device__ __forceinline__ uint32_t kv8_absmax(uint32_t m, const Vec8& v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __vmaxu2(m, v.w[i] & 0x7fff7fffu);
  return m;
}
// ... over the warp, as the bits of a float; values that are not finite give 0x7f800000 or more.
template <class T>
__device__ __forceinline__ uint32_t kv8_warp_amax(uint32_t m) {
  m = max(m & 0xffffu, m >> 16);
  m = __reduce_max_sync(0xffffffffu, m);
  float lo, hi;
  Pair16<T>::unpack(m, lo, hi);
  return __float_as_uint(lo);
}

// Scale of a block after tokens whose largest magnitude has the bits `m` (not finite: 0x7f800000 or more) have joined one of
// scale `old`: the larger of the two; NaN stays.
template <int CODE>
__device__ __forceinline__ float kv8_new_scale(uint32_t m, float old) {
  const float nan = __uint_as_float(0x7fc00000u);
  if (m >= 0x7f800000u) return nan;
  const float s = kv8_least_scale<CODE>(m);
  return old <= s ? s : old;
}
// The first `words` words of codes to a coarser step, by `lanes` lanes.
template <int CODE>
__device__ __forceinline__ void kv8_round_again(uint8_t* codes, int words, int lane, int lanes, float old, float inv) {
  const float again = inv == 0.f ? 0.f : old * inv;           // a power of two below 1, or 0
  uint32_t* c32 = reinterpret_cast<uint32_t*>(codes);
  for (int i = lane; i < words; i += lanes) {
    float f[4];
    kv8_unpack4<CODE>(c32[i], f);
    c32[i] = kv8_pack4<CODE>(f[0] * again, f[1] * again, f[2] * again, f[3] * again);
  }
}
template <class T, int CODE>
__device__ __forceinline__ uint2 kv8_pack8(const Vec8& x, float inv) {
  float f[8];
  unpack8<T>(x, f);
  if (inv == 0.f) return make_uint2(0u, 0u);                  // also for what is not finite
  return make_uint2(kv8_pack4<CODE>(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                    kv8_pack4<CODE>(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
}

// One warp puts n tokens of one (block, head) into slots off .. off + n - 1: the block's new scale, older codes rounded again
// where it grew, the tokens' codes.  x[p] holds 8 channels (from chunk * 8 on) of token p * (tokens a pass) + sub.  Tokens from
// n on are zeros.
template <class T, int D, int CODE, int PASSES>
__device__ __forceinline__ void kv8_store_run(const Vec8* x, int chunk, int sub, int n, int off, float* scale, uint8_t* codes) {
  constexpr int TPW = 256 / D;
  const int lane = threadIdx.x & 31;
  const float old = off > 0 ? *scale : 0.f;
  uint32_t m = 0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) m = kv8_absmax(m, x[p]);
  const float s = kv8_new_scale<CODE>(kv8_warp_amax<T>(m), old), inv = kv8_inverse(s);       // all lanes have read the old scale
  if (off > 0 && s != old) kv8_round_again<CODE>(codes, off * (D / 4), lane, 32, old, inv);
  if (lane == 0 && (off == 0 || s != old)) *scale = s;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int t = p * TPW + sub;
    if (t < n) *reinterpret_cast<uint2*>(codes + (off + t) * D + chunk * 8) = kv8_pack8<T, CODE>(x[p], inv);
  }
}

// One call.  q, out: 16-bit [rows, ld]; dtype 0 bf16, 1 fp16; code 0 int8, 1 e4m3; head_dim 64 or 128.  max_q_len bounds
// q_len, max_ctx sizes the launch.  slots (one query per sequence): the new K and V of row s are at columns k_off and v_off of
// q's row and join the cache at slots[s]; positions and turns (kv8_append): rotary embedding of q and the new k.
struct Kv8AttnCall {
  const void* q;
  void *kcodes, *vcodes;
  float *kscale, *vscale;
  const int *tables, *bt_row, *seq_start, *q_len, *kv_len;
  void* out;
  const int *slots, *positions;
  const unsigned long long* turns;
  void* scratch;
  uint32_t* status;
  long ld_q, rows, num_blocks, table_ld, ld_o, scratch_bytes;
  int table_rows, max_blocks, n_seq, max_q_len, max_ctx, heads, kv_heads, head_dim, causal, dtype, code, k_off, v_off;
  float scale;
};

}  // namespace ronn
