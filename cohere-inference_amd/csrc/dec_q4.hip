// The decoding step over caches held in 4 bits (q4.h's form; 72 bytes a 128-vector where the int8 caches take 132), for
// gfx950. No counterpart in the reference, whose caches are bf16 or int8 (kernels/csrc/decoder_ops.cu, dec_attn.cuh).
//
//   dec_attention_q4   softmax(q k^T scale) v of one new token per row over its slot's cache, `ratio` query heads to a key
//                      head; self-attention first appends the new key and value at position n and attends to them as
//                      computed
//   dec_scatter_kv_q4  keys and values of packed rows into their slots
//   dec_gather_kv_q4   cached keys and values of (slot, position) pairs as bf16 rows
#include "cohere_hip.h"
#include "common.h"
#include "q4.h"

#include <string>

namespace {

using namespace cohere_q4;

// ---- attention of one new token per row ---------------------------------------------------------------------------
// scores and weights are in powers of two: s = q.k scale log2(e), p = 2^(s - m).
//
// A workgroup takes one row, one key head, G of its query heads and one part of the keys; a wave takes 64 keys at a
// time. Both products run on v_mfma_i32_16x16x64_i8, so that the codes need no conversion (three instructions turn a
// word's eight codes into bytes 16 c) and the sums are exact:
//   q k^T: A holds the queries as 31-bit fixed point (a power of two of each group of 32 dimensions) in four digits of 8
//   bits, row 4 g + t digit t of group g (one head fills the 16 rows), with zeros outside the row's group; B is 16 keys,
//   lane (key, group g) holding the group's 16 bytes as loaded. Values down to 2^-23 of the group's largest are exact so;
//   where there are smaller ones, they are held 2^23 larger in digits of their own, multiplied by the same keys (LEVELS of
//   these hold any bf16 values: the queries are exact). Lane (key, g) of the result holds group g's sums, whose maximum it
//   loaded with the codes, and the four groups meet by lane swaps that leave key l of the wave's 64 in lane l.
//   softmax: one key a lane; the running maximum is the wave's.
//   p v: A holds p m_g (m_g the value's maximum in group g) as 31-bit fixed point of the wave's largest, in four digits of
//   8 bits, row 4 g + t digit t of group g (one head fills the 16 rows), B the codes of 64 keys and 16 dimensions 8 n + j
//   (n the lane's column, j the product): lane (n, i) loads one word (8 dimensions) of each of the keys 16 i .. 16 i + 15,
//   and byte permutations put four keys' bytes into one word. Of the result, lanes of row group g = n / 4 hold what
//   counts. A p m_g is so off by half a unit, 2^-31 of the largest of the 64: more than 2^-11 of itself where it is below
//   2^-20 of that, and it may be all that an output has, where the larger ones' codes are zero. If there are such weights,
//   and an output that the units could change by 2^-11 (too_small), what the units left of all 64 is added in units of its
//   own largest, and so on.
// Of fewer than 32 bits before the result, which keeps 8, are thus only these units: an output is off by at most 2^-11 of
// sum p |v| for them.
// Why the matrix cores for one query: with v_dot8_i32_i4 and one fma a value the vector ALU took 110 instructions a wave
// and 16 keys (340 at 4 heads), and every lane's outputs had to meet at the end; here about 330 a wave and 64 keys (1065).
// 64 rows x 8 heads, 0 .. 447 keys: 8.2 us, launch and load latency; 16 rows x 8 x 4 heads, 2 .. 32 K keys, 8 parts: 110
// us, the vector ALU (issuing 57 % of the time); one row x 8 heads, 64 K keys: 14.4 us, 5.2 TB/s from the Infinity Cache.
// The codes, maxima and keys past the end come back as zeros from the buffer loads' own bounds check, so that nothing is
// read of them and they weigh nothing.
struct Q4Args {
  const int32_t* active;
  const uint16_t* q;  // (rows, ldq): H query heads, then (self) KV keys, KV values of the new token
  int64_t ldq;
  uint8_t *k4, *v4;   // (S, KV, T, 64)
  uint16_t *ks, *vs;  // (S, KV, T, 4)
  const int32_t* n;   // per slot; self: position of the new token, cross: keys
  int S, H, KV, T, ratio, chunks, rows_y;  // rows_y: the rows are the grid's second dimension
  float scale;
  uint16_t* out;  // (rows, H * 128)
  float* part;    // (rows, H, splits, 130) when split: outputs, maximum (power of two), sum
};

constexpr float LOG2E = 1.4426950408889634f;
constexpr float CODE = 112.f;   // a product with bytes 16 c is this many times one with c / 7
constexpr float UNIT = 0.875f;  // outputs are summed in this unit, CODE / 128: no larger than they are
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
DEVI float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
DEVI float nan_f() { return __uint_as_float(0x7fc00000u); }

// of a and b: a summed over the two halves of the wave in its lower half, b in the upper; of two such, each summed over
// the rows of 16 lanes of a half. Of a, b, c, d, quarter_sum(half_sum(a, c), half_sum(b, d)) has the sum of the i-th over
// the four rows in row i.
DEVI float half_sum(float a, float b) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
DEVI float quarter_sum(float a, float b) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
// the same with the maxima of four as unsigned numbers
DEVI uint32_t rows_max(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const auto x = __builtin_amdgcn_permlane32_swap(a, c, false, false);
  const auto y = __builtin_amdgcn_permlane32_swap(b, d, false, false);
  const auto z = __builtin_amdgcn_permlane16_swap(max_u(x[0], x[1]), max_u(y[0], y[1]), false, false);
  return max_u(z[0], z[1]);
}

// four words as the words of their bytes 0, 1, 2, 3
DEVI void bytes4(const uint32_t (&v)[4], uint32_t (&x)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(v[1], v[0], 0x05010400u), b = __builtin_amdgcn_perm(v[1], v[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(v[3], v[2], 0x05010400u), d = __builtin_amdgcn_perm(v[3], v[2], 0x07030602u);
  x[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  x[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  x[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  x[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// a score below every finite one that counts, so that differences of scores need no care for two infinities
constexpr float BOTTOM = -3e38f, RISE = 8.f;

// the largest value of the wave, in every lane: as unsigned numbers of the same order, whose maxima take the lane moves
// as operands
DEVI float wave_top(float v) {
  const uint32_t b = __float_as_uint(v);
  uint32_t u = b ^ (uint32_t)((int)b >> 31 | (int)0x80000000u);
  u = max_u(u, dpp_u<DPP_XOR1>(u));
  u = max_u(u, dpp_u<DPP_XOR2>(u));
  u = max_u(u, dpp_u<DPP_ROR4>(u));
  u = max_u(u, dpp_u<DPP_ROR8>(u));
  const auto x = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = max_u(x[0], x[1]);
  const auto y = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  u = max_u(y[0], y[1]);
  return __uint_as_float((int)u < 0 ? u & 0x7fffffffu : ~u);
}

constexpr uint32_t HI4 = 0xf0f0f0f0u;
DEVI int even4(uint32_t w) { return (int)((w << 4) & HI4); }  // the low nibbles as bytes 16 c
DEVI int odd4(uint32_t w) { return (int)(w & HI4); }

// the lane's number, what follows from which is computed where it is used: a few instructions, where a register held
// through the loop for each of a dozen addresses would be spilled
DEVI int lane_here() {
  int v = lane_id();
  asm volatile("" : "+v"(v));
  return v;
}

// whether one of the wave's outputs is smaller than err times the largest weight y (as bits, by groups as weights_to's)
DEVI bool too_small(const float (&acc)[8], uint32_t y, float err) {
  const float c = __uint_as_float(y) * err;
  bool r = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) r |= fabsf(acc[j]) < c;
  const int lane = lane_here();
  return __any(r && lane >> 4 == (lane & 15) >> 2);
}

// B of the second product: of a lane's words of 16 keys the words x of the bytes 0 .. 3 of four keys each, and of those
// the codes of dimension 8 n + j
DEVI void words_of(const uint32_t (&vr)[16], uint32_t (&x)[4][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v[4] = {vr[4 * i], vr[4 * i + 1], vr[4 * i + 2], vr[4 * i + 3]};
    bytes4(v, x[i]);
  }
}
DEVI v4i values_b(const uint32_t (&x)[4][4], int j) {
  const int b = j >> 1;
  return j & 1 ? v4i{odd4(x[0][b]), odd4(x[1][b]), odd4(x[2][b]), odd4(x[3][b])}
               : v4i{even4(x[0][b]), even4(x[1][b]), even4(x[2][b]), even4(x[3][b])};
}

// nothing made of x before this is used after it
DEVI void keep_apart(uint32_t (&x)[4][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(x[i][0]), "+v"(x[i][1]), "+v"(x[i][2]), "+v"(x[i][3]));
}

constexpr int ROW8 = 80;  // 16 rows' b128 reads meet no bank twice, and every write has the lane's one address
// A of the second product, 16 rows (group and digit) of 64 keys' bytes in LDS: w, a key a lane and a weight for each group,
// in units of 2^-k, 2^-7-k in inv; what the units leave of them in w. Returns the wave's largest magnitude of each group
// in row i of lanes group i's, as bits (a NaN's are larger than any number's).
template <bool WRITE>
DEVI uint32_t weights_to(float (&w)[NG], uint8_t* sp8, float& inv) {
  const int lane = lane_here();
  uint32_t a[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) a[i] = __float_as_uint(w[i]) & 0x7fffffffu;
  uint32_t y = rows_max(a[0], a[1], a[2], a[3]);
  y = max_u(y, dpp_u<DPP_XOR1>(y));
  y = max_u(y, dpp_u<DPP_XOR2>(y));
  y = max_u(y, dpp_u<DPP_ROR4>(y));
  y = max_u(y, dpp_u<DPP_ROR8>(y));
  // times 2^k at most 0x7f7f7f7f, four digits of 127: k from the exponent of the next power of two but 0.4 % (0x10200 of a
  // mantissa); 2^-7-k, for sums in UNITs, is not below fp32's smallest number
  const int k = min(157 - (int)((y + 0x10200u) >> 23), 142);
  inv = y < 0x7f800000u ? ldexpf(1.f, -7 - k) : nan_f();
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int ki = __builtin_amdgcn_readlane(k, 16 * i);
    const float f = rintf(ldexpf(w[i], ki));
    w[i] -= ldexpf(f, -ki);  // exact
    if constexpr (WRITE) {
      const uint32_t t = ((uint32_t)(int)f + 0x80808080u) ^ 0x80808080u;
#pragma unroll
      for (int b = 0; b < 4; ++b) sp8[(4 * i + b) * ROW8 + lane] = (uint8_t)(t >> (24 - 8 * b));
    }
  }
  return y;
}
// whether one of this lane's weights, not 0, is below 2^-20 of the largest y: its units left it fewer than 10 bits
DEVI bool coarse(const float (&w)[NG], uint32_t y) {
  const uint32_t c = y > (20u << 23) ? y - (20u << 23) : 1u;
  bool r = false;
#pragma unroll
  for (int i = 0; i < NG; ++i)
    r |= __float_as_uint(w[i]) - 1u < (uint32_t)__builtin_amdgcn_readlane((int)c, 16 * i) - 1u;
  return r;
}
DEVI void weights_of(float e, v2u vm, float (&w)[NG]) {
  w[0] = e * __uint_as_float(vm.x << 16);
  w[1] = e * __uint_as_float(vm.x & 0xffff0000u);
  w[2] = e * __uint_as_float(vm.y << 16);
  w[3] = e * __uint_as_float(vm.y & 0xffff0000u);
}
DEVI v4i weights_a(const uint8_t* sp8) {
  const int lane = lane_here(), col = lane & 15, rowg = lane >> 4;
  return *reinterpret_cast<const v4i*>(&sp8[col * ROW8 + (rowg << 4)]);
}

// the sum of four digits' sums, each of the last two at most 2^28 with the digit above it
DEVI float digits4(const v4i& d) {
  return __builtin_fmaf((float)(d[0] * 256 + d[1]), 65536.f, (float)(d[2] * 256 + d[3]));
}

// what sums of query digits times codes are to be multiplied by, scale 2^unit, in two parts: sums times 2^up and the scale
// stay within fp32's range for queries of any magnitude
struct DigitScale {
  float scale;
  int up, unit;
};
DEVI DigitScale digit_scale(float scale, int unit) {
  const int up = max(-100, min(unit, 60));
  return {ldexpf(scale, unit - up), up, unit};
}

// a wave's outputs, 8 dimensions in each lane that has them, behind each other in LDS
template <int G, int PARTS>
DEVI void outputs_to(float (&so)[G][PARTS][HD], int wave, const float (&acc)[G][8]) {
  const int lane = lane_here(), col = lane & 15;
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (lane >> 4 == col >> 2) {
      float* dst = &so[g][wave][col * 8];
      *reinterpret_cast<float4*>(dst) = make_float4(acc[g][0], acc[g][1], acc[g][2], acc[g][3]);
      *reinterpret_cast<float4*>(dst + 4) = make_float4(acc[g][4], acc[g][5], acc[g][6], acc[g][7]);
    }
}

// Registers: four waves a SIMD (at 4 heads 3 waves give 138 us where 4 give 110: 16 rows of up to 32768 keys, 8 x 4
// heads).
template <bool SELF, int G, int W>
__global__ void __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(4)))
dec_attention_q4_kernel(const Q4Args p) {
  constexpr int PARTS = W + (SELF ? 1 : 0);  // partial results, the new token's last
  // the queries' digits [level][head][group][high .. low][32], behind each head's 32 zeros
  constexpr int QHEAD = HD * 4 + 32, LEVELS = 12;
  __shared__ __attribute__((aligned(16))) uint8_t sq[LEVELS][G][QHEAD];
  __shared__ DigitScale sqs[G][NG];
  __shared__ int slevels[W];
  __shared__ __attribute__((aligned(16))) uint8_t sp8[W][G < 2 ? 1 : 2][16 * ROW8];
  __shared__ __attribute__((aligned(16))) float so[G][PARTS][HD];
  __shared__ float sm[G][PARTS], sl[G][PARTS];
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), col = lane & 15, rowg = lane >> 4;
  const int r = p.rows_y ? blockIdx.y : blockIdx.x, hc = p.rows_y ? blockIdx.x : blockIdx.y;
  const int kvh = hc / p.chunks, ch = hc % p.chunks, sp = blockIdx.z, nsp = gridDim.z;
  // the chunk's query heads h0 .. h0 + G - 1, the last one repeated where the chunk has fewer
  const int h0 = kvh * p.ratio + ch * G, hlast = kvh * p.ratio + p.ratio - 1;
  int s = p.active[r];
  const bool slot_ok = (unsigned)s < (unsigned)p.S;
  s = slot_ok ? s : 0;
  int n = p.n[s];
  const bool row_ok = slot_ok && n >= 0 && (!SELF || n < p.T);
  n = row_ok ? (n < p.T ? n : p.T) : 0;
  const int64_t vec0 = ((int64_t)s * p.KV + kvh) * p.T;
  const int chunk = (n + nsp - 1) / nsp, start = min(n, sp * chunk), end = min(n, start + chunk);
  const auto krs = __builtin_amdgcn_make_buffer_rsrc(p.k4 + vec0 * VB, 0, end * VB, 0x00027000);
  const auto vrs = __builtin_amdgcn_make_buffer_rsrc(p.v4 + vec0 * VB, 0, end * VB, 0x00027000);
  const auto kms = __builtin_amdgcn_make_buffer_rsrc(p.ks + vec0 * NG, 0, end * (2 * NG), 0x00027000);
  const auto vms = __builtin_amdgcn_make_buffer_rsrc(p.vs + vec0 * NG, 0, end * (2 * NG), 0x00027000);

  v4u kr[4];
  uint32_t km[4], vr[16];
  v2u vm;
  auto load_k = [&](int j0) {
    const int ln = lane_here(), col = ln & 15, rowg = ln >> 4;
    uint32_t off = (uint32_t)(j0 + col) * VB + rowg * 16, moff = (uint32_t)(j0 + col) * (2 * NG) + rowg * 2;
    asm volatile("" : "+v"(off), "+v"(moff));  // one register with constant offsets, not one for each load
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      kr[t] = __builtin_amdgcn_raw_buffer_load_b128(krs, off + t * 16 * VB, 0, 0);
      km[t] = __builtin_amdgcn_raw_buffer_load_b16(kms, moff + t * 16 * (2 * NG), 0, 0);
    }
  };
  auto load_v = [&](int j0) {
    const int lane = lane_here(), col = lane & 15, rowg = lane >> 4;
    uint32_t off = (uint32_t)(j0 + rowg * 16) * VB + col * 4;
    asm volatile("" : "+v"(off));
    vm = __builtin_amdgcn_raw_buffer_load_b64(vms, (uint32_t)(j0 + lane) * (2 * NG), 0, 0);
#pragma unroll
    for (int i = 0; i < 16; ++i) vr[i] = __builtin_amdgcn_raw_buffer_load_b32(vrs, off + i * VB, 0, 0);
  };
  int j0 = start + wave * 64;
  load_k(j0);
  load_v(j0);

  // the queries' digits, a dimension per thread; byte 8 (d / 8) + 4 (d % 2) + d % 8 / 2 of its group, as the codes'
  static_assert(G * HD <= W * 64, "a thread per dimension");
  int deep = 0, level = 0, qe = 0;  // of the wave, of the dimension; the dimension's exponent
  float qv = 0.f;
  const auto digits_to = [&](int lv) {
    const int g = tid >> 7, d = tid & (HD - 1), at = d & 31;
    const int v = lv == level ? (int)ldexpf(qv, qe + 23 * lv) : 0;
    const uint32_t t = ((uint32_t)v + 0x80808080u) ^ 0x80808080u;
    uint8_t* dst = &sq[lv][g][(d >> 5) * 128 + (at >> 3) * 8 + (at & 1) * 4 + ((at & 7) >> 1)];
#pragma unroll
    for (int b = 0; b < 4; ++b) dst[b * 32] = (uint8_t)(t >> (24 - 8 * b));
    if (d < 8) *reinterpret_cast<uint32_t*>(&sq[lv][g][HD * 4 + d * 4]) = 0;
  };
  if (tid < G * HD) {
    const int g = tid >> 7, d = tid & (HD - 1);
    const uint32_t bits = (uint32_t)p.q[(int64_t)r * p.ldq + min(h0 + g, hlast) * HD + d] << 16;
    uint32_t mb = bits & 0x7fffffffu;
    mb = max_u(mb, dpp_u<DPP_XOR1>(mb));
    mb = max_u(mb, dpp_u<DPP_XOR2>(mb));
    mb = max_u(mb, dpp_u<DPP_ROR4>(mb));
    mb = max_u(mb, dpp_u<DPP_ROR8>(mb));
    const auto sw = __builtin_amdgcn_permlane16_swap(mb, mb, false, false);
    mb = max_u(sw[0], sw[1]);
    const bool ok = mb < 0x7f800000u;
    const float m = __uint_as_float(ok ? mb : 0u);
    // m 2^qe from 2^30 - 2^22 to 0x7f7f7f7f, four digits of 127 (m has 8 bits: only 255 2^23 would be above). A value, of 8
    // bits too, is whole in level 0 if it is at least 2^7 there, else in the first level where it is, below 2^30
    qe = 31 - __builtin_amdgcn_frexp_expf(m);
    qe -= ldexpf(m, qe) > 2139062143.f;
    qv = ok ? __uint_as_float(bits) : 0.f;
    const int ex = qv != 0.f ? __builtin_amdgcn_frexp_expf(qv) + qe : 8;
    level = ex < 8 ? (30 - ex) / 23 : 0;
    while (__any(level > deep)) ++deep;
    digits_to(0);
    if ((d & 31) == 0) sqs[g][d >> 5] = digit_scale(ok ? p.scale * (LOG2E / CODE) : nan_f(), -qe);
  }
  if (lane == 0) slevels[wave] = deep;
  if constexpr (SELF) {
    const bool fresh = row_ok && sp == 0;
    const uint16_t* row = p.q + (int64_t)r * p.ldq;
    const uint16_t* knew = row + (p.H + kvh) * HD;
    // the new token: a partial result of its own per head, as computed
    for (int g = wave; g < G; g += W) {
      float dot = 0.f;
      if (fresh) {
        const uint32_t a = *reinterpret_cast<const uint32_t*>(row + min(h0 + g, hlast) * HD + lane * 2);
        const uint32_t b = *reinterpret_cast<const uint32_t*>(knew + lane * 2);
        const uint32_t c = *reinterpret_cast<const uint32_t*>(knew + p.KV * HD + lane * 2);
        dot = __uint_as_float(a << 16) * __uint_as_float(b << 16);
        dot = __builtin_fmaf(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u), dot);
        dot = wave_sum64(dot) * (p.scale * LOG2E);
        so[g][W][lane * 2] = UNIT * __uint_as_float(c << 16);
        so[g][W][lane * 2 + 1] = UNIT * __uint_as_float(c & 0xffff0000u);
      }
      if (lane == 0) {
        sm[g][W] = fresh ? dot : -INFINITY;
        sl[g][W] = fresh ? (dot == dot ? 1.f : dot) : 0.f;  // maxima pass over a NaN score, the sum keeps it
      }
    }
    // and into the cache: 16 lanes a vector, 8 values each
    if (fresh && ch == 0 && wave == W - 1 && lane < 32) {
      float x[8];
      const uint32_t mx = quad_max_u(unpack8(*reinterpret_cast<const uint4*>(knew + rowg * p.KV * HD + col * 8), x));
      const Group g = group_of(mx);
      const int64_t vec = vec0 + n;
      *reinterpret_cast<uint32_t*>((rowg ? p.v4 : p.k4) + vec * VB + col * 4) = pack8(g, x);
      if ((col & 3) == 0) (rowg ? p.vs : p.ks)[vec * NG + (col >> 2)] = g.store;
    }
  }
  __syncthreads();
  int levels = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) levels = max(levels, slevels[w]);
  levels = __builtin_amdgcn_readfirstlane(levels) + 1;
  if (__builtin_expect(levels > 1, 0)) {
    if (tid < G * HD)
#pragma unroll 1
      for (int lv = 1; lv < levels; ++lv) digits_to(lv);
    __syncthreads();
  }
  // A of the first product: row 4 g + t is digit t of group g, its halves 16 bytes apart, zeros outside the group
  const int a_at = (col >> 2) == rowg ? rowg * 128 + (col & 3) * 32 : HD * 4;

  float m[G], l[G], acc[G][8];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = BOTTOM;
    l[g] = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[g][k] = 0.f;
  }
  // The units of 64 weights are off by 2^-25 of the largest in all, the passes' by so much each: 2^-11 of an output that is
  // not below err times the largest
  const float err = ldexpf((float)((end - start + W * 64 - 1) / (W * 64)), -14);
  while (j0 < end) {
    // scores of key j0 + lane
    float sc[G];
    {
      // two heads at a time, whose operands fit the registers of four waves a SIMD
#pragma unroll
      for (int g0 = 0; g0 < G; g0 += 2) {
#pragma unroll
        for (int h = 0; h < 2 && g0 + h < G; ++h) sc[g0 + h] = 0.f;
        int lv = 0;
        do {
          v4i aq[2][2];
          float x[2], z[2];
          DigitScale qs[2];
#pragma unroll
          for (int h = 0; h < 2 && g0 + h < G; ++h) {
            aq[h][0] = *reinterpret_cast<const v4i*>(&sq[lv][g0 + h][a_at]);
            aq[h][1] = *reinterpret_cast<const v4i*>(&sq[lv][g0 + h][a_at + 16]);
            qs[h] = sqs[g0 + h][rowg];
            if (__builtin_expect(lv > 0, 0)) qs[h] = digit_scale(p.scale * (LOG2E / CODE), qs[h].unit - 23 * lv);
          }
          // tiles of 16 keys in the order 0, 2, 1, 3: what two of them give meets at once
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = i == 1 ? 2 : i == 2 ? 1 : i;
            asm volatile("" : "+v"(kr[t]));  // its bytes are made here, not kept for the next heads or level
            const v4i b0 = {even4(kr[t].x), odd4(kr[t].x), even4(kr[t].y), odd4(kr[t].y)};
            const v4i b1 = {even4(kr[t].z), odd4(kr[t].z), even4(kr[t].w), odd4(kr[t].w)};
            const float mk = __uint_as_float(km[t] << 16);
#pragma unroll
            for (int h = 0; h < 2 && g0 + h < G; ++h) {
              v4i d = __builtin_amdgcn_mfma_i32_16x16x64_i8(aq[h][0], b0, v4i{0, 0, 0, 0}, 0, 0, 0);
              d = __builtin_amdgcn_mfma_i32_16x16x64_i8(aq[h][1], b1, d, 0, 0, 0);
              const float v = ldexpf(digits4(d), qs[h].up) * (qs[h].scale * mk);
              if (i == 0 || i == 2) x[h] = v;
              else if (i == 1) z[h] = half_sum(x[h], v);
              else sc[g0 + h] += quarter_sum(z[h], half_sum(x[h], v));
            }
          }
        } while (++lv < levels);
      }
    }
    const bool live = j0 + lane < end;
    const int jn = j0 + W * 64;
    load_k(jn);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float sg = live ? sc[g] : -INFINITY;
      // the base of the weights is set RISE above the highest score, and moves only when a score passes it: rarely after
      // the first keys, and otherwise one comparison. The weights are at most 1
      if (__any(sg > m[g])) {
        const float mn = lane_value(wave_top(sg) + RISE, 0), a = exp2_hw(m[g] - mn);
        l[g] *= a;
        m[g] = mn;
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[g][k] *= a;
      }
      sc[g] = exp2_hw(sg - m[g]);
      l[g] += sc[g];
    }
    uint32_t x[4][4];
    words_of(vr, x);
    // p m_g in fixed point into A's rows, and the products; two heads at a time, whose operands fit the registers of four
    // waves a SIMD
#pragma unroll
    for (int g0 = 0; g0 < G; g0 += 2) {
      float inv[2];
      uint32_t top[2];
      bool rest[2];
      keep_apart(x);
#pragma unroll
      for (int h = 0; h < 2 && g0 + h < G; ++h) {
        float w[NG], left[NG];
        weights_of(sc[g0 + h], vm, w);
#pragma unroll
        for (int i = 0; i < NG; ++i) left[i] = w[i];
        top[h] = weights_to<true>(left, sp8[wave][h], inv[h]);
        rest[h] = coarse(w, top[h]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own writes, read back by its other lanes
      v4i ap[2];
#pragma unroll
      for (int h = 0; h < 2 && g0 + h < G; ++h) ap[h] = weights_a(sp8[wave][h]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const v4i bv = values_b(x, j);
#pragma unroll
        for (int h = 0; h < 2 && g0 + h < G; ++h)
          acc[g0 + h][j] = __builtin_fmaf(
              digits4(__builtin_amdgcn_mfma_i32_16x16x64_i8(ap[h], bv, v4i{0, 0, 0, 0}, 0, 0, 0)), inv[h], acc[g0 + h][j]);
      }
#pragma unroll
      for (int h = 0; h < 2 && g0 + h < G; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(acc[g0 + h][j]));  // here, not sunk behind the next branch
      asm volatile("" ::: "memory");  // the next weights are written after these are read
#pragma unroll
      for (int h = 0; h < 2 && g0 + h < G; ++h) {
        if (__builtin_expect(!__any(rest[h]) || !too_small(acc[g0 + h], top[h], err), 1)) continue;
        // what the units left, in units of its own largest
        float w[NG], left[NG];
        asm volatile("" : "+v"(sc[g0 + h]), "+v"(vm));
        weights_of(sc[g0 + h], vm, w);
#pragma unroll
        for (int i = 0; i < NG; ++i) left[i] = w[i];
        float unit;
        uint32_t y = weights_to<false>(left, sp8[wave][h], unit);
        do {
          keep_apart(x);
          y = weights_to<true>(left, sp8[wave][h], unit);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          const v4i a = weights_a(sp8[wave][h]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const v4i d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, values_b(x, j), v4i{0, 0, 0, 0}, 0, 0, 0);
            acc[g0 + h][j] = __builtin_fmaf(digits4(d), unit, acc[g0 + h][j]);
            asm volatile("" : "+v"(acc[g0 + h][j]));
          }
          asm volatile("" ::: "memory");
        } while (__any(coarse(w, y)) && too_small(acc[g0 + h], y, err));
      }
    }
    load_v(jn);  // here, not before the products: the words would live beside the bytes (16 registers)
    j0 = jn;
  }

  outputs_to(so, wave, acc);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float L = wave_sum64(l[g]);
    if (lane == 0) {
      sm[g][wave] = m[g];
      sl[g][wave] = L;
    }
  }
  __syncthreads();
  for (int i = tid; i < G * HD; i += W * 64) {
    const int g = i >> 7, d = i & (HD - 1);
    if (ch * G + g >= p.ratio) continue;
    float M = BOTTOM, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < PARTS; ++w) M = fmaxf(M, sm[g][w]);
#pragma unroll
    for (int w = 0; w < PARTS; ++w) {
      const float f = exp2_hw(sm[g][w] - M);
      L = __builtin_fmaf(f, sl[g][w], L);
      // the new token's outputs are unwritten where it does not count
      if (f != 0.f) O = __builtin_fmaf(f, so[g][w][d], O);
    }
    const int64_t head = (int64_t)r * p.H + h0 + g;
    if (nsp == 1) {
      p.out[head * HD + d] = f2bf(L == 0.f ? 0.f : O / (UNIT * L));
    } else {
      float* part = p.part + (head * nsp + sp) * (HD + 2);
      part[d] = O;
      if (d == 0) {
        part[HD] = M;
        part[HD + 1] = L;
      }
    }
  }
}

// The parts of a (row, head): every wave finds the maximum, the parts' weights (lane s part s's) and the sum; CG groups of
// 128 threads sum N parts each, all their loads in flight at once (a loop over the parts with its loads one after the
// other took 30 us for 64 parts, this 4.5). Up to 4 parts: one group, no meeting in LDS (64 rows x 16 heads in 2 parts: 1.5
// us less than with 512 threads a head).
template <int CG, int N>
__global__ void __launch_bounds__(CG * HD) dec_combine_q4_kernel(const float* __restrict__ part, int nsp, uint16_t* out) {
  const int64_t head = blockIdx.x;
  const int tid = threadIdx.x, lane = lane_id(), d = tid & (HD - 1), grp = wave_id() >> 1;
  const float* base = part + head * nsp * (HD + 2);
  const float* mine = base + min(lane, nsp - 1) * (HD + 2) + HD;
  const float ms = mine[0], ls = mine[1];
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = base[min(grp + CG * i, nsp - 1) * (HD + 2) + d];  // parts past the last weigh nothing
  const float mp = lane < nsp ? ms : -INFINITY, M = wave_max64(mp), w = exp2_hw(mp - M);
  const float L = wave_sum64(lane < nsp ? w * ls : 0.f);
  float o = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float f = lane_value(w, grp + CG * i);
    o = grp + CG * i < nsp ? __builtin_fmaf(f, v[i], o) : o;
  }
  if constexpr (CG == 1) {
    out[head * HD + d] = f2bf(L == 0.f ? 0.f : o / (UNIT * L));
  } else {
    __shared__ float so[CG][HD];
    so[grp][d] = o;
    __syncthreads();
    if (tid < HD) {
      float O = 0.f;
#pragma unroll
      for (int g = 0; g < CG; ++g) O += so[g][d];
      out[head * HD + d] = f2bf(L == 0.f ? 0.f : O / (UNIT * L));
    }
  }
}

// ---- filling and reading back -----------------------------------------------------------------------------------------
// kv (rows, L * 2 * KV * 128): per layer KV keys then KV values; row i is position frame_of[i] of slot slot_of[i];
// caches (L, S, KV, T). 16 lanes per vector, 8 values (one word of codes) each; a quad of lanes holds a group. A
// workgroup takes 16 vectors of a row, in ROWS rows (fewer vectors to a row: more rows), so that a lane has ROWS loads in
// flight and finds its vector's place once. Bound by the memory: 3000 rows x 8 layers x 8 heads (126 MB) 23.3 us to fill,
// 22.4 to read back, 5.4 TB/s.
struct KvArgs {
  uint16_t* kv;
  const int32_t *slot_of, *frame_of;
  uint8_t *k4, *v4;
  uint16_t *ks, *vs;
  int64_t ldkv;
  int rows, S, H, T, vecs, blocks, side;  // vectors a row, workgroups a row, rows side by side in a workgroup
};

// a lane's place: its vector of a row and its rows row, row + side, .. A lane without a place (or a row) looks at the
// last one and writes nothing: a load that only some lanes make is a branch, and the loads behind it would wait.
struct KvPlace {
  int d8, kvi, row;
  int64_t col, head;  // head: the vector's (layer, slot 0, head) as a number of heads; slots are H heads apart
  bool in;
};
template <int ROWS>
DEVI KvPlace kv_place(const KvArgs& p) {
  const int rb = blockIdx.x / p.blocks, vslot = threadIdx.x >> 4;
  int v = (blockIdx.x - rb * p.blocks) * 16 + vslot, at = 0;
  if (p.side > 1) {
    at = vslot / p.vecs;
    v = vslot - at * p.vecs;
  }
  KvPlace k;
  k.in = v < p.vecs && at < p.side;
  v = min(v, p.vecs - 1);
  k.d8 = threadIdx.x & 15;
  k.row = rb * (ROWS * p.side) + at;
  const int lk = v / p.H, l = lk >> 1;
  k.kvi = lk & 1;
  k.col = (int64_t)v * HD + k.d8 * 8;
  k.head = (int64_t)l * p.S * p.H + (v - lk * p.H);
  return k;
}

// row i of a lane: its number, whether it is the lane's, and its vector in the caches (-1: none)
struct KvRow {
  int r;
  bool live;
  int64_t vec;
};
DEVI KvRow kv_row(const KvArgs& p, const KvPlace& k, int i) {
  KvRow w;
  w.r = k.row + i * p.side;
  w.live = k.in && w.r < p.rows;
  w.r = min(w.r, p.rows - 1);
  const int s = p.slot_of[w.r], t = p.frame_of[w.r];
  w.vec = (unsigned)s < (unsigned)p.S && (unsigned)t < (unsigned)p.T ? (k.head + (int64_t)s * p.H) * p.T + t : -1;
  return w;
}

template <int ROWS>
__global__ void __launch_bounds__(256) dec_scatter_kv_q4_kernel(const KvArgs p) {
  const KvPlace k = kv_place<ROWS>(p);
  uint4 u[ROWS];
  KvRow w[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    w[i] = kv_row(p, k, i);
    u[i] = *reinterpret_cast<const uint4*>(p.kv + (int64_t)w[i].r * p.ldkv + k.col);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    float x[8];
    const Group g = group_of(quad_max_u(unpack8(u[i], x)));
    const uint32_t c = pack8(g, x);
    if (!w[i].live || w[i].vec < 0) continue;
    *reinterpret_cast<uint32_t*>((k.kvi ? p.v4 : p.k4) + w[i].vec * VB + k.d8 * 4) = c;
    if ((k.d8 & 3) == 0) (k.kvi ? p.vs : p.ks)[w[i].vec * NG + (k.d8 >> 2)] = g.store;
  }
}

template <int ROWS>
__global__ void __launch_bounds__(256) dec_gather_kv_q4_kernel(const KvArgs p) {
  const KvPlace k = kv_place<ROWS>(p);
  const uint8_t* codes = k.kvi ? p.v4 : p.k4;
  const uint16_t* maxima = k.kvi ? p.vs : p.ks;
  KvRow w[ROWS];
  uint32_t c[ROWS], m[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    w[i] = kv_row(p, k, i);
    const int64_t vec = w[i].vec < 0 ? 0 : w[i].vec;
    c[i] = *reinterpret_cast<const uint32_t*>(codes + vec * VB + k.d8 * 4);
    m[i] = maxima[vec * NG + (k.d8 >> 2)];
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const Step st = step_of(__uint_as_float(w[i].vec < 0 ? 0u : m[i] << 16));
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = w[i].vec < 0 ? 0.f : held(code(c[i], j), st);
    if (w[i].live)
      *reinterpret_cast<uint4*>(p.kv + (int64_t)w[i].r * p.ldkv + k.col) =
          make_uint4(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7]));
  }
}

bool al(const void* q, int n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; }

int kv_entry(bool gather, KvArgs p, int64_t rows, int64_t L, int64_t S, int64_t H, int64_t T, void* stream,
             const char* name) {
  const std::string nm(name);
  const int64_t top = 0x7fffffff;
  COHERE_REQUIRE(rows >= 0 && rows <= (1 << 30) && L > 0 && S > 0 && S <= top && H > 0 && T > 0 && T <= top &&
                     H <= top / (2 * HD) / L && p.ldkv >= L * 2 * H * HD && p.ldkv % 8 == 0,
                 nm + ": bad sizes");
  COHERE_REQUIRE(p.kv && p.slot_of && p.frame_of && al(p.kv, 16), nm + ": bad pointer");
  COHERE_REQUIRE(p.k4 && p.v4 && p.ks && p.vs && al(p.k4, 16) && al(p.v4, 16) && al(p.ks, 8) && al(p.vs, 8),
                 nm + ": bad cache pointer");
  if (rows == 0) return 0;
  p.rows = (int)rows; p.S = (int)S; p.H = (int)H; p.T = (int)T;
  p.vecs = (int)(L * 2 * H);
  p.blocks = (p.vecs + 15) / 16;
  p.side = p.vecs < 16 ? 16 / p.vecs : 1;
  const auto wgs = [&](int n) { return (rows + n * p.side - 1) / (n * p.side) * p.blocks; };
  // four rows a lane where that leaves two workgroups a CU (3000 rows x 8 layers x 8 heads: gather 23.2 us, with one row
  // 30.8; 128 rows: one row 3.6 us, four 4.1)
  const bool many = wgs(4) >= 512;
  const int64_t grid = wgs(many ? 4 : 1);
  COHERE_REQUIRE(grid <= top, nm + ": too many rows for one call");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (gather && many) dec_gather_kv_q4_kernel<4><<<(unsigned)grid, 256, 0, s>>>(p);
  else if (gather) dec_gather_kv_q4_kernel<1><<<(unsigned)grid, 256, 0, s>>>(p);
  else if (many) dec_scatter_kv_q4_kernel<4><<<(unsigned)grid, 256, 0, s>>>(p);
  else dec_scatter_kv_q4_kernel<1><<<(unsigned)grid, 256, 0, s>>>(p);
  return cohere::check_launch(name);
}

// Query heads a workgroup takes (at most 4) and workgroups a key head. A workgroup of 8 heads would read the keys once for
// all of them, but their outputs alone take half of the registers of four waves a SIMD, and the vector ALU, not the
// memory, bounds 4 heads already (32 rows x 4 x 8 heads, up to 1026 keys: 16.3 us; 8 rows x 8 x 8, up to 16 K keys: 64).
struct HeadPlan { int g, chunks; };
HeadPlan head_plan(int64_t ratio) {
  const int chunks = (int)((ratio + 3) / 4);
  return {(int)((ratio + chunks - 1) / chunks), chunks};
}

// waves of a workgroup: 4 for one head (64 rows x 8 heads, up to 448 keys: 8.2 us, with 8 8.6 us), else 8 (64 rows x 8 x 2
// heads, up to 2048 keys: 22.8 us, with 4 23.9 us; more heads need a thread a dimension of each)
constexpr int waves_of(int g) { return g == 1 ? 4 : 8; }

template <bool SELF>
void launch_attention(int g, const Q4Args& p, dim3 grid, hipStream_t s) {
  switch (g) {
    case 1: dec_attention_q4_kernel<SELF, 1, waves_of(1)><<<grid, waves_of(1) * 64, 0, s>>>(p); break;
    case 2: dec_attention_q4_kernel<SELF, 2, waves_of(2)><<<grid, waves_of(2) * 64, 0, s>>>(p); break;
    case 3: dec_attention_q4_kernel<SELF, 3, waves_of(3)><<<grid, waves_of(3) * 64, 0, s>>>(p); break;
    default: dec_attention_q4_kernel<SELF, 4, waves_of(4)><<<grid, waves_of(4) * 64, 0, s>>>(p); break;
  }
}

}  // namespace

extern "C" int64_t cohere_dec_attention_q4_splits(int64_t rows, int64_t heads, int64_t kv_heads, int64_t T) {
  if (rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || T <= 0) return 1;
  const HeadPlan hp = head_plan(heads / kv_heads);
  // The time by a model, in us: the keys of a part in passes of a workgroup (64 keys a wave), at least 3/4 of one (the
  // loads' latency), times a pass and the rounds that the workgroups take, and what the parts' meeting costs (a launch, and
  // 520 bytes a head and part written and read). Several rounds of more than one head even out rows of different lengths.
  // Fitted to sweeps over 1 .. 64 parts of 28 shapes (1 .. 128 rows, 465 .. 64 K keys, 1 .. 16 heads a key head, the rows
  // of one length and from a sixteenth of it): its choice is within 12 % of the best of each. Powers of two: 48 parts of
  // 16384 keys (no whole rounds) take 9.2 us, 32 or 64 8.1 and 7.9.
  const int64_t wgs = rows * kv_heads * hp.chunks;
  const double pass = 64. * waves_of(hp.g), us = hp.g == 1 ? 0.9 : 0.5 * hp.g, slots = hp.g == 1 ? 768. : 512.;
  int64_t best = 1;
  double least = 0.;
  for (int64_t n = 1; n <= 64 && (n == 1 || T / n >= 128); n *= 2) {
    const double keys = (double)T / n / pass, rounds = wgs * n / slots;
    double t = (keys > 0.75 ? keys : 0.75) * us * (rounds > 1. ? rounds : 1.);
    if (n > 1) t += 2. + 0.0016 * rows * heads * n;
    if (hp.g > 1 && rounds >= 2.) t *= 0.85;
    if (n == 1 || t < least * 0.999) best = n, least = t;
  }
  return best;
}

extern "C" int cohere_dec_attention_q4(int32_t self, const int32_t* active, int64_t rows, const uint16_t* q, int64_t ldq,
                                       uint8_t* k4, uint8_t* v4, uint16_t* ks, uint16_t* vs, const int32_t* n,
                                       int64_t slots, int64_t heads, int64_t kv_heads, int64_t T, float scale,
                                       int64_t splits, float* part, int64_t part_len, uint16_t* out, void* stream) {
  cohere::clear_error();
  COHERE_REQUIRE(rows >= 0 && rows <= 0x7fffffff && slots > 0 && slots <= 0x7fffffff && heads > 0 && kv_heads > 0 &&
                     heads % kv_heads == 0 && heads <= 65535 && splits >= 1 && splits <= 64,
                 "dec_attention_q4: bad sizes (heads a multiple of the key heads, 1 to 64 splits)");
  COHERE_REQUIRE(T > 0 && T < (1 << 25), "dec_attention_q4: caches of 1 to 2^25 - 1 positions");  // 64 T in 31 bits
  COHERE_REQUIRE(active && q && n && out && al(q, 16) && ldq % 8 == 0 && al(out, 2) &&
                     ldq >= (heads + (self ? 2 * kv_heads : 0)) * HD,
                 "dec_attention_q4: bad pointer or row stride");
  COHERE_REQUIRE(k4 && v4 && ks && vs && al(k4, 16) && al(v4, 16) && al(ks, 8) && al(vs, 8),
                 "dec_attention_q4: bad cache pointer");
  COHERE_REQUIRE(splits == 1 || (part && part_len >= rows * heads * splits * (HD + 2)),
                 "dec_attention_q4: splits > 1 needs part with rows x heads x splits x 130 floats");
  if (rows == 0) return 0;
  const HeadPlan hp = head_plan(heads / kv_heads);
  COHERE_REQUIRE(kv_heads * hp.chunks <= 65535 && rows * heads <= 0x7fffffff, "dec_attention_q4: too many heads");
  Q4Args p{active, q, ldq, k4, v4, ks, vs, n, (int)slots, (int)heads, (int)kv_heads, (int)T, (int)(heads / kv_heads),
           hp.chunks, rows <= 65535, scale, out, part};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // Workgroups go to the eight XCDs in turn: with a row's heads behind each other every XCD has a share of the long rows
  // (16 rows x 8 x 4 heads, 2 .. 32 K keys, 8 parts: 107 us, with the rows first 127; all of 32 K: 153 and 151)
  const unsigned ny = (unsigned)(kv_heads * hp.chunks);
  const dim3 grid = p.rows_y ? dim3(ny, (unsigned)rows, (unsigned)splits) : dim3((unsigned)rows, ny, (unsigned)splits);
  if (self) launch_attention<true>(hp.g, p, grid, s);
  else launch_attention<false>(hp.g, p, grid, s);
  // few parts: 128 threads a head (64 rows x 16 heads in 2 or in 4 parts 1.5 us less)
  const unsigned hs = (unsigned)(rows * heads);
  if (splits > 4) dec_combine_q4_kernel<4, 16><<<hs, 4 * HD, 0, s>>>(part, (int)splits, out);
  else if (splits > 1) dec_combine_q4_kernel<1, 4><<<hs, HD, 0, s>>>(part, (int)splits, out);
  return cohere::check_launch("dec_attention_q4");
}

extern "C" int cohere_dec_scatter_kv_q4(const uint16_t* kv, int64_t ldkv, int64_t rows, const int32_t* slot_of,
                                        const int32_t* frame_of, uint8_t* ck, uint8_t* cv, uint16_t* cks, uint16_t* cvs,
                                        int64_t L, int64_t S, int64_t H, int64_t T, void* stream) {
  cohere::clear_error();
  const KvArgs p{const_cast<uint16_t*>(kv), slot_of, frame_of, ck, cv, cks, cvs, ldkv, 0, 0, 0, 0, 0, 0, 0};
  return kv_entry(false, p, rows, L, S, H, T, stream, "dec_scatter_kv_q4");
}

extern "C" int cohere_dec_gather_kv_q4(const int32_t* slot_of, const int32_t* frame_of, int64_t rows, const uint8_t* ck,
                                       const uint8_t* cv, const uint16_t* cks, const uint16_t* cvs, int64_t L, int64_t S,
                                       int64_t H, int64_t T, uint16_t* kv, int64_t ldkv, void* stream) {
  cohere::clear_error();
  const KvArgs p{kv, slot_of, frame_of, const_cast<uint8_t*>(ck), const_cast<uint8_t*>(cv), const_cast<uint16_t*>(cks),
                 const_cast<uint16_t*>(cvs), ldkv, 0, 0, 0, 0, 0, 0, 0};
  return kv_entry(true, p, rows, L, S, H, T, stream, "dec_gather_kv_q4");
}
