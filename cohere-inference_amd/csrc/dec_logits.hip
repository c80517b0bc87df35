// Rules on a decoding step's logits, before the greedy choice: penalties for repeated tokens, biases and grammar masks,
// for gfx950. No counterpart in the reference, which picks from the bare logits (kernels/csrc/decoder_ops.cu:106-159).
//
// Row r is slot s = active[r], p = pos[s] the position of its newest token. For token v, seen c times among the slot's
// tokens at first[s]..p, with (rep, presence, frequency) = pen[s]:
//   c > 0:  l = l / rep (l > 0) or l rep (otherwise), then l -= c frequency + presence
//   l += bias[bias_of[s]][v];   l = -inf where the mask row of the grammar's state lacks v
// in fp32, each operation rounded by itself, the result rounded once to bf16 (what the pick reads).
//
// Bound by the memory where no token is penalised (128 rows x 100008 logits: 12.1 us, 4.3 TB/s read and written); the
// penalties add the counts' way through LDS and 14 operations for each of eight logits that some lane of the wave has
// penalised (16.0 us; 128 rows x 32000, up to 300 tokens: 5.1 and 6.2; one row of 16384, 200 tokens: 2.9 and 3.8).
//
// The counts are made anew from the slot's tokens in every call (a workgroup counts, in LDS, the tokens of its own part
// of the vocabulary): no counts to keep per slot (4 bytes x vocabulary x slots), to clear when a slot is taken over or
// to wind back. Integer additions: their order does not show.
// The grammar's state at p is start[s] until the prompt has been read (p < plen[s]), then trans[state at p - 1][class of
// the token at p]; the state at p is kept in state[s][p % 2] beside the one it came from, so that every workgroup can
// derive it, a call repeated at one position gives the same, and a captured step needs nothing from the host.
#include "cohere_hip.h"
#include "common.h"

#include <string>

namespace {

struct LogitArgs {
  const uint16_t* x;
  uint16_t* y;
  int64_t ldx, ldy;
  const int32_t *active, *pos;
  const int64_t* tokens;
  const int32_t *first, *plen;
  const float* pen;  // (S, 3) or null
  const uint16_t* bias;  // (B, V) or null
  const int32_t* bias_of;
  const uint8_t* mask;  // (M, 4 ceil(V / 32)) bytes or null
  const int32_t *classes, *trans, *start;  // classes and trans null: the state stays start[s]
  int32_t* state;
  int S, V, OUT, B, M, C;
};

// J chunks of 8 logits a thread: a workgroup takes J * 8 * NT logits; counts of BITS bits (16: of at most 65535 tokens)
template <int J, int BITS, int NT>
__global__ void __launch_bounds__(NT) dec_logits_kernel(const LogitArgs a) {
  constexpr int SPAN = J * NT * 8;
  constexpr int PER = 32 / BITS;  // counts a word
  __shared__ __attribute__((aligned(16))) uint32_t cnt[SPAN / PER];
  const int r = blockIdx.y, tid = threadIdx.x, v0 = blockIdx.x * SPAN;
  const uint16_t* xr = a.x + (int64_t)r * a.ldx;
  uint16_t* yr = a.y + (int64_t)r * a.ldy;
  uint4 u[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int v = v0 + (j * NT + tid) * 8;
    u[j] = v < a.V ? *reinterpret_cast<const uint4*>(xr + v) : make_uint4(0, 0, 0, 0);
  }
  const int s = a.active[r];
  const bool known = (unsigned)s < (unsigned)a.S;  // a row of no slot is copied
  float rep = 1.f, presence = 0.f, freq = 0.f;
  int p = 0, state = -1, b = -1, lo = 0, hi = -1;
  bool penal = false;
  const int64_t* tokens = a.tokens + (known ? (int64_t)s * a.OUT : 0);
  constexpr int NK = 1024 / NT;
  // tokens lo + tid + k NT of this thread (low and high words): on their way while the rest is looked up and the counts
  // cleared. 1024 a workgroup at a time: with 2048 the loads past a short history's end cost 0.3 us (one row of 16384),
  // with 512 a long one's round trips 0.6 (128 rows x 100008, up to 4096 tokens)
  uint2 t[NK];
  // byte offsets in 32 bits (at most 2^28 tokens a slot)
  const auto at = [&](int i) {
    return *reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(tokens) + (uint32_t)i * 8u);
  };
  if (known) {
    p = a.pos[s];
    if (a.pen) {
      lo = a.first[s] > 0 ? a.first[s] : 0;
      hi = p < a.OUT ? p : a.OUT - 1;
      rep = a.pen[s * (int64_t)3];
      presence = a.pen[s * (int64_t)3 + 1];
      freq = a.pen[s * (int64_t)3 + 2];
      penal = lo <= hi;
      if (penal) {
#pragma unroll
        for (int k = 0; k < NK; ++k) t[k] = at(min(lo + tid + k * NT, hi));
      }
      penal = penal && (rep != 1.f || presence != 0.f || freq != 0.f);
    }
    if (a.bias) b = a.bias_of[s];
    if (a.mask) {
      state = a.start[s];
      if (a.trans && p >= a.plen[s]) {
        state = a.state[s * (int64_t)2 + ((p + 1) & 1)];
        const int64_t v = p >= 0 && p < a.OUT ? tokens[p] : -1;
        const int cls = v >= 0 && v < a.V ? a.classes[v] : -1;
        state = (unsigned)state < (unsigned)a.M && (unsigned)cls < (unsigned)a.C
                    ? a.trans[(int64_t)state * a.C + cls] : -1;
      }
      if (a.trans && blockIdx.x == 0 && tid == 0) a.state[s * (int64_t)2 + (p & 1)] = state;
    }
  }
  // rep = m 2^e with m in [1, 2): the quotient by m neither overflows nor needs a denormal reciprocal
  const int e = __builtin_amdgcn_frexp_expf(rep) - 1;
  const float m = 2.f * __builtin_amdgcn_frexp_mantf(rep), inv = 1.f / m;
  if (penal) {
#pragma unroll
    for (int j = 0; j < 2 * J / PER; ++j)
      *reinterpret_cast<uint4*>(&cnt[(j * NT + tid) * 4]) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i0 = lo;;) {
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const uint32_t d = t[k].x - (uint32_t)v0;  // a token below v0 comes out far above SPAN
        if (i0 + tid + k * NT <= hi && t[k].y == 0 && d < (uint32_t)SPAN)
          atomicAdd(&cnt[d / PER], 1u << (d % PER * (BITS % 32)));
      }
      i0 += NT * NK;
      if (i0 > hi) break;
#pragma unroll
      for (int k = 0; k < NK; ++k) t[k] = at(min(hi, i0 + tid + k * NT));
    }
    __syncthreads();
  }
  const uint16_t* br = (unsigned)b < (unsigned)a.B ? a.bias + (int64_t)b * a.V : nullptr;
  const uint8_t* mr =
      (unsigned)state < (unsigned)a.M ? a.mask + (int64_t)state * ((a.V + 31) / 32 * 4) : nullptr;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int place = (j * NT + tid) * 8, v = v0 + place;
    if (v >= a.V) continue;
    const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(k & 1 ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16);
    if (penal) {
      uint32_t w8[8 / PER], c[8], any = 0;
#pragma unroll
      for (int i = 0; i < 2 / PER; ++i)
        *reinterpret_cast<uint4*>(&w8[4 * i]) = *reinterpret_cast<const uint4*>(&cnt[place / PER + 4 * i]);
#pragma unroll
      for (int i = 0; i < 8 / PER; ++i) any |= w8[i];
#pragma unroll
      for (int k = 0; k < 8; ++k) c[k] = PER == 1 ? w8[k] : k & 1 ? w8[k / 2] >> 16 : w8[k / 2] & 0xffffu;
      // the quotient l / m from the reciprocal, corrected once by the exact remainder (rounded right; the fixup is for
      // infinities), times 2^-e: 5 instructions where the division takes 11
      if (any) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (!__any(c[k])) continue;  // seldom all eight, with few tokens (128 rows x 32000: 6.6 us without this)
          const float t = f[k] * inv, q = __builtin_fmaf(__builtin_fmaf(-t, m, f[k]), inv, t);
          const float l = f[k] > 0.f ? __builtin_amdgcn_div_fixupf(__builtin_amdgcn_ldexpf(q, -e), rep, f[k]) : f[k] * rep;
          f[k] = c[k] ? l - ((float)c[k] * freq + presence) : f[k];
        }
      }
    }
    if (br) {
      const uint4 t = *reinterpret_cast<const uint4*>(br + v);
      const uint32_t bw[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] += __uint_as_float(k & 1 ? bw[k >> 1] & 0xffff0000u : bw[k >> 1] << 16);
    }
    if (mr) {
      const uint32_t bits = mr[v >> 3];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t keep = (uint32_t)((int)(bits << (31 - k)) >> 31);
        f[k] = __uint_as_float((keep & __float_as_uint(f[k])) | (~keep & 0xff800000u));
      }
    }
    *reinterpret_cast<uint4*>(yr + v) =
        make_uint4(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7]));
  }
}

bool al(const void* q, int n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; }

}  // namespace

extern "C" int cohere_dec_logits(const uint16_t* x, int64_t ldx, uint16_t* y, int64_t ldy, int64_t rows, int64_t V,
                                 const int32_t* active, const int32_t* pos, int64_t slots, const int64_t* tokens,
                                 int64_t OUT, const int32_t* first, const int32_t* plen, const float* pen,
                                 const uint16_t* bias, int64_t B, const int32_t* bias_of, const int32_t* mask, int64_t M,
                                 const int32_t* classes, const int32_t* trans, int64_t C, const int32_t* start,
                                 int32_t* state, void* stream) {
  cohere::clear_error();
  const int64_t top = 0x7fffffff;
  COHERE_REQUIRE(rows >= 0 && rows <= 65535 && V > 0 && V % 8 == 0 && V < (int64_t(1) << 30) && slots > 0 &&
                     slots <= top && OUT > 0 && OUT <= (1 << 28),
                 "dec_logits: bad sizes (the vocabulary a multiple of 8)");
  COHERE_REQUIRE(x && y && al(x, 16) && al(y, 16) && ldx >= V && ldy >= V && ldx % 8 == 0 && ldy % 8 == 0,
                 "dec_logits: logits rows must be 16-byte aligned");
  COHERE_REQUIRE(active && pos && (!pen || (tokens && first)), "dec_logits: bad pointer");
  COHERE_REQUIRE(!bias || (bias_of && B > 0 && B <= top && al(bias, 16)), "dec_logits: bias rows need bias_of");
  COHERE_REQUIRE(!mask || (start && M > 0 && M <= top), "dec_logits: masks need start");
  COHERE_REQUIRE(!classes == !trans && (!trans || (mask && tokens && plen && state && C > 0 && C <= top)),
                 "dec_logits: a grammar needs masks, classes, transitions, prompt lengths and states");
  if (rows == 0) return 0;
  const LogitArgs a{x, y, ldx, ldy, active, pos, tokens, first, plen, pen, bias, bias_of,
                    reinterpret_cast<const uint8_t*>(mask), classes, trans, start, state, (int)slots, (int)V, (int)OUT,
                    (int)B, (int)M, (int)C};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // 8192 logits a workgroup of 512 where that leaves two a CU (128 rows x 100008, up to 4096 tokens each: 16.4 us; 4096 a
  // workgroup of 256 18.3, of 512 17.2, 16384 17.2), else 2048: one row of 16384 then has 8 workgroups
  const auto grid = [&](int span) { return dim3((unsigned)((V + span - 1) / span), (unsigned)rows); };
  if (OUT > 65535) dec_logits_kernel<2, 32, 256><<<grid(4096), 256, 0, s>>>(a);
  else if (rows * ((V + 8191) / 8192) >= 512) dec_logits_kernel<2, 16, 512><<<grid(8192), 512, 0, s>>>(a);
  else dec_logits_kernel<1, 16, 256><<<grid(2048), 256, 0, s>>>(a);
  return cohere::check_launch("dec_logits");
}
