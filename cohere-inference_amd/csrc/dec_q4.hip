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
// A workgroup takes one row, one key head, G of its query heads and one part of the keys. Four lanes hold a key, each
// lane one group of 32 dimensions (16 bytes of codes and its maximum), so a wave's load is 16 keys of 64 bytes, one
// after the other. A pass is U keys per quad of lanes, all loads issued before any use.
//   q.k: the query's group as 16-bit fixed point (a power of two of the group's own, so that values down to 2^-6 of the
//   group's largest are exact and the rest within 2^-15 of it: far below the codes' step), split into four signed 4-bit
//   digits that v_dot8_i32_i4 multiplies with the codes as they are: four instructions per eight products, no unpacking,
//   exact sums. One conversion and one multiplication per group and key apply m and the scale.
//   p v: the codes unpacked (3 instructions per 8, then a sign-extending conversion each) and one fma per value in fp32;
//   the value's m goes into the weight.
// Each quad keeps a running maximum, its lanes each a part of the sum (lane i the pass's key i) and 32 outputs; quads
// meet at the end.
struct Q4Args {
  const int32_t* active;
  const uint16_t* q;  // (rows, ldq): H query heads, then (self) KV keys, KV values of the new token
  int64_t ldq;
  uint8_t *k4, *v4;   // (S, KV, T, 64)
  uint16_t *ks, *vs;  // (S, KV, T, 4)
  const int32_t* n;   // per slot; self: position of the new token, cross: keys
  int S, H, KV, T, ratio, chunks;
  float scale;
  uint16_t* out;  // (rows, H * 128)
  float* part;    // (rows, H, splits, 130) when split: outputs, maximum (power of two), sum
};

constexpr float LOG2E = 1.4426950408889634f;
DEVI float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

template <bool SELF, int G, int W>
__global__ void __launch_bounds__(W * 64) dec_attention_q4_kernel(const Q4Args p) {
  constexpr int QUADS = W * 16, U = 4;
  __shared__ __attribute__((aligned(16))) uint32_t sq[G][NG][4][4];  // [head][group][digit][word]
  __shared__ float sqs[G][NG];
  __shared__ __attribute__((aligned(16))) float so[G][W][HD];
  __shared__ float sm[G][W], sl[G][W];
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), c = lane & 3, quad = tid >> 2;
  const int r = blockIdx.x, kvh = blockIdx.y / p.chunks, ch = blockIdx.y % p.chunks, sp = blockIdx.z, nsp = gridDim.z;
  // the chunk's query heads h0 .. h0 + G - 1, the last ones repeated where the chunk has fewer
  const int h0 = kvh * p.ratio + ch * G, hlast = kvh * p.ratio + p.ratio - 1;
  int s = p.active[r];
  const bool slot_ok = (unsigned)s < (unsigned)p.S;
  s = slot_ok ? s : 0;
  int n = p.n[s];
  const bool row_ok = slot_ok && n >= 0 && (!SELF || n < p.T);
  n = row_ok ? (n < p.T ? n : p.T) : 0;
  const int64_t vec0 = ((int64_t)s * p.KV + kvh) * p.T;
  const char* kb = reinterpret_cast<const char*>(p.k4) + vec0 * VB;
  const char* vb = reinterpret_cast<const char*>(p.v4) + vec0 * VB;
  const char* ksb = reinterpret_cast<const char*>(p.ks) + vec0 * (2 * NG);
  const char* vsb = reinterpret_cast<const char*>(p.vs) + vec0 * (2 * NG);
  const int chunk = (n + nsp - 1) / nsp, start = min(n, sp * chunk), end = min(n, start + chunk);

  uint4 kr[U], vr[U];
  uint32_t km[U], vm[U];
  auto load_pass = [&](int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * QUADS;
      const uint32_t jj = j < end ? j : 0;
      kr[u] = *reinterpret_cast<const uint4*>(kb + (jj * VB + c * 16));
      km[u] = *reinterpret_cast<const uint16_t*>(ksb + (jj * (2 * NG) + c * 2));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * QUADS;
      const uint32_t jj = j < end ? j : 0;
      vr[u] = *reinterpret_cast<const uint4*>(vb + (jj * VB + c * 16));
      vm[u] = *reinterpret_cast<const uint16_t*>(vsb + (jj * (2 * NG) + c * 2));
    }
  };
  int j0 = start + quad;
  load_pass(j0);

  // the query's digits, a dimension per thread
  for (int i = tid; i < G * HD; i += W * 64) {
    const int g = i >> 7, d = i & (HD - 1);
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
    // m 2^e in (15291, 30583]: the largest number of four digits -8..7 is 30583
    const int ex = 15 - __builtin_amdgcn_frexp_expf(m), e = ldexpf(m, ex) <= 30583.f ? ex : ex - 1;
    const int t = ok ? (int)rintf(ldexpf(__uint_as_float(bits), e)) : 0;
    const uint32_t u = (uint32_t)(t + 0x8888) ^ 0x8888u;  // digit k + 8 in nibble k, then k in two's complement
    const int at = d & 7;
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t w = ((u >> (4 * k)) & 15u) << (4 * at);
      w |= dpp_u<DPP_XOR1>(w);
      w |= dpp_u<DPP_XOR2>(w);
      w |= dpp_u<DPP_HALF_MIRROR>(w);
      if (at == k) mine = w;
    }
    if (at < 4) sq[g][d >> 5][at][(d >> 3) & 3] = mine;
    if ((d & 31) == 0) sqs[g][d >> 5] = ok ? ldexpf(p.scale * LOG2E / 7.f, -e) : __uint_as_float(0x7fc00000u);
  }

  float m[G], l[G], acc[G][32];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) acc[g][k] = 0.f;
  }
  // self-attention: the first quad of the first part takes the new token, as computed; the cache gets its 4 bits
  if (SELF && row_ok && sp == 0 && quad == 0) {
    const uint16_t* row = p.q + (int64_t)r * p.ldq;
    const uint16_t* kp = row + (p.H + kvh) * HD + c * 32;
    const uint16_t* vp = kp + p.KV * HD;
    float x[4][8];
    uint32_t mx = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = max_u(mx, unpack8(*reinterpret_cast<const uint4*>(kp + w * 8), x[w]));
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint16_t* qp = row + min(h0 + g, hlast) * HD + c * 32;
      float dot = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float qf[8];
        unpack8(*reinterpret_cast<const uint4*>(qp + w * 8), qf);
#pragma unroll
        for (int k = 0; k < 8; ++k) dot = __builtin_fmaf(qf[k], x[w][k], dot);
      }
      dot += dpp_mov<DPP_XOR1>(dot);
      dot += dpp_mov<DPP_XOR2>(dot);
      m[g] = dot * (p.scale * LOG2E);
      l[g] = c == 0 ? (m[g] == m[g] ? 1.f : m[g]) : 0.f;  // the maxima pass over a NaN score, the sum keeps it
    }
    const int64_t vec = vec0 + n;
    if (ch == 0) {
      const Group gk = group_of(mx);
      *reinterpret_cast<uint4*>(p.k4 + vec * VB + c * 16) =
          make_uint4(pack8(gk, x[0]), pack8(gk, x[1]), pack8(gk, x[2]), pack8(gk, x[3]));
      p.ks[vec * NG + c] = gk.store;
    }
    mx = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      mx = max_u(mx, unpack8(*reinterpret_cast<const uint4*>(vp + w * 8), x[w]));
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[g][w * 8 + k] = 7.f * x[w][k];  // outputs are summed in units of a seventh
    }
    if (ch == 0) {
      const Group gv = group_of(mx);
      *reinterpret_cast<uint4*>(p.v4 + vec * VB + c * 16) =
          make_uint4(pack8(gv, x[0]), pack8(gv, x[1]), pack8(gv, x[2]), pack8(gv, x[3]));
      p.vs[vec * NG + c] = gv.store;
    }
  }
  __syncthreads();
  uint32_t qd[G][4][4];
  float qs[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint4 t = *reinterpret_cast<const uint4*>(sq[g][c][k]);
      qd[g][k][0] = t.x; qd[g][k][1] = t.y; qd[g][k][2] = t.z; qd[g][k][3] = t.w;
    }
    qs[g] = sqs[g][c];
  }

  while (j0 - quad < end) {  // the same for the whole workgroup
    // scores of the pass's U keys, in every lane of the quad; keys past the end: -inf
    float pw[G][U];
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t w[4] = {kr[u].x, kr[u].y, kr[u].z, kr[u].w};
        int dg[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) dg[k] = __builtin_amdgcn_sdot8((int)w[i], (int)qd[g][k][i], dg[k], false);
        const int dot = (((dg[3] * 16 + dg[2]) * 16 + dg[1]) * 16) + dg[0];  // below 2^24: exact in fp32
        float t = (float)dot * (__uint_as_float(km[u] << 16) * qs[g]);
        t += dpp_mov<DPP_XOR1>(t);
        t += dpp_mov<DPP_XOR2>(t);
        pw[g][u] = j0 + u * QUADS < end ? t : -INFINITY;
      }
      float mx = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, pw[g][u]);
      const float base = mx == -INFINITY ? 0.f : mx;
      // lane i of the quad raises key i's weight; the others take it from there
      const float mine = c == 0 ? pw[g][0] : c == 1 ? pw[g][1] : c == 2 ? pw[g][2] : pw[g][3];
      const float e = exp2_hw(mine - base), a = exp2_hw(m[g] - base);
      pw[g][0] = dpp_mov<0x00>(e);
      pw[g][1] = dpp_mov<0x55>(e);
      pw[g][2] = dpp_mov<0xAA>(e);
      pw[g][3] = dpp_mov<0xFF>(e);
      l[g] = __builtin_fmaf(l[g], a, e);
      if (__any(a != 1.f)) {
#pragma unroll
        for (int k = 0; k < 32; ++k) acc[g][k] *= a;
      }
      m[g] = mx;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool live = j0 + u * QUADS < end;
      float wt[G];
#pragma unroll
      for (int g = 0; g < G; ++g) wt[g] = live ? pw[g][u] * __uint_as_float(vm[u] << 16) : 0.f;
      const uint32_t w[4] = {vr[u].x, vr[u].y, vr[u].z, vr[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float v = (float)code(w[i], k);
#pragma unroll
          for (int g = 0; g < G; ++g) acc[g][i * 8 + k] = __builtin_fmaf(wt[g], v, acc[g][i * 8 + k]);
        }
    }
    j0 += U * QUADS;
    if (j0 - quad < end) load_pass(j0);
  }

  // a wave's quads: maximum, sum and outputs. The outputs of the 16 quads meet by lane swaps (32 values over the four
  // rows of lanes: two swaps leave row i with dimensions 8 i .. 8 i + 7 of the group), then within the rows.
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float M = wave_max64(m[g]), f = M == -INFINITY ? 0.f : exp2_hw(m[g] - M);
    const float L = wave_sum64(l[g] * f);
    float o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float h[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[g][k + 8 * b] * f),
                                                        __float_as_uint(acc[g][k + 8 * b + 16] * f), false, false);
        h[b] = __uint_as_float(t[0]) + __uint_as_float(t[1]);
      }
      const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(h[0]), __float_as_uint(h[1]), false, false);
      o[k] = __uint_as_float(t[0]) + __uint_as_float(t[1]);
      o[k] += dpp_mov<DPP_ROR4>(o[k]);
      o[k] += dpp_mov<DPP_ROR8>(o[k]);
    }
    if ((lane & 12) == 0) {
      float* dst = &so[g][wave][c * 32 + (lane >> 4) * 8];
      *reinterpret_cast<float4*>(dst) = make_float4(o[0], o[1], o[2], o[3]);
      *reinterpret_cast<float4*>(dst + 4) = make_float4(o[4], o[5], o[6], o[7]);
    }
    if (lane == 0) {
      sm[g][wave] = M;
      sl[g][wave] = L;
    }
  }
  __syncthreads();
  for (int i = tid; i < G * HD; i += W * 64) {
    const int g = i >> 7, d = i & (HD - 1);
    if (ch * G + g >= p.ratio) continue;
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm[g][w]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = sm[g][w] == -INFINITY ? 0.f : exp2_hw(sm[g][w] - M);
      L = __builtin_fmaf(f, sl[g][w], L);
      O = __builtin_fmaf(f, so[g][w][d], O);
    }
    const int64_t head = (int64_t)r * p.H + h0 + g;
    if (nsp == 1) {
      p.out[head * HD + d] = f2bf(L == 0.f ? 0.f : O / (7.f * L));
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

__global__ void __launch_bounds__(HD) dec_combine_q4_kernel(const float* __restrict__ part, int nsp, uint16_t* out) {
  const int64_t head = blockIdx.x;
  const int d = threadIdx.x;
  const float* base = part + head * nsp * (HD + 2);
  float M = -INFINITY;
  for (int s = 0; s < nsp; ++s) M = fmaxf(M, base[s * (HD + 2) + HD]);
  float L = 0.f, O = 0.f;
  for (int s = 0; s < nsp; ++s) {
    const float* q = base + s * (HD + 2);
    const float w = q[HD] == -INFINITY ? 0.f : exp2_hw(q[HD] - M);
    L = __builtin_fmaf(w, q[HD + 1], L);
    O = __builtin_fmaf(w, q[d], O);
  }
  out[head * HD + d] = f2bf(L == 0.f ? 0.f : O / (7.f * L));
}

// ---- filling and reading back -----------------------------------------------------------------------------------------
// kv (rows, L * 2 * KV * 128): per layer KV keys then KV values; row i is position frame_of[i] of slot slot_of[i];
// caches (L, S, KV, T). 16 lanes per vector, 8 values (one word of codes) each; a quad of lanes holds a group.
struct KvArgs {
  uint16_t* kv;
  const int32_t *slot_of, *frame_of;
  uint8_t *k4, *v4;
  uint16_t *ks, *vs;
  int64_t ldkv;
  int rows, L, S, H, T;
};

struct KvPlace {
  bool live, in;  // a row of the call; a position of the caches
  int row, d8, kvi;
  int64_t col, vec;
};

DEVI KvPlace kv_place(const KvArgs& p) {
  const int chunks = p.L * 2 * p.H * (HD / 8);
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  KvPlace k;
  k.live = idx < (int64_t)p.rows * chunks;
  k.row = k.live ? (int)(idx / chunks) : 0;
  const int c = k.live ? (int)(idx % chunks) : 0;
  k.col = (int64_t)c * 8;
  k.d8 = c % (HD / 8);
  const int v = c / (HD / 8), h = v % p.H, l = v / (2 * p.H);
  k.kvi = v / p.H % 2;
  const int s = p.slot_of[k.row], t = p.frame_of[k.row];
  k.in = (unsigned)s < (unsigned)p.S && (unsigned)t < (unsigned)p.T;
  k.vec = k.in ? (((int64_t)l * p.S + s) * p.H + h) * p.T + t : 0;
  return k;
}

__global__ void __launch_bounds__(256) dec_scatter_kv_q4_kernel(const KvArgs p) {
  const KvPlace k = kv_place(p);
  float x[8];
  uint32_t mx = unpack8(*reinterpret_cast<const uint4*>(p.kv + (int64_t)k.row * p.ldkv + k.col), x);
  mx = quad_max_u(mx);
  if (!k.live || !k.in) return;
  const Group g = group_of(mx);
  *reinterpret_cast<uint32_t*>((k.kvi ? p.v4 : p.k4) + k.vec * VB + k.d8 * 4) = pack8(g, x);
  if ((k.d8 & 3) == 0) (k.kvi ? p.vs : p.ks)[k.vec * NG + (k.d8 >> 2)] = g.store;
}

__global__ void __launch_bounds__(256) dec_gather_kv_q4_kernel(const KvArgs p) {
  const KvPlace k = kv_place(p);
  if (!k.live) return;
  uint4 o = make_uint4(0, 0, 0, 0);
  if (k.in) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>((k.kvi ? p.v4 : p.k4) + k.vec * VB + k.d8 * 4);
    const Step m = step_of(bf2f((k.kvi ? p.vs : p.ks)[k.vec * NG + (k.d8 >> 2)]));
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = held(code(w, i), m);
    o = make_uint4(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7]));
  }
  *reinterpret_cast<uint4*>(p.kv + (int64_t)k.row * p.ldkv + k.col) = o;
}

bool al(const void* q, int n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; }

int kv_entry(bool gather, const KvArgs& p, int64_t rows, int64_t L, int64_t S, int64_t H, int64_t T, void* stream,
             const char* name) {
  const std::string nm(name);
  const int64_t top = 0x7fffffff;
  COHERE_REQUIRE(rows >= 0 && rows <= top && L > 0 && S > 0 && S <= top && H > 0 && T > 0 && T <= top &&
                     L <= top / (2 * HD) / H && p.ldkv >= L * 2 * H * HD && p.ldkv % 8 == 0,
                 nm + ": bad sizes");
  COHERE_REQUIRE(p.kv && p.slot_of && p.frame_of && al(p.kv, 16), nm + ": bad pointer");
  COHERE_REQUIRE(p.k4 && p.v4 && p.ks && p.vs && al(p.k4, 16) && al(p.v4, 16) && al(p.ks, 8) && al(p.vs, 8),
                 nm + ": bad cache pointer");
  if (rows == 0) return 0;
  const int64_t n = rows * L * 2 * H * (HD / 8), grid = (n + 255) / 256;
  COHERE_REQUIRE(grid <= top, nm + ": too many rows for one call");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (gather) dec_gather_kv_q4_kernel<<<(unsigned)grid, 256, 0, s>>>(p);
  else dec_scatter_kv_q4_kernel<<<(unsigned)grid, 256, 0, s>>>(p);
  return cohere::check_launch(name);
}

// query heads a workgroup takes (at most 4: 128 fp32 outputs a lane) and workgroups a key head
struct HeadPlan { int g, chunks; };
HeadPlan head_plan(int64_t ratio) {
  const int chunks = (int)((ratio + 3) / 4);
  return {(int)((ratio + chunks - 1) / chunks), chunks};
}

template <bool SELF>
void launch_attention(int g, const Q4Args& p, dim3 grid, hipStream_t s) {
  switch (g) {
    case 1: dec_attention_q4_kernel<SELF, 1, 8><<<grid, 512, 0, s>>>(p); break;
    case 2: dec_attention_q4_kernel<SELF, 2, 4><<<grid, 256, 0, s>>>(p); break;
    case 3: dec_attention_q4_kernel<SELF, 3, 4><<<grid, 256, 0, s>>>(p); break;
    default: dec_attention_q4_kernel<SELF, 4, 4><<<grid, 256, 0, s>>>(p); break;
  }
}

}  // namespace

extern "C" int64_t cohere_dec_attention_q4_splits(int64_t rows, int64_t heads, int64_t kv_heads, int64_t T) {
  if (rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || T <= 0) return 1;
  const HeadPlan hp = head_plan(heads / kv_heads);
  // enough workgroups for two waves of the chip's 256 CUs, each with two passes of keys at least
  const int64_t wgs = rows * kv_heads * hp.chunks, pass = hp.g == 1 ? 512 : 256;
  const int64_t want = (1024 + wgs - 1) / wgs, most = (T + 2 * pass - 1) / (2 * pass);
  const int64_t n = want < most ? want : most;
  return n < 1 ? 1 : n > 64 ? 64 : n;
}

extern "C" int cohere_dec_attention_q4(int32_t self, const int32_t* active, int64_t rows, const uint16_t* q, int64_t ldq,
                                       uint8_t* k4, uint8_t* v4, uint16_t* ks, uint16_t* vs, const int32_t* n,
                                       int64_t slots, int64_t heads, int64_t kv_heads, int64_t T, float scale,
                                       int64_t splits, float* part, int64_t part_len, uint16_t* out, void* stream) {
  cohere::clear_error();
  COHERE_REQUIRE(rows >= 0 && rows <= 0x7fffffff && slots > 0 && slots <= 0x7fffffff && heads > 0 && kv_heads > 0 &&
                     heads % kv_heads == 0 && heads <= 65535 && splits >= 1 && splits <= 64,
                 "dec_attention_q4: bad sizes (heads a multiple of the key heads, 1 to 64 splits)");
  COHERE_REQUIRE(T > 0 && T < (1 << 26), "dec_attention_q4: caches of 1 to 2^26 - 1 positions");  // 64 T in 32 bits
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
           hp.chunks, scale, out, part};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)rows, (unsigned)(kv_heads * hp.chunks), (unsigned)splits);
  if (self) launch_attention<true>(hp.g, p, grid, s);
  else launch_attention<false>(hp.g, p, grid, s);
  if (splits > 1) dec_combine_q4_kernel<<<(unsigned)(rows * heads), HD, 0, s>>>(part, (int)splits, out);
  return cohere::check_launch("dec_attention_q4");
}

extern "C" int cohere_dec_scatter_kv_q4(const uint16_t* kv, int64_t ldkv, int64_t rows, const int32_t* slot_of,
                                        const int32_t* frame_of, uint8_t* ck, uint8_t* cv, uint16_t* cks, uint16_t* cvs,
                                        int64_t L, int64_t S, int64_t H, int64_t T, void* stream) {
  cohere::clear_error();
  const KvArgs p{const_cast<uint16_t*>(kv), slot_of, frame_of, ck, cv, cks, cvs, ldkv, (int)rows, (int)L, (int)S,
                 (int)H, (int)T};
  return kv_entry(false, p, rows, L, S, H, T, stream, "dec_scatter_kv_q4");
}

extern "C" int cohere_dec_gather_kv_q4(const int32_t* slot_of, const int32_t* frame_of, int64_t rows, const uint8_t* ck,
                                       const uint8_t* cv, const uint16_t* cks, const uint16_t* cvs, int64_t L, int64_t S,
                                       int64_t H, int64_t T, uint16_t* kv, int64_t ldkv, void* stream) {
  cohere::clear_error();
  const KvArgs p{kv, slot_of, frame_of, const_cast<uint8_t*>(ck), const_cast<uint8_t*>(cv), const_cast<uint16_t*>(cks),
                 const_cast<uint16_t*>(cvs), ldkv, (int)rows, (int)L, (int)S, (int)H, (int)T};
  return kv_entry(true, p, rows, L, S, H, T, stream, "dec_gather_kv_q4");
}
