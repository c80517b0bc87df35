// Attention of new tokens over caches held in pages (paged.h states the form), and reading pages back, for gfx950. No
// counterpart in the reference, whose caches are one stretch per slot (kernels/csrc/decoder_ops.cu, dec_attn.cuh).
//
//   dec_attention_paged  softmax(q k^T scale) v of a chunk of new tokens per sequence: token j, at position n + j, attends
//                        to the n positions held in pages and to the chunk's tokens 0 .. j as given, whose keys and values
//                        go into the pages at n ..
//   dec_gather_paged     keys and values of (slot, position) pairs as bf16 rows
#include "cohere_hip.h"
#include "paged.h"

#include <string>
#include <type_traits>

namespace {

using namespace cohere_paged;

// ---- attention, few query rows -----------------------------------------------------------------------------------------
// A workgroup takes 16 query rows of a (sequence, key head) and one part of the keys; its waves take blocks of 16 keys in
// turn, and everything of a block stays in the wave's registers:
//   S^T = K Q^T on v_mfma_f32_16x16x32_bf16: lane (key l % 16, l / 16) loads 16-byte pieces of its key, and gets of the
//   result the scores of query l % 16 with keys 4 (l / 16) + i in register i. bf16 products are exact in fp32.
//   O^T = V^T P^T on v_mfma_f32_16x16x4_f32: its B operand is the weight of query l % 16 and one key of lane group l / 16:
//   register i as it stands, for keys 4 (l / 16) + i. Its A operand is 16 dimensions 8 (l % 16) + j of those keys: lane l
//   loads 8 dimensions of each of the 4 keys of its group. Neither product needs a value moved between lanes or through
//   LDS, and the weights and values are not rounded.
// The maximum, the sum and the outputs of a query stay in lanes l % 16 = query: a new maximum rescales without any move.
// Bound by the loads: 16 keys of bf16 are 8 KB and keep the matrix cores 1152 cycles of a SIMD, 16 bytes a cycle and CU at
// four SIMDs, against 8 at the memory's rate.
template <bool Q8, bool BIG, int W>
__global__ void __launch_bounds__(W * 64) paged_rows_kernel(const PagedArgs p) {
  constexpr int LD = HD + 4;
  __shared__ __attribute__((aligned(16))) float so[W][16][LD];
  __shared__ float sm[W][16], sl[W][16];
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), col = lane & 15, grp = lane >> 4;
  const int kvh = blockIdx.x % p.KV, sp = blockIdx.y, nsp = p.parts;
  Tile t = tile_of<16>(p, blockIdx.x / p.KV);
  if (t.rows == 0) return;
  // the lane's query row (the tile's last one repeated), its token and head
  const int x = t.x0 + min(col, t.rows - 1), tok = x / p.ratio, head = kvh * p.ratio + (x - tok * p.ratio);
  v8bf qf[4];
  {
    const uint16_t* qp = p.q + (int64_t)(t.first + tok) * p.ldq + head * HD;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      qf[s] = *reinterpret_cast<const v8bf*>(qp + (Q8 ? (s >> 1) * 64 + grp * 16 + (s & 1) * 8 : s * 32 + grp * 8));
  }
  int n = t.ok ? p.n[t.slot] : -1;
  const bool row_ok = n >= 0;
  n = (int)min((int64_t)max(n, 0), (int64_t)p.W << p.shift);
  // the tile's blocks: of the chunk's tokens up to its last one, then of the positions held
  const int last = (t.x0 + t.rows - 1) / p.ratio, nr = row_ok ? (last >> 4) + 1 : 0, nb = nr + ((n + 15) >> 4);
  const int chunk = (nb + nsp - 1) / nsp, start = min(nb, sp * chunk), end = min(nb, start + chunk);

  v4f acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  // scores d of the lane's query with keys 4 grp + i become weights; m, l, acc follow
  auto softmax = [&](v4f& d) {
    float mx = fmaxf(fmaxf(d[0], d[1]), fmaxf(d[2], d[3]));
    mx = xor32_max(xor16_max(mx));
    if (__any(mx > m)) {
      const float mn = fmaxf(m, mx), a = exp2_hw(m - (mn == -INFINITY ? 0.f : mn));
      l *= a;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] *= a;
      m = mn;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      d[i] = exp2_hw(d[i] - base);
      l += d[i];
    }
  };
  const uint16_t* rowkv = p.q + (int64_t)t.first * p.ldq + (p.H + kvh) * HD;
  int b = start + wave;
  for (; b < min(end, nr); b += W) {  // the chunk's own tokens, as given
    const int j0 = b * 16;
    v4f d = {0.f, 0.f, 0.f, 0.f};
    const uint16_t* kp = rowkv + (int64_t)min(j0 + col, t.c - 1) * p.ldq;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const v8bf kf =
          *reinterpret_cast<const v8bf*>(kp + (Q8 ? (s >> 1) * 64 + grp * 16 + (s & 1) * 8 : s * 32 + grp * 8));
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[s], d, 0, 0, 0);
    }
    uint4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = *reinterpret_cast<const uint4*>(rowkv + (int64_t)min(j0 + grp * 4 + i, t.c - 1) * p.ldq + p.KV * HD + col * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = j0 + grp * 4 + i <= tok ? d[i] * p.scale : -INFINITY;
    softmax(d);
    bool bad = false;  // infinities and NaN: 0 x them is NaN, where a query does not see the key
    float v[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unpack8(u[i], v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) bad |= !(fabsf(v[i][j]) < INFINITY);
    }
    if (__builtin_expect(!__any(bad), 1)) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][j], d[i], acc[j], 0, 0, 0);
    } else {  // key by key, each for the queries that see it
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll 1
        for (int g = 0; g < 4; ++g) {
          const bool sees = j0 + g * 4 + i <= tok;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const v4f o = __builtin_amdgcn_mfma_f32_16x16x4f32(grp == g ? v[i][j] : 0.f, grp == g ? d[i] : 0.f,
                                                               v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[j][k] = sees ? acc[j][k] + o[k] : acc[j][k];
          }
        }
    }
  }

  // positions held: block b's keys are positions 16 (b - nr) ..
  const int32_t* row = p.table + (int64_t)t.slot * p.W;
  const int P1 = (1 << p.shift) - 1;
  for (; b < end; b += W) {
    const int t0 = (b - nr) * 16;
    // the block's vectors: of key col (for the product with q) and of keys 4 grp + i; which of the 16 keys there are
    int64_t kvec, vvec[4];
    uint32_t live;
    if constexpr (BIG) {  // pages of 16 or more: one page
      const int page = __builtin_amdgcn_readfirstlane(row[t0 >> p.shift]);
      const bool there = (unsigned)page < (unsigned)p.pages;
      const int64_t v0 = (((int64_t)(there ? page : 0) * p.KV + kvh) << p.shift) + (t0 & P1);
      live = there ? 0xffffu >> (16 - min(n - t0, 16)) : 0u;
      kvec = v0 + col;
#pragma unroll
      for (int i = 0; i < 4; ++i) vvec[i] = v0 + grp * 4 + i;
    } else {
      const int at = min(t0 + col, n - 1), page = row[at >> p.shift];
      const bool there = (unsigned)page < (unsigned)p.pages && t0 + col < n;
      live = (uint32_t)__ballot(there) & 0xffffu;
      const int pg = there ? page : 0;
      kvec = (((int64_t)pg * p.KV + kvh) << p.shift) + (at & P1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pi = __shfl(pg, grp * 4 + i, 64);
        vvec[i] = (((int64_t)pi * p.KV + kvh) << p.shift) + (min(t0 + grp * 4 + i, n - 1) & P1);
      }
    }
    v4f d = {0.f, 0.f, 0.f, 0.f};
    float v[4][8];
    if constexpr (!Q8) {
      const uint16_t* kp = static_cast<const uint16_t*>(p.k) + kvec * HD;
      v8bf kf[4];
      uint4 u[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) kf[s] = *reinterpret_cast<const v8bf*>(kp + s * 32 + grp * 8);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        u[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.v) + vvec[i] * HD + col * 8);
#pragma unroll
      for (int s = 0; s < 4; ++s) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[s], qf[s], d, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d[i] *= p.scale;
        unpack8(u[i], v[i]);
      }
      if (live != 0xffffu) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(live >> (grp * 4 + i) & 1)) {
            d[i] = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
          }
      }
      softmax(d);
    } else {
      const int8_t* kp = static_cast<const int8_t*>(p.k) + kvec * HD;
      uint4 kr[2];
      uint2 u[4];
      float ks[4], vs[4];
#pragma unroll
      for (int s = 0; s < 2; ++s) kr[s] = *reinterpret_cast<const uint4*>(kp + s * 64 + grp * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ks[i] = p.ks[vvec[i]];
        vs[i] = p.vs[vvec[i]];
        u[i] = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(p.v) + vvec[i] * HD + col * 8);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t a = s & 1 ? kr[s >> 1].z : kr[s >> 1].x, c = s & 1 ? kr[s >> 1].w : kr[s >> 1].y;
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t y = k < 2 ? a : c;
          w[k] = pack_bf2((float)(int8_t)(y >> (16 * (k & 1))), (float)(int8_t)(y >> (16 * (k & 1) + 8)));
        }
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const v8bf*>(w), qf[s], d, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d[i] *= ks[i] * p.scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = (float)(int8_t)((j < 4 ? u[i].x : u[i].y) >> (8 * (j & 3)));
      }
      if (live != 0xffffu) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(live >> (grp * 4 + i) & 1)) {
            d[i] = -INFINITY;
            vs[i] = 0.f;
          }
      }
      softmax(d);
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] *= vs[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][j], d[i], acc[j], 0, 0, 0);
  }

  // the waves' results meet: each wave's outputs by its share of the largest maximum, summed by all threads
  l = xor32_sum(xor16_sum(l));
  if (grp == 0) {
    sm[wave][col] = m;
    sl[wave][col] = l;
  }
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w][col]);
  const float f = m == -INFINITY ? 0.f : exp2_hw(m - M);
  if (col < t.rows) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* dst = &so[wave][col][grp * 32 + i * 8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float4 o;
        // a wave without keys has outputs of 0
        o.x = m == -INFINITY ? 0.f : f * acc[4 * h][i];
        o.y = m == -INFINITY ? 0.f : f * acc[4 * h + 1][i];
        o.z = m == -INFINITY ? 0.f : f * acc[4 * h + 2][i];
        o.w = m == -INFINITY ? 0.f : f * acc[4 * h + 3][i];
        *reinterpret_cast<float4*>(dst + 4 * h) = o;
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < t.rows * HD; i += W * 64) {
    const int r = i >> 7, dim = i & (HD - 1), xr = t.x0 + r, tk = xr / p.ratio;
    float MM = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) MM = fmaxf(MM, sm[w][r]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = sm[w][r];
      L += mw == -INFINITY ? sl[w][r] : exp2_hw(mw - MM) * sl[w][r];
      O += so[w][r][dim];
    }
    const int64_t at = (int64_t)(t.first + tk) * p.H + kvh * p.ratio + (xr - tk * p.ratio);
    if (nsp == 1) {
      p.out[at * HD + dim] = f2bf(L == 0.f ? 0.f : O / L);
    } else {
      float* part = p.part + (at * nsp + sp) * (HD + 2);
      part[dim] = O;
      if (dim == 0) {
        part[HD] = MM;
        part[HD + 1] = L;
      }
    }
  }
  if (sp == 0 && row_ok) append<Q8, W>(p, t, n, kvh, 16);
}

// The parts of a (row, head), for rows of the sequences: every wave finds the maximum, the parts' weights (lane s part s's)
// and the sum; CG groups of 128 threads sum N parts each, all their loads in flight at once.
template <int CG, int N>
__global__ void __launch_bounds__(CG * HD) paged_combine_kernel(const float* __restrict__ part, const int32_t* starts, int S,
                                                                int H, int nsp, uint16_t* out) {
  const int64_t head = blockIdx.x;
  const int tid = threadIdx.x, lane = lane_id(), d = tid & (HD - 1), grp = wave_id() >> 1;
  const float* base = part + head * nsp * (HD + 2);
  const float* mine = base + min(lane, nsp - 1) * (HD + 2) + HD;
  const float ms = mine[0], ls = mine[1];
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = base[min(grp + CG * i, nsp - 1) * (HD + 2) + d];
  if (starts) {
    const int r = blockIdx.x / H;
    if (r < starts[0] || r >= starts[S]) return;
  }
  const float M = wave_max64(lane < nsp ? ms : -INFINITY);
  const float w = lane < nsp && ms != -INFINITY ? exp2_hw(ms - M) : 0.f;
  const float L = wave_sum64(lane < nsp ? (ms == -INFINITY ? ls : w * ls) : 0.f);
  float o = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (grp + CG * i < nsp) o = __builtin_fmaf(lane_value(w, grp + CG * i), v[i], o);
  if constexpr (CG == 1) {
    out[head * HD + d] = f2bf(L == 0.f ? 0.f : o / L);
  } else {
    __shared__ float so[CG][HD];
    so[grp][d] = o;
    __syncthreads();
    if (tid < HD) {
      float O = 0.f;
#pragma unroll
      for (int g = 0; g < CG; ++g) O += so[g][d];
      out[head * HD + d] = f2bf(L == 0.f ? 0.f : O / L);
    }
  }
}

// ---- reading back ------------------------------------------------------------------------------------------------------
// kv (rows, L * 2 * KV * 128): per layer KV keys, then KV values, of position pos_of[i] of slot slot_of[i]; pages (L, pages,
// KV, P, 128). 16 lanes a vector, 8 values each; a workgroup takes 16 vectors of a row, in ROWS rows.
struct GatherArgs {
  const int32_t *slot_of, *pos_of, *table;
  const void *k, *v;
  const float *ks, *vs;
  uint16_t* kv;
  int64_t ldkv;
  int rows, slots, W, pages, shift, KV, vecs, blocks;
};

template <bool Q8, int ROWS>
__global__ void __launch_bounds__(256) paged_gather_kernel(const GatherArgs p) {
  const int rb = blockIdx.x / p.blocks, d8 = threadIdx.x & 15;
  int v = (blockIdx.x - rb * p.blocks) * 16 + (threadIdx.x >> 4);
  const bool in = v < p.vecs;
  v = min(v, p.vecs - 1);  // a lane without a vector looks at the last one and writes nothing
  const int lk = v / p.KV, h = v - lk * p.KV, layer = lk >> 1, kvi = lk & 1;
  int64_t vec[ROWS];
  int col[ROWS], page[ROWS], pos[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = min(rb * ROWS + i, p.rows - 1), s = p.slot_of[r];
    pos[i] = p.pos_of[r];
    col[i] = pos[i] >> p.shift;
    const bool there = (unsigned)s < (unsigned)p.slots && pos[i] >= 0 && col[i] < p.W;
    page[i] = there ? p.table[(int64_t)s * p.W + col[i]] : -1;
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
    vec[i] = (unsigned)page[i] < (unsigned)p.pages
                 ? ((((int64_t)layer * p.pages + page[i]) * p.KV + h) << p.shift) + (pos[i] & ((1 << p.shift) - 1)) : -1;
  uint4 u[ROWS];
  float sc[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t at = vec[i] < 0 ? 0 : vec[i];
    if constexpr (Q8) {
      const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(kvi ? p.v : p.k) + at * HD + d8 * 8);
      sc[i] = (kvi ? p.vs : p.ks)[at];
      u[i].x = c.x;
      u[i].y = c.y;
    } else {
      u[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(kvi ? p.v : p.k) + at * HD + d8 * 8);
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = rb * ROWS + i;
    if (!in || r >= p.rows) continue;
    if constexpr (Q8) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = (float)(int8_t)((j < 4 ? u[i].x : u[i].y) >> (8 * (j & 3))) * sc[i];
      u[i] = make_uint4(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7]));
    }
    if (vec[i] < 0) u[i] = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(p.kv + (int64_t)r * p.ldkv + (int64_t)v * HD + d8 * 8) = u[i];
  }
}

bool al(const void* q, int n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; }

int log2_of(int64_t P) {
  for (int i = 0; i <= 8; ++i)
    if (P == (int64_t(1) << i)) return i;
  return -1;
}

constexpr int64_t TOP = 0x7fffffff;

// whether a call goes to the kernel of 128 query rows a workgroup: more than 32 rows per sequence and key head on average
bool many_rows(int64_t rows, int64_t seqs, int64_t ratio) { return rows * ratio > 32 * seqs; }

template <bool Q8>
int attention_entry(PagedArgs p, int64_t rows, int64_t seqs, int64_t slots, int64_t heads, int64_t kv_heads, int64_t width,
                    int64_t pages, int64_t P, int64_t splits, int64_t part_len, void* stream, const char* name) {
  const std::string nm(name);
  const int shift = log2_of(P);
  COHERE_REQUIRE(rows >= 0 && rows <= TOP && seqs >= 0 && seqs <= TOP && slots > 0 && slots <= TOP && heads > 0 &&
                     kv_heads > 0 && heads % kv_heads == 0 && heads <= 65535 && splits >= 1 && splits <= 64,
                 nm + ": bad sizes (heads a multiple of the key heads, 1 to 64 splits)");
  COHERE_REQUIRE(shift >= 0 && pages > 0 && pages <= TOP && width > 0 && width * P <= (int64_t(1) << 30),
                 nm + ": pages of a power of two up to 256 positions, at most 2^30 positions a slot");
  COHERE_REQUIRE(p.starts || rows == seqs, nm + ": a row per sequence, or starts");
  COHERE_REQUIRE(p.active && p.q && p.n && p.table && p.out && al(p.q, 16) && p.ldq % 8 == 0 && al(p.out, 16) &&
                     p.ldq >= (heads + 2 * kv_heads) * HD,
                 nm + ": bad pointer or row stride");
  COHERE_REQUIRE(p.k && p.v && al(p.k, 16) && al(p.v, 16) && (!Q8 || (p.ks && p.vs && al(p.ks, 4) && al(p.vs, 4))),
                 nm + ": bad page pointer");
  COHERE_REQUIRE(splits == 1 || (p.part && part_len / 130 / splits >= rows * heads),
                 nm + ": splits > 1 needs part with rows x heads x splits x 130 floats");
  if (rows == 0 || seqs == 0) return 0;
  p.R = (int)rows; p.S = (int)seqs; p.slots = (int)slots; p.W = (int)width; p.pages = (int)pages; p.shift = shift;
  p.H = (int)heads; p.KV = (int)kv_heads; p.ratio = (int)(heads / kv_heads); p.parts = (int)splits;
  p.scale *= LOG2E;
  const int64_t wgs = tiles_for(rows, seqs, p.ratio, 16, p.starts != nullptr) * kv_heads;
  COHERE_REQUIRE(wgs <= TOP && rows * heads <= TOP, nm + ": too many rows and heads");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)wgs, (unsigned)splits);
  constexpr int W = 4;
  if (many_rows(rows, seqs, p.ratio) && p.scale != 0.f) launch_chunk(p, Q8, s);
  else if (shift >= 4) paged_rows_kernel<Q8, true, W><<<grid, W * 64, 0, s>>>(p);
  else paged_rows_kernel<Q8, false, W><<<grid, W * 64, 0, s>>>(p);
  const unsigned hs = (unsigned)(rows * heads);
  if (splits > 4) paged_combine_kernel<4, 16><<<hs, 4 * HD, 0, s>>>(p.part, p.starts, p.S, p.H, p.parts, p.out);
  else if (splits > 1) paged_combine_kernel<1, 4><<<hs, HD, 0, s>>>(p.part, p.starts, p.S, p.H, p.parts, p.out);
  return cohere::check_launch(name);
}

template <bool Q8>
int gather_entry(GatherArgs p, int64_t rows, int64_t slots, int64_t width, int64_t L, int64_t pages, int64_t kv_heads,
                 int64_t P, void* stream, const char* name) {
  const std::string nm(name);
  const int shift = log2_of(P);
  COHERE_REQUIRE(rows >= 0 && rows <= (1 << 30) && slots > 0 && slots <= TOP && shift >= 0 && pages > 0 && pages <= TOP &&
                     width > 0 && width * P <= (int64_t(1) << 30) && L > 0 && kv_heads > 0 &&
                     kv_heads <= TOP / (2 * HD) / L && p.ldkv >= L * 2 * kv_heads * HD && p.ldkv % 8 == 0,
                 nm + ": bad sizes (pages of a power of two up to 256 positions)");
  COHERE_REQUIRE(p.slot_of && p.pos_of && p.table && p.kv && al(p.kv, 16), nm + ": bad pointer");
  COHERE_REQUIRE(p.k && p.v && al(p.k, 16) && al(p.v, 16) && (!Q8 || (p.ks && p.vs && al(p.ks, 4) && al(p.vs, 4))),
                 nm + ": bad page pointer");
  if (rows == 0) return 0;
  p.rows = (int)rows; p.slots = (int)slots; p.W = (int)width; p.pages = (int)pages; p.shift = shift; p.KV = (int)kv_heads;
  p.vecs = (int)(L * 2 * kv_heads);
  p.blocks = (p.vecs + 15) / 16;
  const auto wgs = [&](int n) { return (rows + n - 1) / n * p.blocks; };
  const bool many = wgs(4) >= 512;
  COHERE_REQUIRE(wgs(many ? 4 : 1) <= TOP, nm + ": too many rows for one call");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (many) paged_gather_kernel<Q8, 4><<<(unsigned)wgs(4), 256, 0, s>>>(p);
  else paged_gather_kernel<Q8, 1><<<(unsigned)wgs(1), 256, 0, s>>>(p);
  return cohere::check_launch(name);
}

}  // namespace

extern "C" int64_t cohere_dec_attention_paged_splits(int64_t rows, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t T) {
  if (rows <= 0 || seqs <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || T <= 0) return 1;
  const int64_t ratio = heads / kv_heads, wgs =
      tiles_for(rows, seqs, ratio, many_rows(rows, seqs, ratio) ? 128 : 16, rows != seqs) * kv_heads;
  int64_t n = 1;
  while (n < 64 && wgs * n < 512 && T / (2 * n) >= 128) n *= 2;
  return n;
}

extern "C" int cohere_dec_attention_paged(const int32_t* active, const int32_t* starts, int64_t seqs, const uint16_t* q,
                                          int64_t ldq, int64_t rows, uint16_t* k, uint16_t* v, int64_t pages, int64_t P,
                                          const int32_t* table, int64_t width, const int32_t* n, int64_t slots,
                                          int64_t heads, int64_t kv_heads, float scale, int64_t splits, float* part,
                                          int64_t part_len, uint16_t* out, void* stream) {
  cohere::clear_error();
  PagedArgs p{};
  p.active = active; p.starts = starts; p.q = q; p.ldq = ldq; p.k = k; p.v = v; p.table = table; p.n = n;
  p.scale = scale; p.out = out; p.part = part;
  return attention_entry<false>(p, rows, seqs, slots, heads, kv_heads, width, pages, P, splits, part_len, stream,
                                "dec_attention_paged");
}

extern "C" int cohere_dec_attention_paged_q8(const int32_t* active, const int32_t* starts, int64_t seqs, const uint16_t* q,
                                             int64_t ldq, int64_t rows, int8_t* k, int8_t* v, float* ks, float* vs,
                                             int64_t pages, int64_t P, const int32_t* table, int64_t width,
                                             const int32_t* n, int64_t slots, int64_t heads, int64_t kv_heads, float scale,
                                             int64_t splits, float* part, int64_t part_len, uint16_t* out, void* stream) {
  cohere::clear_error();
  PagedArgs p{};
  p.active = active; p.starts = starts; p.q = q; p.ldq = ldq; p.k = k; p.v = v; p.ks = ks; p.vs = vs; p.table = table;
  p.n = n; p.scale = scale; p.out = out; p.part = part;
  return attention_entry<true>(p, rows, seqs, slots, heads, kv_heads, width, pages, P, splits, part_len, stream,
                               "dec_attention_paged_q8");
}

extern "C" int cohere_dec_gather_paged(const int32_t* slot_of, const int32_t* pos_of, int64_t rows, const int32_t* table,
                                       int64_t slots, int64_t width, const uint16_t* k, const uint16_t* v, int64_t L,
                                       int64_t pages, int64_t kv_heads, int64_t P, uint16_t* kv, int64_t ldkv,
                                       void* stream) {
  cohere::clear_error();
  const GatherArgs p{slot_of, pos_of, table, k, v, nullptr, nullptr, kv, ldkv, 0, 0, 0, 0, 0, 0, 0, 0};
  return gather_entry<false>(p, rows, slots, width, L, pages, kv_heads, P, stream, "dec_gather_paged");
}

extern "C" int cohere_dec_gather_paged_q8(const int32_t* slot_of, const int32_t* pos_of, int64_t rows,
                                          const int32_t* table, int64_t slots, int64_t width, const int8_t* k,
                                          const int8_t* v, const float* ks, const float* vs, int64_t L, int64_t pages,
                                          int64_t kv_heads, int64_t P, uint16_t* kv, int64_t ldkv, void* stream) {
  cohere::clear_error();
  const GatherArgs p{slot_of, pos_of, table, k, v, ks, vs, kv, ldkv, 0, 0, 0, 0, 0, 0, 0, 0};
  return gather_entry<true>(p, rows, slots, width, L, pages, kv_heads, P, stream, "dec_gather_paged_q8");
}
