// Caches in pages, as the kernels over them share it (dec_paged.hip, dec_paged_chunk.hip, paged_rows.h).
//
// Pages (pages, KV, P, 128), P a power of two up to 256; position t of slot s is in page table[s][t / P] at t % P. A
// table entry outside 0 .. pages - 1 is an absent page: its positions are neither read nor written. 16 bits: bf16. 8 bits:
// int8 codes with an fp32 scale per vector (pages, KV, P): s = max(m / 127, 2^-126), m the vector's largest magnitude,
// code round_half_even(x fp32(1 / s)); a vector with a NaN or an infinity has a scale that is not finite and reads back as
// NaN throughout.
#pragma once
#include "common.h"

#include <type_traits>

namespace cohere_paged {

constexpr int HD = 128;  // head size
constexpr float LOG2E = 1.4426950408889634f;
typedef short v4s __attribute__((ext_vector_type(4)));

// what absent keys and values are read from
static __device__ __attribute__((aligned(16))) uint32_t zeros[4];

struct PagedArgs {
  const int32_t *active, *starts;  // starts null: sequence i is row i
  const uint16_t* q;               // (rows, ldq): H query heads, then KV keys, KV values of the new tokens
  int64_t ldq;
  void *k, *v;     // bf16 or int8 pages
  float *ks, *vs;  // int8: scales
  const int32_t *table, *n;
  int R, S, slots, W, pages, shift, H, KV, ratio;  // rows, sequences, table width, log2 P
  float scale;  // times log2(e): scores are powers of two
  uint16_t* out;  // (rows, H * 128)
  float* part;    // (rows, H, parts, 130) when split: outputs, maximum (power of two), sum
  int parts;
};

DEVI float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Weights are at most 2^-bits_of(a row's number of keys), so that their sum is below 1 and that of weight x value no larger
// than the largest value: with weights up to 1 two of the type's largest would be infinite before the division.
DEVI int bits_of(uint32_t keys) { return __builtin_amdgcn_readfirstlane(32 - __clz((int)keys)); }
// A mean is no larger than the type's largest, and the sums' roundings must not make it so: a finite sum o of weight x value,
// `weights` the sum of weights. Whether any of several is too large, or not finite, is seen at their magnitudes' sum.
constexpr float TOP = 0x1.fep127f;
DEVI float within(float o, float weights) {
  const float most = TOP * weights;
  return fabsf(o) > most && fabsf(o) < INFINITY ? copysignf(most, o) : o;
}

// One workgroup's sequence and tile of TM query rows (x = token * ratio + head of the key head's): sequence i has the
// tiles base(i) .. , base(i) = floor(starts[i] ratio / TM) + i, which leaves each at least the tiles that it needs, so that
// neither the host nor a prefix sum has to know the chunks. Tiles without rows end at once.
struct Tile {
  int first, c, slot, x0, rows;  // first row, tokens; -1: none
  bool ok;                       // the slot is in range
};
template <int TM>
DEVI Tile tile_of(const PagedArgs& p, int w) {
  Tile t;
  t.x0 = 0;
  t.rows = 0;
  if (p.starts) {
    const int lane = lane_id();
    int i, a, b;
    if (p.S < 64) {  // all of it in one round trip
      const int start = min(max(p.starts[min(lane, p.S)], 0), p.R), slot = p.active[min(lane, p.S - 1)];
      i = __popcll(__ballot(lane < p.S && (int64_t)start * p.ratio / TM + lane <= w)) - 1;
      if (i < 0) return t;
      a = __builtin_amdgcn_readlane(start, i);
      b = max(__builtin_amdgcn_readlane(start, i + 1), a);
      t.slot = __builtin_amdgcn_readlane(slot, i);
    } else {
      int count = 0;
      for (int i0 = 0; i0 < p.S; i0 += 64) {
        const int at = i0 + lane;
        const int64_t start = at < p.S ? min(max(p.starts[at], 0), p.R) : 0;
        count += __popcll(__ballot(at < p.S && start * p.ratio / TM + at <= w));
      }
      i = count - 1;
      if (i < 0) return t;
      a = min(max(p.starts[i], 0), p.R);
      b = min(max(p.starts[i + 1], a), p.R);
      t.slot = p.active[i];
    }
    t.first = a;
    t.c = b - a;
    t.x0 = (w - ((int)((int64_t)a * p.ratio / TM) + i)) * TM;
  } else {
    const int tiles = (p.ratio + TM - 1) / TM, i = w / tiles;
    t.x0 = (w - i * tiles) * TM;
    t.first = i;
    t.c = 1;
    t.slot = p.active[i];
  }
  const int64_t left = (int64_t)t.c * p.ratio - t.x0;
  t.rows = t.x0 < 0 ? 0 : left < TM ? (left > 0 ? (int)left : 0) : TM;  // below 0: starts that do not ascend
  t.ok = (unsigned)t.slot < (unsigned)p.slots;
  t.slot = t.ok ? t.slot : 0;
  return t;
}

// the number of tiles that a grid has to have (the kernel's own: R ratio / TM + S, one a sequence and TM heads without starts)
inline int64_t tiles_for(int64_t R, int64_t S, int64_t ratio, int64_t TM, bool starts) {
  return starts ? R * ratio / TM + S : S * ((ratio + TM - 1) / TM);
}

// the largest magnitude of the 16 lanes' values as bits (a NaN's are above any number's)
DEVI uint32_t row16_max_bits(uint32_t m) {
  const auto mx = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  const auto mv = [](uint32_t v, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, false);
  };
  m = mx(m, mv(m, std::integral_constant<int, DPP_XOR1>{}));
  m = mx(m, mv(m, std::integral_constant<int, DPP_XOR2>{}));
  m = mx(m, mv(m, std::integral_constant<int, DPP_ROR4>{}));
  return mx(m, mv(m, std::integral_constant<int, DPP_ROR8>{}));
}

DEVI void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = __uint_as_float(w[k] << 16);
    f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
  }
}

// Infinities and NaN among a chunk's own values: 0 x them is NaN, where a query does not see the key. They leave the product
// (made zeros; whether there were any in the wave), and come back to the outputs of the rows that see them at the end.
template <int N>
DEVI bool leave_out(v8bf (&v)[N]) {
  const auto marks = [](int w) { return ((uint32_t)w & 0x7f807f80u) + 0x00800080u; };  // bits 15, 31: exponent of all ones
  uint32_t any = 0;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= marks(__builtin_bit_cast(v4i, v[k])[i]);
  const bool some = __any(any & 0x80008000u);
  if (__builtin_expect(some, 0)) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v4i w = __builtin_bit_cast(v4i, v[k]);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] &= (int)~((marks(w[i]) >> 15 & 0x00010001u) * 0xffffu);
      v[k] = __builtin_bit_cast(v8bf, w);
    }
  }
  return some;
}
// the value, if it is infinite or NaN
DEVI float not_finite(float x) { return fabsf(x) < INFINITY ? 0.f : x; }

// Outputs that infinite or NaN values have reached: in the products they meet weights that are rounded to 0 and remainders of
// weights, and become NaN, where the definition has them whole. These outputs are the sums of such values alone, which are
// read once more: 4 dimensions from `dim` on, of token j as given (rowv: the chunk's first values) or of position t held.
DEVI void add_given(v4f& s, const uint16_t* rowv, int64_t ldq, int j, int dim) {
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] += not_finite(__uint_as_float((uint32_t)rowv[j * ldq + dim + i] << 16));
}
template <bool Q8>
DEVI void add_held(v4f& s, const PagedArgs& p, const int32_t* row, int kvh, int t, int dim) {
  const int page = row[t >> p.shift];
  if ((unsigned)page >= (unsigned)p.pages) return;
  const int64_t vec = (((int64_t)page * p.KV + kvh) << p.shift) + (t & ((1 << p.shift) - 1));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Q8) s[i] += not_finite((float)static_cast<const int8_t*>(p.v)[vec * HD + dim + i] * p.vs[vec]);
    else s[i] += not_finite(__uint_as_float((uint32_t)static_cast<const uint16_t*>(p.v)[vec * HD + dim + i] << 16));
  }
}
// a part's output by its weight; one that is not finite however small that is
DEVI float add_part(float w, float v, float o) { return fabsf(v) < INFINITY ? __builtin_fmaf(w, v, o) : o + v; }

// a vector (16 lanes, 8 values each, u) as it is held, at vector `vec` of the pages; every lane takes part, `live` writes
template <bool Q8>
DEVI void store_vec(const uint4& u, void* pages, float* scales, int64_t vec, int d8, bool live) {
  if constexpr (!Q8) {
    if (live) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(pages) + vec * HD + d8 * 8) = u;
  } else {
    float f[8];
    unpack8(u, f);
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t b = __float_as_uint(f[k]) & 0x7fffffffu;
      m = b > m ? b : m;
    }
    // (the bits of the largest magnitude, not fmaxf, which passes over a NaN)
    const float mx = __uint_as_float(row16_max_bits(m)), d = mx / 127.f;
    const float s = d < 0x1p-126f ? 0x1p-126f : d, inv = 1.f / s;
    if (!live) return;
    *reinterpret_cast<uint2*>(static_cast<int8_t*>(pages) + vec * HD + d8 * 8) =
        make_uint2(q8x4(f[0], f[1], f[2], f[3], inv), q8x4(f[4], f[5], f[6], f[7], inv));
    // an infinity's scale would read back its vector's zeros as NaN and the others as infinite or NaN: all NaN
    if (d8 == 0) scales[vec] = mx < __uint_as_float(0x7f800000u) ? s : __uint_as_float(0x7fc00000u);
  }
}

// The keys and values of the tile's own tokens (those whose first query row is in the tile) into their pages, by W waves,
// the last one first (the first one has more to do where there are few keys), 4 vectors a wave and step: N steps from step
// i on are loaded, and stored later.
// No workgroup reads them there in the same launch: a chunk attends to its own tokens as given.
template <bool Q8, int W, int N>
struct Append {
  v4i u[N];
  int page[N], first;

  // whether there is something to do
  DEVI bool load(const PagedArgs& p, const Tile& t, int n, int kvh, int TMrows, int i) {
    const int lane = lane_id(), kvi = (lane >> 4) & 1;
    const int j0 = (t.x0 + p.ratio - 1) / p.ratio, j1 = min(t.c, (t.x0 + TMrows + p.ratio - 1) / p.ratio);
    first = j0 * 2 + (i * W + W - 1 - wave_id()) * 4 + (lane >> 4);
    if (first - (lane >> 4) >= j1 * 2) return false;
    const uint16_t* src = p.q + (int64_t)t.first * p.ldq + (p.H + kvi * p.KV + kvh) * HD + (lane & 15) * 8;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = (first + k * W * 4) >> 1;
      const int64_t column = ((int64_t)n + j) >> p.shift;
      page[k] = p.table[(int64_t)t.slot * p.W + min(column, (int64_t)p.W - 1)];
      if (j >= j1 || column >= p.W) page[k] = -1;
      u[k] = *reinterpret_cast<const v4i*>(src + (int64_t)min(j, t.c - 1) * p.ldq);
    }
    return true;
  }
  DEVI void store(const PagedArgs& p, int n, int kvh) const {
    const int lane = lane_id(), kvi = (lane >> 4) & 1;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t pos = (int64_t)n + ((first + k * W * 4) >> 1);
      const bool live = (unsigned)page[k] < (unsigned)p.pages;
      const int64_t vec = live ? (((int64_t)page[k] * p.KV + kvh) << p.shift) + (pos & ((1 << p.shift) - 1)) : 0;
      store_vec<Q8>(__builtin_bit_cast(uint4, u[k]), kvi ? p.v : p.k, kvi ? p.vs : p.ks, vec, lane & 15, live);
    }
  }
};

// the kernel for chunks (dec_paged_chunk.hip)
int64_t chunk_workgroups(const PagedArgs& p);
void launch_chunk(const PagedArgs& p, bool q8, hipStream_t s);

}  // namespace cohere_paged
