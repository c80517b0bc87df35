// dec_attention_paged for chunks (paged.h states the pages' form; dec_paged.hip has the kernel of single tokens and the entry
// points), for gfx950. A workgroup whose sequence has at most 16 query rows to a key head does paged_rows.h's work on it: how
// a sequence is worked on must not hang on what else is in the call, and only the GPU knows how long each is.
//
// Else a workgroup takes 128 query rows of a (sequence, key head), 32 a wave, and one part of the keys, 64 at a time: of the
// positions held, then of the chunk's own tokens. A tile's keys and values lie in LDS as bf16 (bf16 pages straight from
// memory, int8 ones converted on the way: codes are exact in bf16, their scales go into the scores and weights); two tiles,
// so that the next one's loads run under this one's products. (Not those of int8 pages yet: a lane chooses between the scales
// of keys and values as soon as it has asked for them, which waits for the wave's loads.)
//   S^T = K Q^T on v_mfma_f32_32x32x16_bf16: queries in registers, a lane's result is 16 keys of query l % 32.
//   O^T = V^T P^T on the same instruction: the weights as they stand are its B operand (the order of the 16 keys of a
//   product is free, and taken as the lanes hold them), V^T comes through the transposing LDS read.
// What bounds it: a tile's 32 products keep a SIMD's matrix core 1024 cycles and its 200 vector instructions (32 exponentials
// at 8 cycles) about as long; a wave does one after the other, and two waves a SIMD, what the registers allow, overlap them
// only in part. 4 x 2048 tokens x 32 heads behind 6 to 8 K positions: 1044 us, 1054 TFLOP/s (a large product of the library:
// 1188); a tile alone on its CU takes 1.2 us, int8 1.7 (that wait, and their conversion).
// Maximum, sum and outputs of a query stay in lanes l % 32 = query. The base of a query's weights is set 2^8 above what its
// largest score needs (bits_of), and moves only when a score needs more, so that rescaling is rare.
// Rounded to fewer bits: the weights, to bf16 for the second product (off by at most 2^-9 of themselves; exact ones would
// need three products for one).
#include "paged_rows.h"

namespace {

using namespace cohere_paged;

constexpr int KT = 64, TM = 128, W = 4;
// tiles that a part has at least, so that its start and the joining pay (17 tokens over 8 K, int8, 32 parts asked for: 21 us,
// with 10 32)
constexpr int LEAST = 3;
constexpr float RISE = 8.f;

// 16 bytes a lane from src into LDS at dst + 16 lane. Written out, because for the builtin the compiler waits for all such
// copies in front of the next LDS read, whichever buffer that is of; the waits are tile_barrier's. No register is written,
// and the compiler's own counts of loads in flight stay safe: more are in flight than it counts, so it waits for more.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved, and named so that nothing is taken to live in it
DEVI void copy_to_lds(const void* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory", "m0");
}
// the same through a buffer: from `offset` behind its start, zeros behind its end. Five wait states lie between a vector
// instruction's write of a scalar register and a memory instruction's read of it.
DEVI void buffer_to_lds(v4i buffer, uint32_t offset, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(offset), "s"(buffer)
               : "memory", "m0");
}
#pragma clang diagnostic pop
DEVI v4i buffer_of(const void* base, int64_t offset, uint32_t bytes) {
  const uint64_t at = (uint64_t)base + offset;
  const auto uniform = [](uint32_t x) { return (int)__builtin_amdgcn_readfirstlane((int)x); };
  return v4i{uniform((uint32_t)at), uniform((uint32_t)(at >> 32) & 0xffffu), uniform(bytes), 0x00027000};
}
DEVI uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(LDS_AS const void*)p; }

// the wave's LDS operations done, and its loads
DEVI void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// G: groups of W waves, each with every G-th tile and buffers of its own, whose results meet in LDS (p.parts is 2 then, and
// there are none in memory); SPLIT: up to p.parts parts
template <bool Q8, bool BIG, bool SPLIT, int G>
__global__ void __launch_bounds__(G * W * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
paged_chunk_kernel(const PagedArgs p) {
  __shared__ __attribute__((aligned(256))) char buffers[2][G * 2][KT * 256];
  auto &kbuf = buffers[0], &vbuf = buffers[1];
  __shared__ __attribute__((aligned(16))) float sscale[Q8 ? G * 2 : 1][2][Q8 ? KT : 1];  // of a tile's keys and values
  const int lane = lane_id(), col = lane & 31, half = lane >> 5;
  const int wave = G == 1 ? wave_id() : wave_id() % W, group = G == 1 ? 0 : wave_id() / W;
  const int kvh = blockIdx.x % p.KV, sp = SPLIT ? blockIdx.y : 0, nsp = SPLIT ? p.parts : 1;
  // a chunk's last tiles first: they see the most keys, and what starts last ends last
  const Tile t = tile_of<TM>(p, gridDim.x / p.KV - 1 - blockIdx.x / p.KV);
  if (t.rows == 0) return;
  if ((int64_t)t.c * p.ratio <= FEW) {
    static_assert(sizeof(FewRows<G * W>) <= sizeof(buffers), "the few-row body's LDS");
    few_rows<Q8, BIG, SPLIT, G * W>(p, t, kvh, *reinterpret_cast<FewRows<G * W>*>(buffers));
    return;
  }
  // the lane's query row (the tile's last one repeated), its token and head
  const int x = t.x0 + min(wave * 32 + col, t.rows - 1), tok = x / p.ratio, head = kvh * p.ratio + (x - tok * p.ratio);
  const bool idle = wave * 32 >= t.rows;  // no row of the wave's
  const int tok0 = __builtin_amdgcn_readfirstlane(tok), tok1 = __builtin_amdgcn_readlane(tok, 31);
  v8bf qf[8];
  {
    const uint16_t* qp = p.q + (int64_t)(t.first + tok) * p.ldq + head * HD + half * 8;
    const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0u;  // scores are scaled by |scale|, behind the maximum
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      v4i u = *reinterpret_cast<const v4i*>(qp + s * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] ^= sign;
      qf[s] = __builtin_bit_cast(v8bf, u);
    }
  }
  const float scale = p.scale == 0.f ? 0x1p-149f : fabsf(p.scale);  // 0 x -inf, a key that is not there, would be NaN
  int n = t.ok ? p.n[t.slot] : -1;
  const int32_t* row = p.table + (int64_t)t.slot * p.W;
  const int entry0 = row[min(lane >> p.shift, p.W - 1)];  // of a first part's first tile, on its way beside n
  const bool row_ok = n >= 0;
  n = (int)min((int64_t)max(n, 0), (int64_t)p.W << p.shift);
  const int hi = row_ok ? (t.x0 + t.rows - 1) / p.ratio + 1 : 0;  // the chunk's tokens that the tile's last row sees
  const float rise = (float)bits_of((uint32_t)n + hi);
  const int np = (n + KT - 1) / KT, nb = np + (hi + KT - 1) / KT;
  // as many parts as there are for LEAST tiles each
  const int parts = SPLIT ? max(1, min(nsp, nb / LEAST)) : 1;
  if (sp >= parts) return;
  const int chunk = (nb + parts - 1) / parts, start = min(nb, sp * chunk), end = min(nb, start + chunk);
  const int P1 = (1 << p.shift) - 1;
  const uint16_t* rowkv = p.q + (int64_t)t.first * p.ldq + (p.H + kvh) * HD;

  // tile b: whether it is of the chunk's tokens, its first position, the table's entry of key `lane`, which keys there are
  const auto first_of = [&](int b) { return (b < np ? b : b - np) * KT; };
  const auto entry_of = [&](int b) { return b < np ? row[min(b * KT + lane, n - 1) >> p.shift] : 0; };
  const auto live_of = [&](int b, int entry) {
    const int at = first_of(b) + lane;
    return (uint64_t)__ballot(b < np ? at < n && (unsigned)entry < (unsigned)p.pages : at < hi);
  };
  // the vector of key kk of a tile of small pages; every lane has to be active
  const auto vec_of = [&](int t0, int entry, int kk) {
    return (((int64_t)__shfl(entry, kk, 64) * p.KV + kvh) << p.shift) + ((t0 + kk) & P1);
  };
  // A wave brings 16 keys of a tile. In LDS the 16-byte pieces c of a key's 256 bytes lie at 16 (c ^ key % 16), of a value's at
  // 16 (c ^ 4 (key % 4)); the i-th copy is of 4 keys, 16 lanes each. int8 pages come through registers.
  v4i kr[2], vr[2];
  float sr;
  const int kk0 = wave * 16, k4 = lane >> 4;
  const uint32_t piece_v = (uint32_t)((lane & 15) ^ (k4 << 2)) * 16;
  const auto piece_k = [&](int i) { return (uint32_t)((lane & 15) ^ (i * 4 + k4)) * 16; };
  const auto issue = [&](int b, int entry, uint64_t live, int buf) {
    const int t0 = first_of(b);
    const uint32_t kdst = __builtin_amdgcn_readfirstlane(lds_address(kbuf[group * 2 + buf])) + kk0 * 256,
                   vdst = __builtin_amdgcn_readfirstlane(lds_address(vbuf[group * 2 + buf])) + kk0 * 256;
    if (b >= np) {  // of the chunk's tokens
      const uint32_t stride = (uint32_t)p.ldq * 2, bytes = (uint32_t)max(min(hi - t0 - kk0, 16), 0) * stride;
      const int64_t at = (int64_t)(t0 + kk0) * stride;
      const v4i kb = buffer_of(rowkv, at, bytes), vb = buffer_of(rowkv + p.KV * HD, at, bytes);
      uint32_t first = k4;
      asm volatile("" : "+v"(first));  // the offsets are made here: kept over the tiles they would take 8 registers
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t offset = (i * 4 + first) * stride, c = lane & 15;
        buffer_to_lds(kb, offset + (c ^ (i * 4 + first)) * 16, kdst + i * 1024);
        buffer_to_lds(vb, offset + (c ^ first << 2) * 16, vdst + i * 1024);
      }
      sr = 1.f;
    } else if constexpr (BIG) {  // the wave's keys are one page's
      const int page = __builtin_amdgcn_readlane(entry, kk0);
      const bool ok = (unsigned)page < (unsigned)p.pages;
      const int64_t vec = (((int64_t)(ok ? page : 0) * p.KV + kvh) << p.shift) + ((t0 + kk0) & P1);
      const uint32_t keys = ok ? (uint32_t)max(min(n - t0 - kk0, 16), 0) : 0;
      if constexpr (Q8) {
        const auto from = [&](const void* pages, int size) {
          const v4i r = buffer_of(pages, vec * size, keys * size);  // scalar: the compiler does not see that it is
          return __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)(uint32_t)r[1] << 32 | (uint32_t)r[0]), 0, r[2], r[3]);
        };
        const auto kb = from(p.k, HD), vb = from(p.v, HD);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          kr[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(kb, lane * 16, i * 1024, 0));
          vr[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(vb, lane * 16, i * 1024, 0));
        }
        const int at = (lane & 15) * 4;
        const uint32_t ks = __builtin_amdgcn_raw_buffer_load_b32(from(p.ks, 4), at, 0, 0),
                       vs = __builtin_amdgcn_raw_buffer_load_b32(from(p.vs, 4), at, 0, 0);
        sr = __uint_as_float(lane < 16 ? ks : vs);
      } else {
        const v4i kb = buffer_of(p.k, vec * (2 * HD), keys * (2 * HD)), vb = buffer_of(p.v, vec * (2 * HD), keys * (2 * HD));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          buffer_to_lds(kb, (i * 4 + k4) * 256 + piece_k(i), kdst + i * 1024);
          buffer_to_lds(vb, (i * 4 + k4) * 256 + piece_v, vdst + i * 1024);
        }
      }
    } else if constexpr (Q8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int kk = kk0 + i * 8 + (lane >> 3);
        const int64_t vec = vec_of(t0, entry, kk);
        const bool there = live >> kk & 1;
        const int64_t at = (there ? vec : 0) * HD + (lane & 7) * 16;
        kr[i] = *reinterpret_cast<const v4i*>(static_cast<const int8_t*>(p.k) + at);
        vr[i] = *reinterpret_cast<const v4i*>(static_cast<const int8_t*>(p.v) + at);
        if (!there) kr[i] = vr[i] = v4i{0, 0, 0, 0};
      }
      const int kk = kk0 + (lane & 15);
      const int64_t vec = vec_of(t0, entry, kk);
      const bool there = live >> kk & 1;
      sr = (lane < 16 ? p.ks : p.vs)[there ? vec : 0];
      sr = there ? sr : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kk = kk0 + i * 4 + k4;
        const int64_t at = vec_of(t0, entry, kk) * (2 * HD);
        const bool there = live >> kk & 1;
        const char* zero = reinterpret_cast<const char*>(zeros);
        copy_to_lds(there ? static_cast<const char*>(p.k) + at + piece_k(i) : zero, kdst + i * 1024);
        copy_to_lds(there ? static_cast<const char*>(p.v) + at + piece_v : zero, vdst + i * 1024);
      }
    }
  };
  // int8: what is in the registers goes into LDS
  const auto convert = [&](int b, int buf) {
    if constexpr (Q8) {
      if (b < np) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int kk = wave * 16 + i * 8 + (lane >> 3);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const v4i u = z ? vr[i] : kr[i];
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int y = u[k >> 1] >> (16 * (k & 1));
              w[k] = pack_bf2((float)(int8_t)y, (float)(int8_t)(y >> 8));
            }
            const int sw = z ? (kk & 3) << 2 : kk & 15;
            char* dst = (z ? vbuf : kbuf)[group * 2 + buf] + kk * 256;
#pragma unroll
            for (int c = 0; c < 2; ++c)
              *reinterpret_cast<uint4*>(dst + ((((lane & 7) * 2 + c) ^ sw) * 16)) =
                  make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
          }
        }
      }
      if (lane < 32) sscale[group * 2 + buf][lane >> 4][wave * 16 + (lane & 15)] = sr;
    }
  };

  v16f acc[4];  // dimensions 32 dt + 8 (r / 4) + 4 half + r % 4 of query col in acc[dt][r]
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
  float base = -INFINITY, l = 0.f;
  bool bad = false;  // some values of the chunk's own tokens are infinite or NaN

  // a tile's products; OWN: of the chunk's tokens
  constexpr int AHEAD = Q8 ? 4 : 6;  // keys' pieces on their way from LDS
  const auto read_k = [&](v8bf (&kf)[AHEAD], int buf, int j) {
    kf[j % AHEAD] = *reinterpret_cast<const v8bf*>(kbuf[group * 2 + buf] + ((j >> 3) * 32 + col) * 256 +
                                                   ((((j & 7) * 2 + half) ^ (col & 15)) * 16));
  };
  const auto tile = [&](int b, int buf, uint64_t live, v8bf (&kf)[AHEAD], auto own) {
    constexpr bool OWN = decltype(own)::value;
    const int t0 = first_of(b);
    if (idle || (OWN && t0 > tok1)) return;  // no row of the wave's sees them
    const bool causal = OWN && t0 + KT - 1 > tok0;
    // The order of these steps is this source's, kept by the fences: vector work stands between the matrix products, for the
    // other wave's products to run under, and what is read from LDS is asked for some products ahead.
    v16f s[2];  // scores, then weights, of 32 keys each
    // keys 16 u + 4 half + (lane % 16) / 4 (and 8 on), dimensions 32 dt + 16 (lane / 16 % 2) + 4 (lane % 4) ..
    v8bf vf[2][4];
    const auto read_v = [&](int u) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        const int kk = half * 4 + ((lane & 15) >> 2), c = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
        const char* src = vbuf[group * 2 + buf] + (u * 16 + kk) * 256 + ((c ^ ((kk & 3) << 2)) * 16) + (lane & 1) * 8;
        const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS v4s*)src);
        const v4s d = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS v4s*)(src + 8 * 256));
        vf[u & 1][dt] = __builtin_bit_cast(v8bf, __builtin_shufflevector(a, d, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    };
    v4f ks[Q8 ? 4 : 1], vs[Q8 ? 2 : 1][2];  // scales of the lane's keys of 32, of 16
    const auto read_ks = [&](int z) {
      if constexpr (Q8)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          ks[g] = *reinterpret_cast<const v4f*>(&sscale[group * 2 + buf][0][z * 32 + g * 8 + half * 4]);
    };
    const auto read_vs = [&](int u) {
      if constexpr (Q8)
#pragma unroll
        for (int g = 0; g < 2; ++g)
          vs[u & 1][g] = *reinterpret_cast<const v4f*>(&sscale[group * 2 + buf][1][u * 16 + g * 8 + half * 4]);
    };
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
    float mx = -INFINITY;
    // Within a wave nothing runs under a matrix product, another wave's vector work does: of the two waves of a SIMD the one
    // with products alone to do goes first (4 x 2048 tokens 1068 -> 1050 us).
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      s[j >> 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[j % AHEAD], qf[j & 7], s[j >> 3], 0, 0, 0);
      if (j + AHEAD < 16) read_k(kf, buf, j + AHEAD);
      if (j + AHEAD == 16) read_v(0);
      if constexpr (Q8) {  // the first half's scales under the second half's products
        if (j == 5) read_ks(0);
        if (j >= 10 && j < 14)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[0][4 * (j - 10) + k] *= ks[j - 10][k];
        if (j == 14) read_ks(1);
        if (j == 15) read_vs(0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (Q8)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[1][r] *= ks[r >> 2][r & 3];
    if (causal || live != ~0ull) {
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        // bit 8 (r / 4) + r % 4: key z 32 + 8 (r / 4) + 4 half + r % 4 is there, and not behind the query's token
        const int upto = causal ? tok - t0 - z * 32 : 31;
        const uint32_t seen = (uint32_t)(live >> (z * 32)) & (upto < 0 ? 0u : ~0u >> max(31 - upto, 0));
        const uint32_t mine = seen >> (half * 4);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int kk = (r >> 2) * 8 + (r & 3);
          const uint32_t keep = (uint32_t)((int)(mine << (31 - kk)) >> 31);
          s[z][r] = __uint_as_float((__float_as_uint(s[z][r]) & keep) | (0xff800000u & ~keep));
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 32; ++r) mx = fmaxf(mx, s[r >> 4][r & 15]);
    mx = xor32_max(mx) * scale + rise;
    if (__any(mx > base)) {
      const float to = mx > base ? mx + RISE : base, a = to == -INFINITY ? 1.f : exp2_hw(base - to);
      l *= a;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[dt][r] *= a;
      base = to;
    }
    const float off = base == -INFINITY ? 0.f : -base;
    __builtin_amdgcn_s_setprio(0);
    // 16 keys a product: weights of keys u 16 .. as the lane's scores s[u / 2][8 (u % 2) ..], a quarter of them at a time
    v4i w[2];
    const auto weigh = [&](int u, int k) {
      float e[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        e[i] = exp2_hw(__builtin_fmaf(s[u >> 1][(u & 1) * 8 + 2 * k + i], scale, off));
        l += e[i];
        if constexpr (Q8) e[i] *= vs[u & 1][k >> 1][(k & 1) * 2 + i];
      }
      w[u & 1][k] = (int)pack_bf2(e[0], e[1]);
    };
#pragma unroll
    for (int k = 0; k < 4; ++k) weigh(0, k);
    read_vs(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (u < 3) read_v(u + 1);
      if constexpr (OWN)
        if (causal) bad |= leave_out(vf[u & 1]);
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[u & 1][dt], __builtin_bit_cast(v8bf, w[u & 1]), acc[dt], 0, 0, 0);
        if (u < 3) weigh(u + 1, dt);
        if (dt == 3 && u < 2) read_vs(u + 2);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  int entry = 0, b = start + group;
  uint64_t next = 0;
  if (b < end) {
    entry = b == 0 ? entry0 : entry_of(b);
    next = live_of(b, entry);
    issue(b, entry, next, 0);
  }
  if (sp == 0 && row_ok) {
    Append<Q8, G * W, 8 / G> own;
    for (int i = 0; own.load(p, t, n, kvh, TM, i); i += 8 / G) own.store(p, n, kvh);
  }
  if (b < end) {
    convert(b, 0);
    entry = b + G < end ? entry_of(b + G) : 0;
  }
  int buf = 0;
  const auto tiles = [&](int to, auto own) {
    for (; b < to; b += G, buf ^= 1) {
      asm volatile("" : "+v"(entry));  // waited for here, not behind the next tile's loads
      tile_barrier();                  // this tile is in LDS, and no wave reads the other buffer any more
      const uint64_t live = next;
      v8bf kf[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) read_k(kf, buf, j);
      if (b + G < end) {
        next = live_of(b + G, entry);
        issue(b + G, entry, next, buf ^ 1);
        if (b + 2 * G < end) entry = entry_of(b + 2 * G);
      }
      tile(b, buf, live, kf, own);
      if (b + G < end) convert(b + G, buf ^ 1);
    }
  };
  tiles(min(end, np), std::false_type{});
  tiles(end, std::true_type{});
  if constexpr (G == 2) {
    // every wave has passed as many barriers; the second group's results go through the buffers, which nobody reads now
    if (group == 1 && (end - start) % 2) tile_barrier();
    tile_barrier();
    v4f* outputs = reinterpret_cast<v4f*>(kbuf) + wave * 16 * 64 + lane;
    float* rest = reinterpret_cast<float*>(vbuf) + wave * 3 * 64 + lane;
    if (group == 1) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        outputs[j * 64] = v4f{acc[j >> 2][(j & 3) * 4], acc[j >> 2][(j & 3) * 4 + 1], acc[j >> 2][(j & 3) * 4 + 2],
                              acc[j >> 2][(j & 3) * 4 + 3]};
      rest[0] = base;
      rest[64] = l;
      rest[128] = bad ? 1.f : 0.f;
    }
    tile_barrier();
    if (group == 1) return;
    const float other = rest[0], to = fmaxf(base, other), mine = base == -INFINITY ? 0.f : exp2_hw(base - to),
                its = other == -INFINITY ? 0.f : exp2_hw(other - to);
    l = l * mine + rest[64] * its;
    base = to;
    bad |= rest[128] != 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const v4f o = outputs[j * 64];
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[j >> 2][(j & 3) * 4 + k] = acc[j >> 2][(j & 3) * 4 + k] * mine + o[k] * its;
    }
  }
  l = xor32_sum(l);
  if (wave * 32 + col < t.rows) {
    float size[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) size[dt] += fabsf(acc[dt][r]);
    if (__builtin_expect((bad || !((size[0] + size[1]) + (size[2] + size[3]) <= TOP * l)) && fabsf(l) < INFINITY, 0)) {
      v4f s[16];  // of the part's keys that the row sees: those held, and up to its own token
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int j = start * KT, to = (int)min((int64_t)n, (int64_t)end * KT); j < to; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) add_held<Q8>(s[i], p, row, kvh, j, i * 8 + half * 4);
#pragma unroll 1
      for (int j = max(start - np, 0) * KT, to = min(tok + 1, (end - np) * KT); j < to; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) add_given(s[i], rowkv + p.KV * HD, p.ldq, j, i * 8 + half * 4);
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = (i & 3) * 4 + k;
          acc[i >> 2][r] = s[i][k] == 0.f ? within(acc[i >> 2][r], l) : s[i][k];
        }
    }
    const int64_t at = (int64_t)(t.first + tok) * p.H + head;
    if (parts == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint16_t* dst = p.out + at * HD + half * 4;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = l == 0.f ? 0.f : acc[dt][4 * g + k] * inv;
          *reinterpret_cast<uint2*>(dst + dt * 32 + g * 8) = make_uint2(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]));
        }
    } else {
      float* part = p.part + (at * nsp + sp) * (HD + 2);
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int k = 0; k < 4; k += 2)  // parts are 520 bytes apart: 8-byte stores
            *reinterpret_cast<float2*>(part + dt * 32 + g * 8 + half * 4 + k) =
                make_float2(acc[dt][4 * g + k], acc[dt][4 * g + k + 1]);
      if (half == 0) *reinterpret_cast<float2*>(part + HD) = make_float2(base, l);
    }
    // for the joining: a negative sum, there is nothing to join; nothing in the parts that are not made
    if (sp == 0 && half == 0) {
      float* part = p.part + at * nsp * (HD + 2) + HD;
      if (nsp > 1 && parts == 1) *reinterpret_cast<float2*>(part) = make_float2(0.f, -1.f);
      for (int i = parts == 1 ? nsp : parts; i < nsp; ++i)
        *reinterpret_cast<float2*>(part + i * (HD + 2)) = make_float2(-INFINITY, 0.f);
    }
  }
}

}  // namespace

namespace cohere_paged {

int64_t chunk_workgroups(const PagedArgs& p) {
  return tiles_for(p.R, p.S, p.ratio, TM, p.starts != nullptr) * p.KV;
}

void launch_chunk(const PagedArgs& p, bool q8, hipStream_t s) {
  // Two parts are two groups of waves of one workgroup (it then has a CU to itself): the longest tile takes half as long, and
  // its results meet without a way through memory. 9 ragged sequences in bf16 52 us, in one part 65, in two through memory
  // 67; 8 x 512 tokens over nothing 22 and 25; 512 workgroups of one length 92 and 83.
  const dim3 grid((unsigned)chunk_workgroups(p), p.parts > 2 ? (unsigned)p.parts : 1);
#define CHUNK(Q, BIG) \
  (p.parts == 1   ? paged_chunk_kernel<Q, BIG, false, 1><<<grid, W * 64, 0, s>>>(p)     \
   : p.parts == 2 ? paged_chunk_kernel<Q, BIG, false, 2><<<grid, 2 * W * 64, 0, s>>>(p) \
                  : paged_chunk_kernel<Q, BIG, true, 1><<<grid, W * 64, 0, s>>>(p))
  if (q8) p.shift >= 4 ? CHUNK(true, true) : CHUNK(true, false);
  else p.shift >= 4 ? CHUNK(false, true) : CHUNK(false, false);
#undef CHUNK
}

}  // namespace cohere_paged
