// Attention over pages for sequences of at most 16 query rows a key head (paged.h states the pages' form): the body of
// dec_paged.hip's kernel of single tokens, and of such sequences' workgroups in dec_paged_chunk.hip's.
//
// A workgroup takes the query rows of a (sequence, key head) and one part of the keys; its waves take blocks of 32 keys in
// turn, each by itself:
//   S^T = K Q^T on v_mfma_f32_16x16x32_bf16, twice 16 keys: lane (key l % 16, l / 16) loads 16-byte pieces of its keys, and
//   gets of the result the scores of query l % 16 with keys 4 (l / 16) + i in register i. bf16 products are exact in fp32.
//   O^T = V^T P^T on the same instruction, 32 keys at once: the weights as they stand are its B operand (the order of the
//   32 keys is free, and taken as the lanes hold them); V^T comes from the wave's own 8 KB of LDS, into which the loads go
//   straight (int8: through registers, converted), by the transposing read. A weight is held as the sum of two bf16 numbers
//   (to 2^-17 of itself), two products.
// The maximum, the sum and the outputs of a query stay in lanes l % 16 = query: a new maximum rescales without any move.
// Why not fp32 products, which need no LDS and no second bf16 number: 16 keys would keep a SIMD's matrix core 1024 cycles
// where this takes 128, and a wave alone took 2570 cycles for 16 keys.
#pragma once
#include "paged.h"

namespace cohere_paged {

constexpr int KB = 32, FEW = 16;

// the workgroup's LDS
template <int W>
struct FewRows {
  static constexpr int LD = HD + 4, REGION = FEW * LD * 4;  // a wave's values (32 x 256 bytes), later its outputs
  static_assert(REGION >= KB * 256 && REGION % 256 == 0, "a wave's region");
  alignas(256) char region[W * REGION];
  float m[W][FEW], l[W][FEW];
  int bad[W];
};

// 16 bytes a lane from `offset` + `more` behind a buffer's start, zeros behind its end, into LDS at dst + 16 lane
DEVI void buffer_to_lds(__amdgpu_buffer_rsrc_t r, int offset, int more, char* dst) {
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass refuses the builtin
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LDS_AS void*)dst, 16, offset, more, 0, 0);
#endif
}

// The rows of tile t, which is a sequence's only one, with key head kvh; part blockIdx.y of p.parts with SPLIT, else all keys
template <bool Q8, bool BIG, bool SPLIT, int W>
DEVI void few_rows(const PagedArgs& p, const Tile& t, int kvh, FewRows<W>& lds) {
  constexpr int LD = FewRows<W>::LD, REGION = FewRows<W>::REGION;
  constexpr int nr = 1;  // blocks of the chunk's own tokens
  auto& sm = lds.m;
  auto& sl = lds.l;
  auto& sbad = lds.bad;
  char* const region = lds.region;
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), col = lane & 15, grp = lane >> 4;
  const int sp = SPLIT ? blockIdx.y : 0, nsp = SPLIT ? p.parts : 1;
  char* sv = region + wave * REGION;
  const int32_t* row = p.table + (int64_t)t.slot * p.W;
  const int P1 = (1 << p.shift) - 1;
  // the blocks: of the chunk's own tokens, 16 at most, then of the positions held; wave w has every W-th
  int n = 0, nb = 0, start = 0, end = 0, b = wave;
  float most = 0.f;  // a weight's
  bool row_ok = false;
  const int held = p.n[t.slot];  // on its way
  const auto bounds = [&]() {
    n = t.ok ? held : -1;
    row_ok = n >= 0;
    n = (int)min((int64_t)max(n, 0), (int64_t)p.W << p.shift);
    nb = row_ok ? nr + (n + KB - 1) / KB : 0;
    most = __uint_as_float((uint32_t)(127 - bits_of((uint32_t)n + t.c)) << 23);
  };
  if constexpr (SPLIT) {  // without parts nothing up to the first loads waits for n
    bounds();
    const int chunk = (nb + nsp - 1) / nsp;
    start = min(nb, sp * chunk);
    end = min(nb, start + chunk);
    b = start + wave;
  }
  // The first of the wave's blocks of positions held, and the pages of these. BIG (pages of 16 or more): of half h of the
  // k-th one in lane 2 (k % 32) + h. Else one a key (lane % 32), one block ahead.
  const int b0 = b == 0 ? W : b;
  const auto entry_of = [&](int block) {
    const int64_t at = BIG ? (int64_t)(block + (lane >> 1) * W - nr) * KB + (lane & 1) * 16
                           : (int64_t)(block - nr) * KB + (lane & 31);
    return row[min(at >> p.shift, (int64_t)p.W - 1)];
  };
  int entry = entry_of(b0);

  // the lane's query row (the tile's last one repeated), its token and head
  const bool single = t.c == 1, first = single && b == 0;
  const int x = min(col, t.rows - 1), tok = single ? 0 : x / p.ratio,
            head = kvh * p.ratio + (x - tok * p.ratio);
  // the dimensions that a lane holds of a product's step s: as 16-byte loads of int8 or bf16 vectors bring them
  const auto dims = [&](int s) { return Q8 ? (s >> 1) * 64 + grp * 16 + (s & 1) * 8 : s * 32 + grp * 8; };
  v8bf qf[4];
  {
    const uint16_t* qp = p.q + (int64_t)(t.first + tok) * p.ldq + head * HD;
#pragma unroll
    for (int s = 0; s < 4; ++s) qf[s] = *reinterpret_cast<const v8bf*>(qp + dims(s));
  }

  const uint16_t* rowkv = p.q + (int64_t)t.first * p.ldq + (p.H + kvh) * HD;
  // A chunk of one token has one key of its own, which every row sees: its score is the first maximum and its value the
  // first outputs, without a product; the loads are made here, and waited for behind the first block's.
  v8bf k1[4];
  uint2 v1[8];
  if (first) {
#pragma unroll
    for (int s = 0; s < 4; ++s) k1[s] = *reinterpret_cast<const v8bf*>(rowkv + dims(s));
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) v1[dt] = *reinterpret_cast<const uint2*>(rowkv + p.KV * HD + dt * 16 + grp * 4);
  }

  v4f acc[8];  // dimensions 16 dt + 4 grp + i of query col in acc[dt][i]
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) acc[dt] = v4f{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  // scores d of the lane's query with keys 16 h + 4 grp + i become weights; m, l, acc follow
  const auto softmax = [&](v4f (&d)[2]) {
    float mx = fmaxf(fmaxf(fmaxf(d[0][0], d[0][1]), fmaxf(d[0][2], d[0][3])),
                     fmaxf(fmaxf(d[1][0], d[1][1]), fmaxf(d[1][2], d[1][3])));
    mx = xor32_max(xor16_max(mx));
    if (__any(mx > m)) {
      const float mn = fmaxf(m, mx), a = exp2_hw(m - (mn == -INFINITY ? 0.f : mn));
      l *= a;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) acc[dt] *= a;
      m = mn;
    }
    const float to = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d[h][i] = exp2_hw(d[h][i] - to) * most;
        l += d[h][i];
      }
  };
  // Values lie in LDS as bf16: key k's 16-byte pieces c at 256 k + 16 (c ^ 2 (k % 8)), so that the transposing reads, 16
  // keys' 32 bytes each, meet no bank twice.
  v8bf vf[8];
  const auto read_v = [&]() {
    const int k = grp * 4 + (col >> 2), at = k * 256 + (k & 7) * 32 + (col & 3) * 8;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      const char* src = sv + (at ^ (dt * 32));
      const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS v4s*)src);
      const v4s c = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS v4s*)(src + 16 * 256));
      vf[dt] = __builtin_bit_cast(v8bf, __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read, before other values are on their way
  };
  // weights as the product's B operand, twice: rounded, and what that left
  const auto products = [&](const v4f (&d)[2]) {
    v4i hi, lo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = d[k >> 1][(k & 1) * 2], c = d[k >> 1][(k & 1) * 2 + 1];
      hi[k] = (int)pack_bf2(a, c);
      lo[k] = (int)pack_bf2(a - __uint_as_float((uint32_t)hi[k] << 16), c - __uint_as_float((uint32_t)hi[k] & 0xffff0000u));
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
      acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[dt], __builtin_bit_cast(v8bf, hi), acc[dt], 0, 0, 0);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
      acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[dt], __builtin_bit_cast(v8bf, lo), acc[dt], 0, 0, 0);
  };

  // the chunk's own tokens, as given; bad: some of their values are infinite or NaN
  bool bad = false;
  if (!single && b == 0) {
    if constexpr (!SPLIT) bounds();  // what a weight is at most
    const auto own_row = [&](int j) { return rowkv + (int64_t)min(j, t.c - 1) * p.ldq; };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = i * 4 + grp;
      const char* at = reinterpret_cast<const char*>(own_row(k) + p.KV * HD) + (col ^ ((k & 7) * 2)) * 16;
      at = k < t.c ? at : reinterpret_cast<const char*>(zeros);
      __builtin_amdgcn_global_load_lds(at, (LDS_AS void*)(sv + i * 4 * 256), 16, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    v4f d[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t* kp = own_row(h * 16 + col);
      d[h] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s)
        d[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const v8bf*>(kp + dims(s)), qf[s], d[h], 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) d[h][i] = h * 16 + grp * 4 + i <= tok ? d[h][i] * p.scale : -INFINITY;
    }
    __builtin_amdgcn_sched_barrier(0);
    softmax(d);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    read_v();
    bad = leave_out(vf);
    products(d);
  }

  // Positions held. A block's keys and values on their way. BIG: through buffers of a half (nothing, where it has no page),
  // addressed by constants; else an absent page's keys read page 0, and its values zeros.
  constexpr int VEC = Q8 ? HD : 2 * HD, KS = Q8 ? 2 : 4;  // bytes of a vector, loads of a key
  v4i kf[2][KS], vr[Q8 ? 4 : 1];
  v4f ks[2], vs[2];
  uint32_t there = 0;  // keys with a page
  int pages_of = 0;
  int64_t base[2];
  const auto rsrc = [&](const void* pages, int h, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(pages)) + base[h] * bytes, 0,
                                             there >> (16 * h) & 1 ? 16 * bytes : 0, 0x00027000);
  };
  const auto vec_of = [&](int block, int k) {  // vectors are counted in 32 bits
    return (((uint32_t)__shfl(pages_of, k, 64) * (uint32_t)p.KV + kvh) << p.shift) + (((block - nr) * KB + k) & P1);
  };
  const auto load_k = [&](int block, bool any) {  // any: the block is one
    if constexpr (BIG) {
      there = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int page = __builtin_amdgcn_readlane(entry, ((block - b0) / W & 31) * 2 + h);
        const bool ok = any & ((unsigned)page < (unsigned)p.pages);
        base[h] = (((int64_t)(ok ? page : 0) * p.KV + kvh) << p.shift) + (((block - nr) * KB + h * 16) & P1);
        there |= ok ? 0xffffu << (16 * h) : 0u;
      }
    } else {
      const bool ok = any && (unsigned)entry < (unsigned)p.pages;
      there = (uint32_t)__ballot(ok);  // lanes 32 .. hold the same
      pages_of = ok ? entry : 0;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (BIG) {
        const auto r = rsrc(p.k, h, VEC);
#pragma unroll
        for (int s = 0; s < KS; ++s)
          kf[h][s] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, col * VEC + grp * 16 + s * 64, 0, 0));
        if constexpr (Q8) {
          ks[h] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rsrc(p.ks, h, 4), grp * 16, 0, 0));
          vs[h] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rsrc(p.vs, h, 4), grp * 16, 0, 0));
        }
      } else {
        const char* at = static_cast<const char*>(p.k) + (uint64_t)vec_of(block, h * 16 + col) * VEC;
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[h][s] = *reinterpret_cast<const v4i*>(at + grp * 16 + s * 64);
        if constexpr (Q8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t vec = vec_of(block, h * 16 + grp * 4 + i);
            ks[h][i] = p.ks[vec];
            vs[h][i] = p.vs[vec];
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
  };
  const auto load_v = [&](int block) {
    if constexpr (Q8) {  // 8 keys a load, 16 dimensions a lane
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (BIG)
          vr[i] = __builtin_bit_cast(
              v4i, __builtin_amdgcn_raw_buffer_load_b128(rsrc(p.v, i >> 1, VEC), lane * 16 + (i & 1) * 8 * VEC, 0, 0));
        else
          vr[i] = *reinterpret_cast<const v4i*>(static_cast<const char*>(p.v) +
                                                (uint64_t)vec_of(block, i * 8 + (lane >> 3)) * VEC + (lane & 7) * 16);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = i * 4 + grp, c = col ^ ((k & 7) * 2);
        if constexpr (BIG) {
          buffer_to_lds(rsrc(p.v, i >> 2, VEC), grp * VEC + c * 16, (i & 3) * 4 * VEC, sv + i * 4 * 256);
        } else {
          const char* at = static_cast<const char*>(p.v) + (uint64_t)vec_of(block, k) * VEC + c * 16;
          at = there >> k & 1 ? at : reinterpret_cast<const char*>(zeros);
          __builtin_amdgcn_global_load_lds(at, (LDS_AS void*)(sv + i * 4 * 256), 16, 0, 0);
          __builtin_amdgcn_sched_barrier(0);  // one address after the other: together they would take 16 registers
        }
      }
    }
  };
  load_k(b0, true);
  load_v(b0);
  if constexpr (!BIG) entry = entry_of(b0 + W);
  if constexpr (!SPLIT) {
    bounds();
    end = nb;
  }
  Append<Q8, W, 2> own;  // 16 tokens at most: two steps
  const bool writes = sp == 0 && row_ok && own.load(p, t, n, kvh, 16, 0);
  if (first) {
    float dot = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float a[8], c[8];
      unpack8(__builtin_bit_cast(uint4, qf[s]), a);
      unpack8(__builtin_bit_cast(uint4, k1[s]), c);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = __builtin_fmaf(a[i], c[i], dot);
    }
    dot = xor32_sum(xor16_sum(dot)) * p.scale;
    m = dot == dot ? dot : -INFINITY;  // maxima pass over a NaN, the sum keeps it
    const float e = dot == -INFINITY ? 0.f : exp2_hw(dot - m) * most;
    l = grp == 0 ? e : 0.f;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
      acc[dt] = e * v4f{__uint_as_float(v1[dt].x << 16), __uint_as_float(v1[dt].x & 0xffff0000u),
                        __uint_as_float(v1[dt].y << 16), __uint_as_float(v1[dt].y & 0xffff0000u)};
  }

  // Each block's loads are made under the products of the one before it.
  for (b = b0; b < end; b += W) {
    const int left = n - (b - nr) * KB;
    const uint32_t live = (left < KB ? ~0u >> (KB - left) : ~0u) & there;
    v4f d[2], vscale[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      d[h] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        v4i w;
        if constexpr (Q8) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int y = kf[h][s >> 1][(s & 1) * 2 + (k >> 1)];
            w[k] = (int)pack_bf2((float)(int8_t)(y >> (16 * (k & 1))), (float)(int8_t)(y >> (16 * (k & 1) + 8)));
          }
        } else {
          w = kf[h][s];
        }
        d[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), qf[s], d[h], 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) d[h][i] *= Q8 ? ks[h][i] * p.scale : p.scale;
    }
    if constexpr (Q8) {  // values from the registers into LDS
      vscale[0] = vs[0];
      vscale[1] = vs[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = i * 8 + (lane >> 3);
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int y = vr[i][j >> 1] >> (16 * (j & 1));
          w[j] = pack_bf2((float)(int8_t)y, (float)(int8_t)(y >> 8));
        }
        char* dst = sv + k * 256 + (((lane & 7) ^ (k & 7)) * 32);
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(dst + 16) = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
    if (live != ~0u) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = live >> (h * 16 + grp * 4 + i) & 1;
          d[h][i] = in ? d[h][i] : -INFINITY;
          if constexpr (Q8) vscale[h][i] = in ? vscale[h][i] : 0.f;
        }
      if constexpr (!Q8) {  // what lies behind the last position may be NaN, and 0 x it too
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll 1
        for (int k = grp; k < KB; k += 4)
          if (!(live >> k & 1)) *reinterpret_cast<uint4*>(sv + k * 256 + col * 16) = make_uint4(0, 0, 0, 0);
      }
    }
    if constexpr (!Q8) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the copies, the last loads but for an entry's
    read_v();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (BIG) {
      if (__builtin_expect(((b + W - b0) / W & 31) == 0, 0)) entry = entry_of(b + W);
    }
    load_k(b + W, b + W < end);
    load_v(b + W);
    if constexpr (!BIG) entry = entry_of(b + 2 * W);
    __builtin_amdgcn_sched_barrier(0);
    softmax(d);
    if constexpr (Q8) {
      d[0] *= vscale[0];
      d[1] *= vscale[1];
    }
    products(d);
  }
  if (!row_ok) {
    m = -INFINITY;
    l = 0.f;
  }

  if (writes) own.store(p, n, kvh);

  // the waves' results meet: each wave's outputs by its share of the largest maximum, summed by all threads
  l = xor32_sum(xor16_sum(l));
  if (lane == 0) sbad[wave] = bad;
  if (grp == 0) {
    sm[wave][col] = m;
    sl[wave][col] = l;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last loads into the region
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w][col]);
  const float f = m == -INFINITY ? 0.f : exp2_hw(m - M);
  if (col < t.rows) {
    float* dst = reinterpret_cast<float*>(sv) + col * LD + grp * 4;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      v4f o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = m == -INFINITY ? 0.f : f * acc[dt][i];  // a wave without keys has outputs of 0
      *reinterpret_cast<v4f*>(dst + dt * 16) = o;
    }
  }
  __syncthreads();
  int left_out = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) left_out |= sbad[w];
  const int dim = (tid & 31) * 4;  // 32 threads a row, 4 dimensions each
  for (int r = tid >> 5; r < t.rows; r += W * 2) {
    const int tk = single ? 0 : r / p.ratio;
    float MM = -INFINITY, L = 0.f;
    v4f O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) MM = fmaxf(MM, sm[w][r]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = sm[w][r];
      L += mw == -INFINITY ? sl[w][r] : exp2_hw(mw - MM) * sl[w][r];
      O += *reinterpret_cast<const v4f*>(region + w * REGION + (r * LD + dim) * 4);
    }
    const float size = (fabsf(O[0]) + fabsf(O[1])) + (fabsf(O[2]) + fabsf(O[3]));
    if (__builtin_expect((left_out || !(size <= TOP * L)) && row_ok && fabsf(L) < INFINITY, 0)) {
      v4f s = {0.f, 0.f, 0.f, 0.f};  // of the part's keys that the row sees: up to its own token, and those held
      for (int j = 0, to = start == 0 && end > 0 ? tk + 1 : 0; j < to; ++j) add_given(s, rowkv + p.KV * HD, p.ldq, j, dim);
      for (int j = max(start - nr, 0) * KB, to = min((int64_t)n, (int64_t)(end - nr) * KB); j < to; ++j)
        add_held<Q8>(s, p, row, kvh, j, dim);
#pragma unroll
      for (int i = 0; i < 4; ++i) O[i] = s[i] == 0.f ? within(O[i], L) : s[i];
    }
    const int64_t at = (int64_t)(t.first + tk) * p.H + kvh * p.ratio + (r - tk * p.ratio);
    if (nsp == 1) {
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = L == 0.f ? 0.f : O[i] / L;
      *reinterpret_cast<uint2*>(p.out + at * HD + dim) = make_uint2(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]));
    } else {
      float* part = p.part + (at * nsp + sp) * (HD + 2);  // parts are 520 bytes apart: 8-byte stores
      *reinterpret_cast<float2*>(part + dim) = make_float2(O[0], O[1]);
      *reinterpret_cast<float2*>(part + dim + 2) = make_float2(O[2], O[3]);
      if (dim == 0) *reinterpret_cast<float2*>(part + HD) = make_float2(MM, L);
    }
  }
}

}  // namespace cohere_paged
