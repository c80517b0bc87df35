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
// A workgroup takes 16 query rows of a (sequence, key head) and one part of the keys; its waves take blocks of 32 keys in
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
constexpr int KB = 32;
typedef short v4s __attribute__((ext_vector_type(4)));

// what absent values are read from
__device__ __attribute__((aligned(16))) uint32_t zero_row[4];

// 16 bytes a lane from `offset` + `more` behind a buffer's start, zeros behind its end, into LDS at dst + 16 lane
DEVI void buffer_to_lds(__amdgpu_buffer_rsrc_t r, int offset, int more, char* dst) {
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass refuses the builtin
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LDS_AS void*)dst, 16, offset, more, 0, 0);
#endif
}

template <bool Q8, bool BIG, bool SPLIT, int W>
__global__ void __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2))) paged_rows_kernel(const PagedArgs p) {
  constexpr int LD = HD + 4, REGION = 16 * LD * 4;  // a wave's values (32 x 256 bytes), later its outputs
  static_assert(REGION >= KB * 256 && REGION % 256 == 0, "a wave's region");
  __shared__ __attribute__((aligned(256))) char region[W * REGION];
  __shared__ float sm[W][16], sl[W][16];
  __shared__ int sbad[W];
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), col = lane & 15, grp = lane >> 4;
  const int kvh = blockIdx.x % p.KV, sp = SPLIT ? blockIdx.y : 0, nsp = SPLIT ? p.parts : 1;
  const Tile t = tile_of<16>(p, blockIdx.x / p.KV);
  if (t.rows == 0) return;
  char* sv = region + wave * REGION;
  const int32_t* row = p.table + (int64_t)t.slot * p.W;
  const int P1 = (1 << p.shift) - 1;
  // the tile's blocks: of the chunk's tokens up to its last one, then of the positions held; wave w has every W-th
  const int last = p.starts ? (t.x0 + t.rows - 1) / p.ratio : 0, nr = last / KB + 1;
  int n = 0, nb = 0, start = 0, end = 0, b = wave;
  float rise = 0.f;
  bool row_ok = false;
  const int held = p.n[t.slot];  // on its way
  const auto bounds = [&]() {
    n = t.ok ? held : -1;
    row_ok = n >= 0;
    n = (int)min((int64_t)max(n, 0), (int64_t)p.W << p.shift);
    nb = row_ok ? nr + (n + KB - 1) / KB : 0;
    rise = rise_of((uint32_t)n + last + 1);
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
  const int b0 = b >= nr ? b : b + (nr - b + W - 1) / W * W;
  const auto entry_of = [&](int block) {
    const int64_t at = BIG ? (int64_t)(block + (lane >> 1) * W - nr) * KB + (lane & 1) * 16
                           : (int64_t)(block - nr) * KB + (lane & 31);
    return row[min(at >> p.shift, (int64_t)p.W - 1)];
  };
  int entry = entry_of(b0);

  // the lane's query row (the tile's last one repeated), its token and head
  const int x = t.x0 + min(col, t.rows - 1), tok = p.starts ? x / p.ratio : 0,
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
  const bool single = t.c == 1, first = single && b == 0;
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
        d[h][i] = exp2_hw(d[h][i] - to - rise);
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

  // the chunk's own blocks, as given; bad: of the wave's some values are infinite or NaN
  bool bad = false;
  if constexpr (!SPLIT) {
    if (!single) bounds();  // the weights' rise
  }
  for (; !single && b < (SPLIT ? min(end, nr) : nr); b += W) {
    const int j0 = b * KB;
    const auto own_row = [&](int j) { return rowkv + (int64_t)min(j, t.c - 1) * p.ldq; };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = i * 4 + grp;
      const char* at = reinterpret_cast<const char*>(own_row(j0 + k) + p.KV * HD) + (col ^ ((k & 7) * 2)) * 16;
      at = j0 + k < t.c ? at : reinterpret_cast<const char*>(zero_row);
      __builtin_amdgcn_global_load_lds(at, (LDS_AS void*)(sv + i * 4 * 256), 16, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    v4f d[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t* kp = own_row(j0 + h * 16 + col);
      d[h] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s)
        d[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const v8bf*>(kp + dims(s)), qf[s], d[h], 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) d[h][i] = j0 + h * 16 + grp * 4 + i <= tok ? d[h][i] * p.scale : -INFINITY;
    }
    __builtin_amdgcn_sched_barrier(0);
    softmax(d);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    read_v();
    bad |= leave_out(vf);
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
          at = there >> k & 1 ? at : reinterpret_cast<const char*>(zero_row);
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
    const float e = dot == -INFINITY ? 0.f : exp2_hw(dot - m - rise);
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
    const int xr = t.x0 + r, tk = p.starts ? xr / p.ratio : 0;
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
    const bool finite = fabsf(O[0]) < INFINITY && fabsf(O[1]) < INFINITY && fabsf(O[2]) < INFINITY && fabsf(O[3]) < INFINITY;
    if (__builtin_expect((left_out || !finite) && row_ok && fabsf(L) < INFINITY, 0)) {
      v4f s = {0.f, 0.f, 0.f, 0.f};  // of the part's keys that the row sees: up to its own token, and those held
      for (int j = start * KB, to = min(tk + 1, end * KB); j < to; ++j) add_given(s, rowkv + p.KV * HD, p.ldq, j, dim);
      for (int j = max(start - nr, 0) * KB, to = min((int64_t)n, (int64_t)(end - nr) * KB); j < to; ++j)
        add_held<Q8>(s, p, row, kvh, j, dim);
#pragma unroll
      for (int i = 0; i < 4; ++i) O[i] = s[i] == 0.f ? O[i] : s[i];
    }
    const int64_t at = (int64_t)(t.first + tk) * p.H + kvh * p.ratio + (xr - tk * p.ratio);
    if (nsp == 1) {
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = L == 0.f ? 0.f : mean_of(O[i], O[i] / L);
      *reinterpret_cast<uint2*>(p.out + at * HD + dim) = make_uint2(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]));
    } else {
      float* part = p.part + (at * nsp + sp) * (HD + 2);  // parts are 520 bytes apart: 8-byte stores
      *reinterpret_cast<float2*>(part + dim) = make_float2(O[0], O[1]);
      *reinterpret_cast<float2*>(part + dim + 2) = make_float2(O[2], O[3]);
      if (dim == 0) *reinterpret_cast<float2*>(part + HD) = make_float2(MM, L);
    }
  }
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
    if (grp + CG * i < nsp) o = add_part(lane_value(w, grp + CG * i), v[i], o);
  if constexpr (CG == 1) {
    out[head * HD + d] = f2bf(L == 0.f ? 0.f : mean_of(o, o / L));
  } else {
    __shared__ float so[CG][HD];
    so[grp][d] = o;
    __syncthreads();
    if (tid < HD) {
      float O = 0.f;
#pragma unroll
      for (int g = 0; g < CG; ++g) O += so[g][d];
      out[head * HD + d] = f2bf(L == 0.f ? 0.f : mean_of(O, O / L));
    }
  }
}

// The same behind the kernel of many rows, whose rows have parts of their own number: a wave a (row, head), which reads those
// parts alone that it has, N at a time.
template <int N>
__global__ void __launch_bounds__(256) paged_combine_many_kernel(const float* __restrict__ part, const int32_t* starts, int S,
                                                                 int64_t count, int H, int nsp, uint16_t* out) {
  const int lane = lane_id();
  const int64_t head = (int64_t)blockIdx.x * 4 + wave_id();
  if (head >= count) return;
  const float* base = part + head * nsp * (HD + 2);
  const float2 ml = *reinterpret_cast<const float2*>(base + min(lane, nsp - 1) * (HD + 2) + HD);
  const int r = (int)(head / H);
  if (starts && (r < starts[0] || r >= starts[S])) return;
  if (lane_value(ml.y, 0) < 0.f) return;  // one part, which wrote the outputs
  const bool in = lane < nsp && ml.x != -INFINITY;
  const float M = wave_max64(in ? ml.x : -INFINITY), w = in ? exp2_hw(ml.x - M) : 0.f;
  const float L = wave_sum64(lane < nsp ? (in ? w * ml.y : ml.y) : 0.f);
  float o0 = 0.f, o1 = 0.f;
  const uint64_t there = __ballot(in);
  const int last = 64 - __clzll(there);
  for (int i0 = 0; i0 < last; i0 += N) {
    float2 v[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = *reinterpret_cast<const float2*>(base + min(i0 + i, last - 1) * (HD + 2) + lane * 2);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i0 + i < last && there >> (i0 + i) & 1) {  // in the others nothing has to have been written
        const float wi = lane_value(w, i0 + i);
        o0 = add_part(wi, v[i].x, o0);
        o1 = add_part(wi, v[i].y, o1);
      }
  }
  *reinterpret_cast<uint32_t*>(out + head * HD + lane * 2) = L == 0.f ? 0u : pack_bf2(mean_of(o0, o0 / L), mean_of(o1, o1 / L));
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

template <bool Q8>
void launch_rows(const PagedArgs& p, dim3 grid, hipStream_t s) {
  constexpr int W = 4;
  if (p.shift >= 4 && p.parts > 1) paged_rows_kernel<Q8, true, true, W><<<grid, W * 64, 0, s>>>(p);
  else if (p.shift >= 4) paged_rows_kernel<Q8, true, false, W><<<grid, W * 64, 0, s>>>(p);
  else if (p.parts > 1) paged_rows_kernel<Q8, false, true, W><<<grid, W * 64, 0, s>>>(p);
  else paged_rows_kernel<Q8, false, false, W><<<grid, W * 64, 0, s>>>(p);
}

// whether a call goes to the kernel of 128 query rows a workgroup: more than 16 rows per sequence and key head on average
bool many_rows(int64_t rows, int64_t seqs, int64_t ratio) { return rows * ratio > 16 * seqs; }

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
  COHERE_REQUIRE(pages * kv_heads <= (int64_t(1) << 32) / P - 1, nm + ": more than 2^32 vectors");
  COHERE_REQUIRE(p.starts || rows == seqs, nm + ": a row per sequence, or starts");
  COHERE_REQUIRE(p.active && p.q && p.n && p.table && p.out && al(p.q, 16) && p.ldq % 8 == 0 && al(p.out, 16) &&
                     p.ldq >= (heads + 2 * kv_heads) * HD && p.ldq <= (1 << 24),
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
  const bool many = many_rows(rows, seqs, p.ratio) && p.scale != 0.f;
  if (many) launch_chunk(p, Q8, s);
  else launch_rows<Q8>(p, grid, s);
  const unsigned hs = (unsigned)(rows * heads);
  const unsigned hs4 = (hs + 3) / 4;
  if (many && splits > 4)
    paged_combine_many_kernel<16><<<hs4, 256, 0, s>>>(p.part, p.starts, p.S, hs, p.H, p.parts, p.out);
  else if (many && splits > 1)
    paged_combine_many_kernel<4><<<hs4, 256, 0, s>>>(p.part, p.starts, p.S, hs, p.H, p.parts, p.out);
  else if (splits > 4) paged_combine_kernel<4, 16><<<hs, 4 * HD, 0, s>>>(p.part, p.starts, p.S, p.H, p.parts, p.out);
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
  // Parts until the GPU is full, and then, where they stay long, until long and short sequences even out. Few-row kernel,
  // of 256 CUs x 2 workgroups: 1 x 8 heads over 64 K positions in 1, 16 and 64 parts 564, 50 and 44 us; 32 x 8 (x 4) over 1
  // .. 16 K, int8, 1, 2 and 8 parts 187, 152 and 126; 64 x 8 over up to 1 K 21, 2 parts 25. Kernel of 128 rows: 256 tokens
  // over 32 K 606, 16 parts 72, 32 63; 8 x 512 tokens over nothing 25, 2 parts 31.
  const int64_t ratio = heads / kv_heads;
  const bool many = many_rows(rows, seqs, ratio);
  const int64_t wgs = tiles_for(rows, seqs, ratio, many ? 128 : 16, rows != seqs) * kv_heads;
  const int64_t full = many ? 256 : 512, most = many ? 1024 : 2048, least = 192, longer = many ? 768 : 1024;
  if (many && wgs >= 192 && wgs <= 448) return 1;  // workgroups of two groups of waves
  int64_t n = 1;
  while (n < 64 && wgs * 2 * n <= most && T / (2 * n) >= (wgs * n < full ? least : longer)) n *= 2;
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
