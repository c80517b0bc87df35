// dec_attention_paged for chunks of many query rows (paged.h states the pages' form; dec_paged.hip has the few-row kernel
// and the entry points), for gfx950.
//
// A workgroup takes 128 query rows of a (sequence, key head), 32 a wave, and one part of the keys, 64 at a time: of the
// positions held, then of the chunk's own tokens. A tile's keys and values lie in LDS as bf16 (bf16 pages straight from
// memory, int8 ones converted on the way: codes are exact in bf16, their scales go into the scores and weights); two tiles,
// so that the next one's loads run under this one's products.
//   S^T = K Q^T on v_mfma_f32_32x32x16_bf16: queries in registers, a lane's result is 16 keys of query l % 32.
//   O^T = V^T P^T on the same instruction: the weights as they stand are its B operand (the order of the 16 keys of a
//   product is free, and taken as the lanes hold them), V^T comes through the transposing LDS read.
// Maximum, sum and outputs of a query stay in lanes l % 32 = query. The base of a query's weights is set 2^8 above its
// largest score and moves only when a score passes it, so that rescaling is rare and weights are at most 1.
// Rounded to fewer bits: the weights, to bf16 for the second product (off by at most 2^-9 of themselves; exact ones would
// need three products for one).
#include "paged.h"

namespace {

using namespace cohere_paged;

constexpr int KT = 64, TM = 128, W = 4;
constexpr float RISE = 8.f;

// what absent keys are read from
__device__ __attribute__((aligned(16))) uint4 zero_row[1];

typedef short v4s __attribute__((ext_vector_type(4)));

// 16 bytes a lane from src into LDS at dst + 16 lane. Written out, because for the builtin the compiler waits for all such
// copies in front of the next LDS read, whichever buffer that is of; the waits are tile_barrier's. No register is written,
// and the compiler's own counts of loads in flight stay safe: more are in flight than it counts, so it waits for more. m0 is
// used by nothing else in these kernels.
DEVI void copy_to_lds(const void* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory");
}
DEVI uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(LDS_AS const void*)p; }

// the wave's LDS operations done, and its loads
DEVI void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <bool Q8, bool BIG>
__global__ void __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
paged_chunk_kernel(const PagedArgs p) {
  __shared__ __attribute__((aligned(16))) char kbuf[2][KT * 256], vbuf[2][KT * 256];
  __shared__ __attribute__((aligned(16))) float sscale[Q8 ? 2 : 1][2][Q8 ? KT : 1];  // of a tile's keys and values
  const int lane = lane_id(), wave = wave_id(), col = lane & 31, half = lane >> 5;
  const int kvh = blockIdx.x % p.KV, sp = blockIdx.y, nsp = p.parts;
  const Tile t = tile_of<TM>(p, blockIdx.x / p.KV);
  if (t.rows == 0) return;
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
  const float scale = fabsf(p.scale);
  int n = t.ok ? p.n[t.slot] : -1;
  const bool row_ok = n >= 0;
  n = (int)min((int64_t)max(n, 0), (int64_t)p.W << p.shift);
  const int hi = row_ok ? (t.x0 + t.rows - 1) / p.ratio + 1 : 0;  // the chunk's tokens that the tile's last row sees
  const int np = (n + KT - 1) / KT, nb = np + (hi + KT - 1) / KT;
  const int chunk = (nb + nsp - 1) / nsp, start = min(nb, sp * chunk), end = min(nb, start + chunk);
  const int32_t* row = p.table + (int64_t)t.slot * p.W;
  const int P1 = (1 << p.shift) - 1;
  const uint16_t* rowkv = p.q + (int64_t)t.first * p.ldq + (p.H + kvh) * HD;

  // tile b: whether it is of the chunk's tokens, its first position, the table's entry of key `lane`, which keys there are
  const auto first_of = [&](int b) { return (b < np ? b : b - np) * KT; };
  const auto entry_of = [&](int b) { return b < np ? row[min(b * KT + lane, n - 1) >> p.shift] : 0; };
  const auto live_of = [&](int b, int entry) {
    const int at = first_of(b) + lane;
    return (uint64_t)__ballot(b < np ? at < n && (unsigned)entry < (unsigned)p.pages : at < hi);
  };
  // the vector of key kk of a page tile; every lane has to be active
  const auto vec_of = [&](int t0, int entry, int kk) {
    const int page = BIG ? __builtin_amdgcn_readlane(entry, wave * 16) : __shfl(entry, kk, 64);
    return (((int64_t)page * p.KV + kvh) << p.shift) + ((t0 + kk) & P1);
  };
  // int8 pages: 16 keys a wave on their way through registers
  v4i kr[2], vr[2];
  float sr;
  const auto issue = [&](int b, int entry, uint64_t live, int buf) {
    const int t0 = first_of(b);
    if (Q8 && b < np) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int kk = wave * 16 + i * 8 + (lane >> 3);
        const int64_t vec = vec_of(t0, entry, kk);
        const bool there = live >> kk & 1;
        const int64_t at = (there ? vec : 0) * HD + (lane & 7) * 16;
        kr[i] = *reinterpret_cast<const v4i*>(static_cast<const int8_t*>(p.k) + at);
        vr[i] = *reinterpret_cast<const v4i*>(static_cast<const int8_t*>(p.v) + at);
        if (!there) kr[i] = vr[i] = v4i{0, 0, 0, 0};
      }
      const int kk = wave * 16 + (lane & 15);
      const int64_t vec = vec_of(t0, entry, kk);
      const bool there = live >> kk & 1;
      sr = (lane < 16 ? p.ks : p.vs)[there ? vec : 0];
      sr = there ? sr : 0.f;
      return;
    }
    // one way for both kinds of tile: a branch would make the compiler wait for the loads in flight
    const bool own = Q8 || b >= np;
    const char* kb = own ? reinterpret_cast<const char*>(rowkv) : static_cast<const char*>(p.k);
    const char* vb = own ? reinterpret_cast<const char*>(rowkv + p.KV * HD) : static_cast<const char*>(p.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int kk = wave * 16 + i * 4 + (lane >> 4), ck = (lane & 15) ^ (kk & 15), cv = (lane & 15) ^ ((kk & 3) << 2);
      const int64_t held = Q8 ? 0 : vec_of(t0, entry, kk) * (2 * HD), given = (int64_t)(t0 + kk) * p.ldq * 2;
      const int64_t at = own ? given : held;
      const bool there = live >> kk & 1;
      const char* kp = there ? kb + at + ck * 16 : reinterpret_cast<const char*>(zero_row);
      const char* vp = there ? vb + at + cv * 16 : reinterpret_cast<const char*>(zero_row);
      copy_to_lds(kp, __builtin_amdgcn_readfirstlane(lds_address(kbuf[buf])) + (wave * 16 + i * 4) * 256);
      copy_to_lds(vp, __builtin_amdgcn_readfirstlane(lds_address(vbuf[buf])) + (wave * 16 + i * 4) * 256);
    }
    sr = 1.f;
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
            char* dst = (z ? vbuf : kbuf)[buf] + kk * 256;
#pragma unroll
            for (int c = 0; c < 2; ++c)
              *reinterpret_cast<uint4*>(dst + ((((lane & 7) * 2 + c) ^ sw) * 16)) =
                  make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
          }
        }
      }
      if (lane < 32) sscale[buf][lane >> 4][wave * 16 + (lane & 15)] = sr;
    }
  };

  v16f acc[4];  // dimensions 32 dt + 8 (r / 4) + 4 half + r % 4 of query col in acc[dt][r]
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
  float base = -INFINITY, l = 0.f;
  bool bad = false;  // some values of the chunk's own tokens are infinite or NaN

  int entry = 0;
  uint64_t live = 0, next = 0;
  if (start < end) {
    entry = entry_of(start);
    next = live_of(start, entry);
    issue(start, entry, next, 0);
    convert(start, 0);
    entry = start + 1 < end ? entry_of(start + 1) : 0;
  }
  for (int b = start; b < end; ++b) {
    const int buf = (b - start) & 1;
    asm volatile("" : "+v"(entry));  // waited for here, not behind the next tile's loads
    tile_barrier();                  // this tile is in LDS, and no wave reads the other buffer any more
    live = next;
    if (b + 1 < end) {
      next = live_of(b + 1, entry);
      issue(b + 1, entry, next, buf ^ 1);
      if (b + 2 < end) entry = entry_of(b + 2);
    }
    const int t0 = first_of(b);
    // rows of the chunk that no row of the wave's sees
    if (!(idle || (b >= np && t0 > tok1))) {
      const bool causal = b >= np && t0 + KT - 1 > tok0;
#pragma unroll
      for (int z = 0; z < 2; ++z) {  // 32 keys
        v16f s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
        const char* src = kbuf[buf] + (z * 32 + col) * 256;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const v8bf kf = *reinterpret_cast<const v8bf*>(src + (((c * 2 + half) ^ (col & 15)) * 16));
          s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[c], s, 0, 0, 0);
        }
        if constexpr (Q8) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const v4f k4 = *reinterpret_cast<const v4f*>(&sscale[buf][0][z * 32 + g * 8 + half * 4]);
#pragma unroll
            for (int k = 0; k < 4; ++k) s[4 * g + k] *= k4[k];
          }
        }
        if (causal || live != ~0ull) {
          // bit r of seen: key z 32 + 8 (r / 4) + 4 half + r % 4 is there, and not behind the query's token
          const uint32_t there = (uint32_t)(live >> (z * 32)) >> (half * 4);
          const int upto = causal ? tok - t0 - z * 32 - half * 4 : 32;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int kk = (r >> 2) * 8 + (r & 3);
            s[r] = (there >> kk & 1) && kk <= upto ? s[r] : -INFINITY;
          }
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx = xor32_max(mx) * scale;
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
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = exp2_hw(__builtin_fmaf(s[r], scale, off));
          l += s[r];
        }
        if constexpr (Q8) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const v4f v4 = *reinterpret_cast<const v4f*>(&sscale[buf][1][z * 32 + g * 8 + half * 4]);
#pragma unroll
            for (int k = 0; k < 4; ++k) s[4 * g + k] *= v4[k];
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // 16 keys a product
          v4i w;
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = (int)pack_bf2(s[u * 8 + 2 * k], s[u * 8 + 2 * k + 1]);
          const v8bf pf = __builtin_bit_cast(v8bf, w);
          const int k0 = z * 32 + u * 16;
          v8bf vf[4];
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) {
            // keys k0 + 4 half + (lane % 16) / 4 (and 8 on), dimensions 32 dt + 16 (lane / 16 % 2) + 4 (lane % 4) ..
            const int kk = half * 4 + ((lane & 15) >> 2), c = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
            const char* src = vbuf[buf] + (k0 + kk) * 256 + ((c ^ ((kk & 3) << 2)) * 16) + (lane & 1) * 8;
            const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS v4s*)src);
            const v4s d = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS v4s*)(src + 8 * 256));
            vf[dt] = __builtin_bit_cast(v8bf, __builtin_shufflevector(a, d, 0, 1, 2, 3, 4, 5, 6, 7));
          }
          if (causal) bad |= leave_out(vf);
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[dt], pf, acc[dt], 0, 0, 0);
        }
      }
    }
    if (b + 1 < end) convert(b + 1, buf ^ 1);
  }
  l = xor32_sum(l);
  if (wave * 32 + col < t.rows) {
    if (__builtin_expect(bad, 0)) {
      // of the part's tiles of the chunk's tokens those that some row of the wave's does not see whole
      const int from = max((tok0 + 1) / KT, max(start - np, 0)) * KT, to = min(tok + 1, (end - np) * KT);
#pragma unroll 1
      for (int j = from; j < to; ++j) {
        const uint16_t* src = rowkv + (int64_t)j * p.ldq + p.KV * HD + half * 4;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[dt][4 * g + k] += not_finite(src[dt * 32 + g * 8 + k]);
      }
    }
    const int64_t at = (int64_t)(t.first + tok) * p.H + head;
    if (nsp == 1) {
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
  }
  if (sp == 0 && row_ok) append<Q8, W>(p, t, n, kvh, TM);
}

}  // namespace

namespace cohere_paged {

int64_t chunk_workgroups(const PagedArgs& p) {
  return tiles_for(p.R, p.S, p.ratio, TM, p.starts != nullptr) * p.KV;
}

void launch_chunk(const PagedArgs& p, bool q8, hipStream_t s) {
  const dim3 grid((unsigned)chunk_workgroups(p), (unsigned)p.parts);
  if (q8 && p.shift >= 4) paged_chunk_kernel<true, true><<<grid, W * 64, 0, s>>>(p);
  else if (q8) paged_chunk_kernel<true, false><<<grid, W * 64, 0, s>>>(p);
  else if (p.shift >= 4) paged_chunk_kernel<false, true><<<grid, W * 64, 0, s>>>(p);
  else paged_chunk_kernel<false, false><<<grid, W * 64, 0, s>>>(p);
}

}  // namespace cohere_paged
