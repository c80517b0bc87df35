// Beam search on a decoding step's logits, for gfx950. No counterpart in the reference, which decodes greedily
// (kernels/csrc/decoder_ops.cu:106-159). A group is one request's B beams (1 .. 16): slots g B .. g B + B - 1, best first.
//
//   dec_beam_select   the B best continuations over the beams and the vocabulary
//   dec_beam_reorder  every beam takes over its parent's history: table, tokens, states, the page in part filled
//   dec_beam_advance  the chosen tokens go into the slots' state; the next step's embeddings
//
// Selection. total[b][v] = score[b] + l[v] - max l - log sum exp(l - max l). Whether a candidate is in or out must not hang
// on roundings: the sums are in 64 bits, of exponentials that are right to 6e-11 of themselves, and candidates are compared
// in 64 bits. Within a beam the order is that of the logits (then of the indexes), so the first launch needs no sums to
// find a part's B best: it compares 16-bit numbers.
#include "cohere_hip.h"
#include "common.h"
#include "rows.h"

#include <algorithm>
#include <string>
#include <type_traits>

namespace {

using namespace cohere_rows;

constexpr int MAXB = 16, MK = 8;
constexpr double LOG2E64 = 1.4426950408889634074;

// a finite bf16 logit as a number of the same order, -0 as 0
DEVI uint32_t order_of(uint32_t h) {
  if (h == 0x8000u) h = 0;
  return h & 0x8000u ? h ^ 0xffffu : h | 0x8000u;
}
DEVI float logit_of(uint32_t o) { return __uint_as_float((o & 0x8000u ? o & 0x7fffu : o ^ 0xffffu) << 16); }

// a part's result: maximum, sum of exp(l - maximum), then B keys order << 32 | ~index of logits above -inf, best first (0:
// none). Where a beam has fewer than B of these, its other candidates, all of -inf, are the lowest indexes without a key.
struct Part {
  float m;
  uint32_t unused;
  double sum;
};
__host__ __device__ inline int64_t part_bytes(int B) { return (int64_t)sizeof(Part) + 8 * B; }

DEVI uint64_t wave_max_u64(uint64_t v) {
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t w = __shfl_xor(v, o, 64);
    v = w > v ? w : v;
  }
  return v;
}
DEVI double wave_sum_d(double v) {
  const auto moved = [](double x, auto ctrl) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, decltype(ctrl)::value, 0xF, 0xF, false),
                   hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), decltype(ctrl)::value, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  v += moved(v, std::integral_constant<int, DPP_XOR1>{});
  v += moved(v, std::integral_constant<int, DPP_XOR2>{});
  v += moved(v, std::integral_constant<int, DPP_ROR4>{});
  v += moved(v, std::integral_constant<int, DPP_ROR8>{});
  const auto lane = [&](int i) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), i) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, i));
  };
  return (lane(15) + lane(31)) + (lane(47) + lane(63));
}

// of the first n lanes' keys (0: none, the others different) the place of this lane's among them
DEVI int rank_of(uint64_t key, int n) {
  int r = 0;
  for (int i = 0; i < n; i += 4)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), i + k) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)key, i + k);
      r += o > key;
    }
  return r;
}

// exp(d) for d <= 0 to 6e-11 of itself, d below -700 or NaN as -700: 2^(y - round y) by the Chebyshev interpolant of 2^x on
// -1/2 .. 1/2 of degree 7, times a power of two, y = d log2 e. N at once, whose chains of products fill each other's waits.
template <int N>
DEVI void exp_64(double (&d)[N]) {
  const double magic = 6755399441055744.0;  // 1.5 2^52: the sum's last bit is 1
  constexpr double C[7] = {0.00015469729140704658, 0.0013333478480888061, 0.009618025613598036, 0.055504109063177154,
                           0.24022651213495422,    0.6931471805568341,    0.9999999999595622};
  double t[N], f[N];
#pragma unroll
  for (int e = 0; e < N; ++e) d[e] = fmax(d[e], -700.);
#pragma unroll
  for (int e = 0; e < N; ++e) t[e] = __builtin_fma(d[e], LOG2E64, magic);
#pragma unroll
  for (int e = 0; e < N; ++e) f[e] = __builtin_fma(d[e], LOG2E64, magic - t[e]);
#pragma unroll
  for (int e = 0; e < N; ++e) d[e] = 1.5303699001378845e-05;
#pragma unroll
  for (int i = 0; i < 7; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) d[e] = __builtin_fma(d[e], f[e], C[i]);
#pragma unroll
  for (int e = 0; e < N; ++e) d[e] = __builtin_amdgcn_ldexp(d[e], (int)__builtin_bit_cast(uint64_t, t[e]));
}
DEVI double exp_64(double d) {
  double x[1] = {d};
  exp_64(x);
  return x[0];
}

struct SelectArgs {
  const uint16_t* logits;
  int64_t ld;
  const int32_t* groups;
  const float* score;
  const uint8_t* finished;
  const int32_t* made;  // null: no norm
  const float* norm;
  int32_t* parent;
  int64_t* token;
  float* total;
  char* work;
  int n, G, B, V, N, pad, parts;
  int eos;  // -1: none
};

// A workgroup takes J * 2048 logits of a row: their maximum, the sum, and the B best. A wave finds its B best among few:
// T, the B-th largest of its lanes' maxima, is no larger than the B-th best, and hardly more than B logits reach it; these
// are ranked by counting, one a lane. Where more than 64 do (many equal logits, few lanes with a logit above -inf), the B
// best are taken one by one. What bounds it is the vector unit: of 25 instructions a logit 15 are the exponential (205 rows
// of 100008 in 27.8 us: 9.3 M instructions, which alone take 15.5; reading 41 MB takes 8).
template <int J>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(6))) beam_parts_kernel(const SelectArgs a) {
  __shared__ uint64_t cand[4][64], best[4][MAXB];
  __shared__ float smax[4];
  __shared__ double ssum[4];
  const int lane = lane_id(), wave = wave_id(), B = a.B;
  const int r = blockIdx.y, v0 = (blockIdx.x * 4 + wave) * (J * 512);
  const uint16_t* row = a.logits + (int64_t)r * a.ld;
  uint32_t w[J][4];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int v = v0 + (j * 64 + lane) * 8;
    const uint4 u = *reinterpret_cast<const uint4*>(row + min(v, a.V - 8));
    const bool in = v < a.V;
    w[j][0] = in ? u.x : 0xff80ff80u;
    w[j][1] = in ? u.y : 0xff80ff80u;
    w[j][2] = in ? u.z : 0xff80ff80u;
    w[j][3] = in ? u.w : 0xff80ff80u;
  }
  if constexpr (J > 1) {  // an ended beam's candidates are known without its logits; few logits are done before that is
    const int i = r / B, g = a.groups[i];
    if ((unsigned)g >= (unsigned)a.G) return;
    const int slot = g * B + (r - i * B);
    if (a.finished[slot] || !(a.score[slot] > -INFINITY)) return;
  }
  const auto logit = [&](int j, int k) { return __uint_as_float(k & 1 ? w[j][k >> 1] & 0xffff0000u : w[j][k >> 1] << 16); };
  float of[J], top = -INFINITY;  // maxima, which pass over NaN
  const auto maxima = [&]() {
    top = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      of[j] = -INFINITY;
#pragma unroll
      for (int k = 0; k < 8; ++k) of[j] = fmaxf(of[j], logit(j, k));
      top = fmaxf(top, of[j]);
    }
  };
  maxima();
  if (__builtin_expect(__any(top == INFINITY), 0)) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if ((w[j][k] & 0xffffu) == 0x7f80u) --w[j][k];
        if (w[j][k] >> 16 == 0x7f80u) w[j][k] -= 0x10000u;
      }
    maxima();
  }
  const auto key_of = [&](int j, int k) {
    return (uint64_t)order_of(__float_as_uint(logit(j, k)) >> 16) << 32 | ~(uint32_t)(v0 + (j * 64 + lane) * 8 + k);
  };
  // the B-th largest of the lanes' maxima
  float t = top, T = -INFINITY, m = -INFINITY;
  for (int k = 0; k < B; ++k) {
    T = wave_max64(t);
    if (k == 0) m = T;
    const uint64_t who = __ballot(t == T);
    if (lane == __ffsll((unsigned long long)who) - 1) t = -INFINITY;
  }
  T = fmaxf(T, -3.3895313892515355e38f);  // the lowest finite number
  if (lane < MAXB) best[wave][lane] = 0;
  int count = 0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (!__any(of[j] >= T)) continue;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool in = logit(j, k) >= T;
      const uint64_t who = __ballot(in);
      if (who) {
        const int at = count + __popcll(who & ((1ull << lane) - 1));
        if (in && at < 64) cand[wave][at] = key_of(j, k);
        count += __popcll(who);
      }
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own writes, read back by its other lanes
  if (__builtin_expect(count <= 64, 1)) {
    const uint64_t key = lane < count ? cand[wave][lane] : 0;
    const int place = rank_of(key, count);
    if (key && place < B) best[wave][place] = key;
  } else {
    uint64_t last = ~0ull;
    for (int k = 0; k < B; ++k) {
      uint64_t mine = 0;
#pragma unroll 1
      for (int j = 0; j < J; ++j) {
        uint32_t x[4] = {w[0][0], w[0][1], w[0][2], w[0][3]};
#pragma unroll
        for (int q = 1; q < J; ++q)
#pragma unroll
          for (int y = 0; y < 4; ++y) x[y] = q == j ? w[q][y] : x[y];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const uint32_t h = y & 1 ? x[y >> 1] >> 16 : x[y >> 1] & 0xffffu;
          const uint64_t key = (uint64_t)order_of(h) << 32 | ~(uint32_t)(v0 + (j * 64 + lane) * 8 + y);
          if (__uint_as_float(h << 16) > -INFINITY && key < last && key > mine) mine = key;
        }
      }
      last = wave_max_u64(mine);
      if (lane == 0) best[wave][k] = last;
      if (!last) break;
    }
  }
  double sum = 0.;
  if (m > -INFINITY) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        double d[2] = {(double)logit(j, k) - (double)m, (double)logit(j, k + 1) - (double)m};  // exact, or nearly so
        exp_64(d);
        sum += d[0];
        sum += d[1];
      }
    sum = wave_sum_d(sum);
  }
  if (lane == 0) {
    smax[wave] = m;
    ssum[wave] = sum;
  }
  __syncthreads();
  if (wave != 0) return;
  Part* out = reinterpret_cast<Part*>(a.work + ((int64_t)r * a.parts + blockIdx.x) * part_bytes(B));
  uint64_t* keys = reinterpret_cast<uint64_t*>(out + 1);
  const float M = fmaxf(fmaxf(smax[0], smax[1]), fmaxf(smax[2], smax[3])), mw = smax[lane & 3];
  sum = mw > -INFINITY ? ssum[lane & 3] * exp_64((double)mw - (double)M) : 0.;
  sum += __shfl_xor(sum, 1, 64);
  sum += __shfl_xor(sum, 2, 64);
  if (lane == 0) {
    out->m = M;
    out->sum = sum;
  }
  const uint64_t key = lane < 4 * B ? best[lane / B][lane % B] : 0;
  const int place = rank_of(key, 4 * B), have = __popcll(__ballot(key != 0));
  if (key && place < B) keys[place] = key;
  if (lane < B && lane >= have) keys[lane] = 0;
}

// Of a wave's keys, N a lane, the B best: the e-th best in lane e, lanes behind them 0. As above, by the logits' order alone
// until few are left.
template <int N>
DEVI uint64_t best_of(const uint64_t (&key)[N], int B, uint64_t* cand, uint64_t* best) {
  const int lane = lane_id();
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) top = fmaxf(top, (float)(uint32_t)(key[e] >> 32));  // 16 bits: exact
  float t = top, T = 0.f;
  for (int k = 0; k < B; ++k) {
    T = wave_max64(t);
    const uint64_t who = __ballot(t == T);
    if (lane == __ffsll((unsigned long long)who) - 1) t = 0.f;
  }
  T = fmaxf(T, 1.f);
  int count = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const bool in = (float)(uint32_t)(key[e] >> 32) >= T;
    const uint64_t who = __ballot(in);
    const int at = count + __popcll(who & ((1ull << lane) - 1));
    if (in && at < 64) cand[at] = key[e];
    count += __popcll(who);
  }
  if (lane < MAXB) best[lane] = 0;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own writes, read back by its other lanes
  if (__builtin_expect(count <= 64, 1)) {
    const uint64_t mine = lane < count ? cand[lane] : 0;
    const int place = rank_of(mine, count);
    if (mine && place < B) best[place] = mine;
  } else {
    uint64_t last = ~0ull;
    for (int k = 0; k < B; ++k) {
      uint64_t mine = 0;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (key[e] < last && key[e] > mine) mine = key[e];
      last = wave_max_u64(mine);
      if (lane == 0) best[k] = last;
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const uint64_t mine = lane < B ? best[lane] : 0;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read, before the next are written
  return mine;
}

// A workgroup takes a group: a wave a beam's parts (their sum, and of their B best each the beam's B best), then the B x B
// candidates are ranked by counting, a thread each.
__global__ void __launch_bounds__(64 * MAXB) beam_merge_kernel(const SelectArgs a) {
  __shared__ double srank[MAXB * MAXB], stotal[MAXB * MAXB];
  __shared__ uint64_t sid[MAXB * MAXB];
  __shared__ int splace[MAXB * MAXB];
  __shared__ uint64_t cand[MAXB][64], best[MAXB][MAXB];
  const int tid = threadIdx.x, lane = lane_id(), b = wave_id(), B = a.B, i = blockIdx.x;
  const char* at = a.work + ((int64_t)i * B + b) * a.parts * part_bytes(B);
  const uint32_t inverse = 0xffffffffu / B + 1;
  const auto key_at = [&](int k) {
    const int p = B == 1 ? k : (int)__umulhi(k, inverse);  // k / B: k B < 2^32
    return k < a.parts * B ? reinterpret_cast<const uint64_t*>(at + p * part_bytes(B) + sizeof(Part))[k - p * B] : 0;
  };
  // Read before it is known whether they count, and worked on while that is on its way: an ended beam's parts may hold
  // anything, and nothing is taken from them.
  Part q = {-INFINITY, 0, 0.};
  if (lane < a.parts) q = *reinterpret_cast<const Part*>(at + lane * part_bytes(B));
  uint64_t next[MK];
  const auto load = [&](int k0) {
#pragma unroll
    for (int e = 0; e < MK; ++e) next[e] = key_at(k0 + e * 64 + lane);
  };
  load(0);
  const int g = a.groups[i];
  if ((unsigned)g >= (unsigned)a.G) {
    if (tid < B) {
      a.parent[i * B + tid] = tid;
      a.token[i * B + tid] = a.pad;
      a.total[i * B + tid] = -INFINITY;
    }
    return;
  }
  const bool ended = a.finished[g * B + b] != 0;
  const double start = (double)a.score[g * B + b];
  const int made = a.norm ? a.made[g * B + b] : 0;
  float M = q.m;
  for (int p = lane + 64; p < a.parts; p += 64) M = fmaxf(M, reinterpret_cast<const Part*>(at + p * part_bytes(B))->m);
  M = wave_max64(M);
  double S = q.m > -INFINITY ? q.sum * exp_64((double)q.m - (double)M) : 0.;
  for (int p = lane + 64; p < a.parts; p += 64) {
    const Part* o = reinterpret_cast<const Part*>(at + p * part_bytes(B));
    S += o->m > -INFINITY ? o->sum * exp_64((double)o->m - (double)M) : 0.;
  }
  S = wave_sum_d(S);
  const float weight = a.norm ? a.norm[min(max(made + (ended ? 0 : 1), 0), a.N - 1)] : 1.f;
  // the best so far in lanes 0 .. B - 1, best first, and MK keys a lane more in each round; 64 keys or fewer are ranked as
  // they are
  uint64_t cur = 0;
  const int all_keys = a.parts * B;
  if (all_keys <= 64) {
    const int place = rank_of(next[0], all_keys);
    if (lane < MAXB) best[b][lane] = 0;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (next[0] && place < B) best[b][place] = next[0];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    cur = lane < B ? best[b][lane] : 0;
  } else {
    for (int k0 = 0; k0 < all_keys; k0 += 64 * MK) {
      uint64_t key[MK + 1];
#pragma unroll
      for (int e = 0; e < MK; ++e) key[e] = next[e];
      key[MK] = cur;
      if (k0 + 64 * MK < all_keys) load(k0 + 64 * MK);
      cur = best_of(key, B, cand[b], best[b]);
    }
  }
  double total = -INFINITY;
  int v = 0;
  if (!(start > -INFINITY)) {  // nothing but candidates of -inf (NaN counts as it): by their indexes
    v = lane;
  } else if (ended) {
    v = lane == 0 ? a.pad : lane - 1 + (lane - 1 >= a.pad);
    total = lane == 0 ? start : -INFINITY;
  } else {
    const int have = __popcll(__ballot(cur != 0));
    const bool nothing = have == 0 && a.eos >= 0;  // it ends here, at no cost
    v = (int)~(uint32_t)cur;
    if (cur) total = start + ((double)logit_of((uint32_t)(cur >> 32)) - (double)M - log(S));
    if (nothing) {
      v = lane == 0 ? a.eos : lane - 1 + (lane - 1 >= a.eos);
      total = lane == 0 ? start : -INFINITY;
    } else if (have < B) {  // the lowest indexes that have no key
      int free = 0;
      for (int u = 0, to = have; to < B; ++u) {
        if (__any(cur != 0 && v == u)) continue;
        if (lane == to) free = u;
        ++to;
      }
      if (lane >= have) v = free;
    }
  }
  if (lane < B) {
    const double rank = total * (double)weight;
    stotal[b * B + lane] = total == total ? total : -INFINITY;
    srank[b * B + lane] = rank == rank ? rank : -INFINITY;
    sid[b * B + lane] = (uint64_t)b << 32 | (uint32_t)v;
  }
  if (tid < B * B) splace[tid] = 0;
  __syncthreads();
  // a candidate's place: 64 / B threads, each counts the better ones in a share of all
  const int all = B * B, c = tid % all, shares = 64 / B, each = (all + shares - 1) / shares, first = tid / all * each;
  const double mine = srank[c];
  const uint64_t id = sid[c];
  int better = 0;
  for (int j = 0; j < each; j += 8)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int at = min(first + j + k, all - 1);
      const double other = srank[at];
      const bool counts = j + k < each && first + j + k < all;
      better += counts && (other > mine || (other == mine && sid[at] < id));
    }
  if (better) atomicAdd(&splace[c], better);
  __syncthreads();
  const int place = tid < B * B ? splace[tid] : B;
  if (place < B) {
    a.parent[i * B + place] = (int)(id >> 32);
    a.token[i * B + place] = (uint32_t)id;
    a.total[i * B + place] = (float)stotal[c];
  }
}

// Logits a workgroup over 2048: 8 where that makes a workgroup a CU still, so that a wave's search for its B best is paid
// for by more logits (4 x 16 beams, 64000 logits: 30 us, with 1 45; 64 x 4, 16384: 14.2 and 15.7). Below that 1, for the
// wave's own length (1 x 4, 16384: 9.7 us, with 8 12.3; 16 x 4: 11.1 and 13.5).
int select_j(int64_t rows, int64_t V) { return rows * ((V + 16383) / 16384) >= 256 ? 8 : 1; }
int64_t select_parts(int64_t rows, int64_t V) {
  const int64_t span = 2048 * select_j(rows, V);
  return (V + span - 1) / span;
}

// ---- reordering --------------------------------------------------------------------------------------------------------
struct ReorderArgs {
  const int32_t *groups, *parent, *n;
  const uint8_t* done;
  int32_t* table;
  int64_t* tokens;
  int32_t* states;
  char *k, *v;
  float *ks, *vs;
  int G, B, W, OUT, NS, L, pages, shift, KV, bytes;  // NS: states a row, bytes of a vector held
  int tables, columns;  // blocks of 256 columns: of the tables, of all rows (tables, tokens, states)
  uint32_t chunks;      // of 16 bytes of a page in part filled, all layers, keys and values
};

// The first `columns` blocks of a group move its rows of the tables, tokens and states, a thread a column of all B beams;
// the others move what the page in part filled holds, a thread 16 bytes of all B beams: read before any is written, so that
// nothing has to wait for anything. Four round trips one behind the other: group, its state, the pages, what they hold.
template <int MB>
__global__ void __launch_bounds__(256) beam_reorder_kernel(const ReorderArgs a) {
  const int i = blockIdx.y, g = a.groups[i], B = a.B, tid = threadIdx.x;
  int from[MB];
  bool moved = false;
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    const int q = a.parent[(int64_t)i * B + min(b, B - 1)];
    from[b] = b < B && (unsigned)q < (unsigned)B ? q : b;
    moved |= from[b] != b;
  }
  const bool there = (unsigned)g < (unsigned)a.G;
  const int64_t slot0 = (int64_t)(there ? g : 0) * B;
  const int n = max(a.n[slot0], 0);
  const bool done = a.done && a.done[there ? g : 0];
  if (!there || done || !moved) return;
  if ((int)blockIdx.x < a.columns) {
    const auto move = [&](auto* rows, int width, int c, int count) {
      using T = std::remove_reference_t<decltype(*rows)>;
      if (c >= count) return;
      T x[MB];
#pragma unroll
      for (int b = 0; b < MB; ++b) x[b] = rows[(slot0 + (b < B ? from[b] : 0)) * width + c];
#pragma unroll
      for (int b = 0; b < MB; ++b)
        if (b < B && from[b] != b) rows[(slot0 + b) * width + c] = x[b];
    };
    const int block = blockIdx.x, tokens = a.tokens ? (a.OUT + 255) / 256 : 0;
    if (block < a.tables) move(a.table, a.W, block * 256 + tid, min(n >> a.shift, a.W));
    else if (block < a.tables + tokens) move(a.tokens, a.OUT, (block - a.tables) * 256 + tid, min(n, a.OUT));
    else move(a.states, a.NS, (block - a.tables - tokens) * 256 + tid, a.NS);
    return;
  }
  const int filled = n & ((1 << a.shift) - 1), place = n >> a.shift;
  if (filled == 0 || place >= a.W) return;
  const uint32_t c = (blockIdx.x - a.columns) * 256 + tid;
  if (c >= a.chunks) return;
  const int part = (int)(c & (a.bytes / 16 - 1));  // 16 of bf16, 8 of int8
  uint32_t rest = c >> (a.bytes == 256 ? 4 : 3);
  const int off = (int)(rest & ((1 << a.shift) - 1));
  if (off >= filled) return;
  rest >>= a.shift;
  const uint32_t q = rest / (uint32_t)a.KV;
  const int h = (int)(rest - q * a.KV), kvi = (int)(q & 1), layer = (int)(q >> 1);
  char* pages = kvi ? a.v : a.k;
  float* scales = kvi ? a.vs : a.ks;
  int page[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) page[b] = b < B ? a.table[(slot0 + b) * a.W + place] : -1;
  const auto vec = [&](int pg) { return ((((int64_t)layer * a.pages + pg) * a.KV + h) << a.shift) + off; };
  // bit b: beam b's own page and its parent's are there, and two pages. The loads are made for every beam (of page 0
  // where the bit is 0), the stores by the bit.
  uint32_t go = 0;
  v4i x[MB];
  float sc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    int src = -1;
#pragma unroll
    for (int q = 0; q < MB; ++q) src = from[b] == q ? page[q] : src;
    const bool ok = from[b] != b && (unsigned)src < (unsigned)a.pages && (unsigned)page[b] < (unsigned)a.pages;
    go |= ok ? 1u << b : 0u;
    const int64_t at = vec(ok ? src : 0);
    x[b] = *reinterpret_cast<const v4i*>(pages + at * a.bytes + part * 16);
    sc[b] = scales ? scales[at] : 0.f;
  }
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    if (!(go >> b & 1)) continue;
    const int64_t at = vec(page[b]);
    *reinterpret_cast<v4i*>(pages + at * a.bytes + part * 16) = x[b];
    if (scales && part == 0) scales[at] = sc[b];
  }
}

// ---- the chosen tokens -------------------------------------------------------------------------------------------------
struct AdvanceArgs {
  const int32_t *groups, *parent;
  const int64_t* token;
  const float* total;
  int64_t* tok;
  int32_t *pos, *held;
  float* score;
  uint8_t *finished, *done, *flags;
  int32_t* made;
  const int32_t* limit;
  int64_t* out;
  int64_t eos;
  int G, B, OUT, dummy, by_length;
  const uint16_t *emb, *ptab, *w0, *b0, *w1, *b1;
  float eps0, eps1;
  uint16_t *x, *h;
  int width, tokens, positions;  // rows of emb and ptab
};

template <int VEC>
__global__ void __launch_bounds__(256) beam_advance_kernel(const AdvanceArgs a) {
  __shared__ int64_t stok[MAXB];
  __shared__ int spos[MAXB];
  const int i = blockIdx.x, lane = lane_id(), wave = wave_id(), B = a.B;
  const int g = a.groups[i];
  if ((unsigned)g >= (unsigned)a.G) return;
  const int64_t slot0 = (int64_t)g * B;
  if (wave == 0) {
    const bool live = g != a.dummy && !a.done[g], mine = lane < B;
    const int b = mine ? lane : 0;
    int64_t t = a.tok[slot0 + b];
    int p = a.pos[slot0 + b];
    if (live) {
      const int q = a.parent[(int64_t)i * B + b], from = (unsigned)q < (unsigned)B ? q : b;
      const bool was = a.finished[slot0 + from] != 0;
      const int made = a.made[slot0 + from] + (was ? 0 : 1);
      const float total = a.total[(int64_t)i * B + b];
      t = a.token[(int64_t)i * B + b];
      p = a.pos[slot0 + b] + 1;
      const bool fin = was || t == a.eos || !(total > -INFINITY);
      // the best beam of a group without norm stays the best once it has ended: the others' scores only fall
      const uint64_t all = __ballot(fin || !mine), first = __ballot(mine && lane == 0 && fin);
      const bool end = all == ~0ull || (!a.by_length && first) || p >= a.limit[g];
      // every lane's loads came before any lane's stores: one wave, in order
      if (mine) {
        a.finished[slot0 + b] = fin;
        a.made[slot0 + b] = made;
        a.score[slot0 + b] = total;
        a.tok[slot0 + b] = t;
        a.pos[slot0 + b] = p;
        if (a.held) a.held[slot0 + b] = p + 1;
        if ((unsigned)p < (unsigned)a.OUT) a.out[(slot0 + b) * a.OUT + p] = t;
        if (lane == 0 && end) {
          a.done[g] = 1;
          if (a.flags) a.flags[g] = 1;
        }
      }
    }
    if (mine) {
      stok[lane] = t;
      spos[lane] = p;
    }
  }
  __syncthreads();
  for (int b = wave; b < B; b += 4) {
    const int64_t t = stok[b];
    const int p = spos[b];
    const int64_t r = ((int64_t)i * B + b) * a.width;
    embed_row<VEC>(t >= 0 && t < a.tokens ? t : 0, min(max(p, 0), a.positions - 1), a.emb, a.ptab, a.w0, a.b0, a.eps0, a.w1,
                   a.b1, a.eps1, a.x + r, a.h + r, a.width, lane);
  }
}

bool al(const void* q, int n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; }
constexpr int64_t TOP = 0x7fffffff;

}  // namespace

// what a call of so many rows needs
static int64_t select_work(int64_t rows, int64_t V, int64_t beams) {
  return rows * select_parts(rows, V) * part_bytes((int)beams);
}

extern "C" int64_t cohere_dec_beam_select_work(int64_t rows, int64_t V, int64_t beams) {
  if (rows <= 0 || V <= 0 || beams < 1 || beams > MAXB) return 0;
  // the most rows whose workgroups take 2048 logits each: they have the more parts
  const int64_t most = 255 / ((V + 16383) / 16384);
  const int64_t need = select_work(rows, V, beams);
  return rows > most && most > 0 ? std::max(need, select_work(most, V, beams)) : need;
}

extern "C" int cohere_dec_beam_select_eos(const uint16_t* logits, int64_t ld, int64_t n, int64_t beams, int64_t V,
                                          const int32_t* groups, int64_t slots, const float* score,
                                          const uint8_t* finished, const int32_t* made, const float* norm,
                                          int64_t norm_len, int64_t pad, int64_t eos, int32_t* parent, int64_t* token,
                                          float* total, void* work, int64_t work_bytes, void* stream) {
  cohere::clear_error();
  COHERE_REQUIRE(eos >= -1 && eos < V, "dec_beam_select: the end token must be in the vocabulary (-1: none)");
  COHERE_REQUIRE(n >= 0 && beams >= 1 && beams <= MAXB && n * beams <= 65535 && slots > 0 && slots * beams <= TOP,
                 "dec_beam_select: 1 to 16 beams, at most 65535 rows");
  COHERE_REQUIRE(V >= beams && V % 8 == 0 && V < (int64_t(1) << 30) && ld >= V && ld % 8 == 0 && pad >= 0 && pad < V,
                 "dec_beam_select: a vocabulary of at least `beams`, a multiple of 8, rows 16 bytes aligned, pad in it");
  COHERE_REQUIRE(logits && groups && score && finished && parent && token && total && al(logits, 16),
                 "dec_beam_select: bad pointer");
  COHERE_REQUIRE(!norm || (made && norm_len > 0 && norm_len <= TOP), "dec_beam_select: norm needs made");
  if (n == 0) return 0;
  COHERE_REQUIRE(work && al(work, 8) && work_bytes >= select_work(n * beams, V, beams),
                 "dec_beam_select: work of dec_beam_select_work bytes");
  const int64_t rows = n * beams;
  const SelectArgs a{logits, ld, groups, score, finished, made, norm, parent, token, total, static_cast<char*>(work),
                     (int)n, (int)slots, (int)beams, (int)V, (int)norm_len, (int)pad, (int)select_parts(rows, V),
                     (int)eos};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)a.parts, (unsigned)rows);
  if (select_j(rows, V) == 8) beam_parts_kernel<8><<<grid, 256, 0, s>>>(a);
  else beam_parts_kernel<1><<<grid, 256, 0, s>>>(a);
  beam_merge_kernel<<<(unsigned)n, (unsigned)beams * 64, 0, s>>>(a);
  return cohere::check_launch("dec_beam_select");
}

extern "C" int cohere_dec_beam_select(const uint16_t* logits, int64_t ld, int64_t n, int64_t beams, int64_t V,
                                      const int32_t* groups, int64_t slots, const float* score, const uint8_t* finished,
                                      const int32_t* made, const float* norm, int64_t norm_len, int64_t pad,
                                      int32_t* parent, int64_t* token, float* total, void* work, int64_t work_bytes,
                                      void* stream) {
  return cohere_dec_beam_select_eos(logits, ld, n, beams, V, groups, slots, score, finished, made, norm, norm_len, pad, -1,
                                    parent, token, total, work, work_bytes, stream);
}

extern "C" int cohere_dec_beam_reorder(const int32_t* groups, int64_t n_groups, int64_t beams, const int32_t* parent,
                                       const int32_t* n, const uint8_t* done, int64_t slots, int32_t* table, int64_t width,
                                       int64_t* tokens, int64_t OUT, int32_t* states, int64_t n_states, void* k, void* v,
                                       float* ks, float* vs, int64_t L, int64_t pages, int64_t kv_heads, int64_t P,
                                       int32_t bits, void* stream) {
  cohere::clear_error();
  int shift = -1;
  for (int i = 0; i <= 8; ++i)
    if (P == (int64_t(1) << i)) shift = i;
  COHERE_REQUIRE(n_groups >= 0 && n_groups <= 65535 && beams >= 1 && beams <= MAXB && slots > 0 && slots * beams <= TOP,
                 "dec_beam_reorder: 1 to 16 beams, at most 65535 groups");
  COHERE_REQUIRE(groups && parent && n, "dec_beam_reorder: bad pointer");
  COHERE_REQUIRE((!tokens || (OUT > 0 && OUT <= TOP)) && (!states || (n_states > 0 && n_states <= TOP)),
                 "dec_beam_reorder: bad sizes");
  COHERE_REQUIRE(!table || (width > 0 && width <= TOP && shift >= 0),
                 "dec_beam_reorder: pages of a power of two up to 256 positions");
  COHERE_REQUIRE(!k == !v && (!k || (table && (bits == 16 || bits == 8) && L > 0 && pages > 0 && pages <= TOP &&
                                     kv_heads > 0 && al(k, 16) && al(v, 16) && (bits == 16 || (ks && vs)))),
                 "dec_beam_reorder: pages in 16 or 8 bits (with scales) need a table");
  if (n_groups == 0) return 0;
  const int bytes = bits == 16 ? 256 : 128;
  // a page of one position is never in part filled
  COHERE_REQUIRE(!k || kv_heads <= TOP / (2 * 256 * 16) / L, "dec_beam_reorder: too many layers and heads");
  const int64_t chunks = k && shift > 0 ? L * 2 * kv_heads * P * (bytes / 16) : 0;
  const auto blocks = [](int64_t of) { return (of + 255) / 256; };
  const int64_t tables = table ? blocks(width) : 0,
                columns = tables + (tokens ? blocks(OUT) : 0) + (states ? blocks(n_states) : 0);
  const ReorderArgs a{groups, parent, n, done, table, tokens, states, static_cast<char*>(k), static_cast<char*>(v),
                      bits == 8 ? ks : nullptr, bits == 8 ? vs : nullptr, (int)slots, (int)beams, (int)width, (int)OUT,
                      (int)n_states, (int)L, (int)pages, shift < 0 ? 0 : shift, (int)kv_heads, bytes,
                      (int)tables, (int)columns, (uint32_t)chunks};
  const dim3 grid((unsigned)(columns + blocks(chunks)), (unsigned)n_groups);
  if (grid.x == 0) return 0;  // nothing that could move
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (beams <= 4) beam_reorder_kernel<4><<<grid, 256, 0, s>>>(a);
  else if (beams <= 8) beam_reorder_kernel<8><<<grid, 256, 0, s>>>(a);
  else beam_reorder_kernel<16><<<grid, 256, 0, s>>>(a);
  return cohere::check_launch("dec_beam_reorder");
}

extern "C" int cohere_dec_beam_advance(const int32_t* groups, int64_t n_groups, int64_t beams, const int32_t* parent,
                                       const int64_t* token, const float* total, int64_t slots, int64_t dummy, int64_t* tok,
                                       int32_t* pos, int32_t* held, float* score, uint8_t* finished, int32_t* made,
                                       uint8_t* done, const int32_t* limit, int64_t* out, int64_t OUT, int64_t eos,
                                       int32_t by_length, const uint16_t* emb, int64_t vocabulary, const uint16_t* ptab,
                                       int64_t positions, const uint16_t* w0, const uint16_t* b0, float eps0, const uint16_t* w1,
                                       const uint16_t* b1, float eps1, uint16_t* x, uint16_t* h, int64_t width,
                                       uint8_t* flags_host, void* stream) {
  cohere::clear_error();
  COHERE_REQUIRE(n_groups >= 0 && n_groups <= TOP && beams >= 1 && beams <= MAXB && slots > 0 && slots * beams <= TOP &&
                     OUT > 0 && OUT <= TOP,
                 "dec_beam_advance: bad sizes (1 to 16 beams)");
  COHERE_REQUIRE(groups && parent && token && total && tok && pos && score && finished && made && done && limit && out,
                 "dec_beam_advance: bad pointer");
  COHERE_REQUIRE(width > 0 && width % 8 == 0 && width <= 2048 && vocabulary > 0 && vocabulary <= TOP && positions > 0 &&
                     positions <= TOP,
                 "dec_beam_advance: width must be a multiple of 8, at most 2048");
  COHERE_REQUIRE(emb && ptab && w0 && b0 && w1 && b1 && x && h && al(emb, 16) && al(ptab, 16) && al(x, 16) && al(h, 16) &&
                     al(w0, 16) && al(b0, 16) && al(w1, 16) && al(b1, 16),
                 "dec_beam_advance: bad embedding pointer");
  uint8_t* flags = nullptr;
  if (flags_host) {
    void* d = nullptr;
    COHERE_REQUIRE(hipHostGetDevicePointer(&d, flags_host, 0) == hipSuccess && d,
                   "dec_beam_advance: the end flags must be pinned host memory");
    flags = static_cast<uint8_t*>(d);
  }
  if (n_groups == 0) return 0;
  const AdvanceArgs a{groups, parent, token, total, tok, pos, held, score, finished, done, flags, made, limit, out, eos,
                      (int)slots, (int)beams, (int)OUT, (int)dummy, by_length, emb, ptab, w0, b0, w1, b1, eps0, eps1, x, h,
                      (int)width, (int)vocabulary, (int)positions};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define ADVANCE(V) beam_advance_kernel<V><<<(unsigned)n_groups, 256, 0, s>>>(a)
  switch ((width + 511) / 512) {
    case 1: ADVANCE(1); break;
    case 2: ADVANCE(2); break;
    case 3: ADVANCE(3); break;
    default: ADVANCE(4); break;
  }
#undef ADVANCE
  return cohere::check_launch("dec_beam_advance");
}
