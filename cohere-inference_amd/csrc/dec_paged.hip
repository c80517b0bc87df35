// Attention of new tokens over caches held in pages (paged.h states the form), and reading pages back, for gfx950. No
// counterpart in the reference, whose caches are one stretch per slot (kernels/csrc/decoder_ops.cu, dec_attn.cuh).
//
//   dec_attention_paged  softmax(q k^T scale) v of a chunk of new tokens per sequence: token j, at position n + j, attends
//                        to the n positions held in pages and to the chunk's tokens 0 .. j as given, whose keys and values
//                        go into the pages at n ..
//   dec_gather_paged     keys and values of (slot, position) pairs as bf16 rows
#include "cohere_hip.h"
#include "paged_rows.h"

#include <string>
#include <type_traits>

namespace {

using namespace cohere_paged;

// ---- attention of a token per sequence --------------------------------------------------------------------------------
template <bool Q8, bool BIG, bool SPLIT, int W>
__global__ void __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2))) paged_rows_kernel(const PagedArgs p) {
  __shared__ FewRows<W> lds;
  const int i = blockIdx.x / p.KV;
  Tile t;
  t.first = i;
  t.c = 1;
  t.x0 = 0;
  t.rows = p.ratio;
  t.slot = p.active[i];
  t.ok = (unsigned)t.slot < (unsigned)p.slots;
  t.slot = t.ok ? t.slot : 0;
  few_rows<Q8, BIG, SPLIT, W>(p, t, blockIdx.x % p.KV, lds);
}

// The parts of a (row, head): every wave finds the maximum, the parts' weights (lane s part s's) and the sum; CG groups of 128
// threads sum N parts each, all their loads in flight at once.
template <int CG, int N>
__global__ void __launch_bounds__(CG * HD) paged_combine_kernel(const float* __restrict__ part, int nsp, uint16_t* out) {
  const int64_t head = blockIdx.x;
  const int tid = threadIdx.x, lane = lane_id(), d = tid & (HD - 1), grp = wave_id() >> 1;
  const float* base = part + head * nsp * (HD + 2);
  const float* mine = base + min(lane, nsp - 1) * (HD + 2) + HD;
  const float ms = mine[0], ls = mine[1];
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = base[min(grp + CG * i, nsp - 1) * (HD + 2) + d];
  const float M = wave_max64(lane < nsp ? ms : -INFINITY);
  const float w = lane < nsp && ms != -INFINITY ? exp2_hw(ms - M) : 0.f;
  const float L = wave_sum64(lane < nsp ? (ms == -INFINITY ? ls : w * ls) : 0.f);
  float o = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (grp + CG * i < nsp) o = __builtin_fmaf(lane_value(w, grp + CG * i), v[i], o);
  if (__builtin_expect(!(fabsf(o) < INFINITY), 0)) {
    o = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (grp + CG * i < nsp) o = add_part(lane_value(w, grp + CG * i), v[i], o);
  }
  if constexpr (CG == 1) {
    out[head * HD + d] = f2bf(L == 0.f ? 0.f : within(o, L) / L);
  } else {
    __shared__ float so[CG][HD];
    so[grp][d] = o;
    __syncthreads();
    if (tid < HD) {
      float O = 0.f;
#pragma unroll
      for (int g = 0; g < CG; ++g) O += so[g][d];
      out[head * HD + d] = f2bf(L == 0.f ? 0.f : within(O, L) / L);
    }
  }
}

// The same behind the kernel of chunks, for rows of the sequences, which may have parts of their own number: a wave a (row,
// head), which reads those parts alone that it has, N at a time.
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
  const auto join = [&](auto add) {
    o0 = o1 = 0.f;
    for (int i0 = 0; i0 < last; i0 += N) {
      float2 v[N];
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = *reinterpret_cast<const float2*>(base + min(i0 + i, last - 1) * (HD + 2) + lane * 2);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i0 + i < last && there >> (i0 + i) & 1) {  // in the others nothing has to have been written
          const float wi = lane_value(w, i0 + i);
          o0 = add(wi, v[i].x, o0);
          o1 = add(wi, v[i].y, o1);
        }
    }
  };
  join([](float a, float x, float o) { return __builtin_fmaf(a, x, o); });
  if (__builtin_expect(__any(!(fabsf(o0) + fabsf(o1) < INFINITY)), 0)) join(add_part);
  *reinterpret_cast<uint32_t*>(out + head * HD + lane * 2) = L == 0.f ? 0u : pack_bf2(within(o0, L) / L, within(o1, L) / L);
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
  // Which kernel a sequence goes to hangs on it alone, and so do its bits: up to 16 query rows a key head few_rows, in a
  // kernel of its own where every sequence is one token, else in the chunks' kernel, which finds out how long each is.
  const bool chunks = p.starts || p.ratio > FEW;
  const int64_t wgs = chunks ? chunk_workgroups(p) : seqs * kv_heads;
  COHERE_REQUIRE(wgs <= TOP && rows * heads <= TOP, nm + ": too many rows and heads");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (chunks) launch_chunk(p, Q8, s);
  else launch_rows<Q8>(p, dim3((unsigned)wgs, (unsigned)splits), s);
  const unsigned hs = (unsigned)(rows * heads), hs4 = (hs + 3) / 4;
  if (chunks && splits > 4)
    paged_combine_many_kernel<16><<<hs4, 256, 0, s>>>(p.part, p.starts, p.S, hs, p.H, p.parts, p.out);
  else if (chunks && splits > 2)
    paged_combine_many_kernel<4><<<hs4, 256, 0, s>>>(p.part, p.starts, p.S, hs, p.H, p.parts, p.out);
  else if (!chunks && splits > 4) paged_combine_kernel<4, 16><<<hs, 4 * HD, 0, s>>>(p.part, p.parts, p.out);
  else if (!chunks && splits > 1) paged_combine_kernel<1, 4><<<hs, HD, 0, s>>>(p.part, p.parts, p.out);
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
  const int64_t ratio = heads / kv_heads;
  const bool many = rows * ratio > FEW * seqs;
  const int64_t wgs = tiles_for(rows, seqs, ratio, many ? 128 : FEW, rows != seqs) * kv_heads;
  int64_t n = 1, full = 512, most = 2048, longer = 1024;
  if (many) {
    // Two parts are one workgroup's groups of waves. Chunks of 128 tokens over nothing, 64 to 256 workgroups, in 1 and 2 parts
    // 11.0 to 12.1 and 12.8 to 13.7 us, 320 15.8 and 24; of 512 tokens 25 and 22; of 100 over 2 K, 224, 336 and 456
    // workgroups, 49 and 42, 64 and 46, 77 and 92; 168, 2 and 4 parts 41 and 35, 224 42 and 49.
    if (T < 384 || wgs > 448) return 1;
    if (T < 768 || wgs >= 192) return 2;
    n = 4; full = 256; most = 1024; longer = 768;
  }
  // Parts until the GPU is full, and then, where they stay long, until long and short sequences even out. Few-row kernel,
  // of 256 CUs x 2 workgroups: 1 x 8 heads over 64 K positions in 1, 16 and 64 parts 564, 50 and 44 us; 32 x 8 (x 4) over 1
  // .. 16 K, int8, 1, 2 and 8 parts 187, 152 and 126; 64 x 8 over up to 1 K 21, 2 parts 25. Kernel of 128 rows: 256 tokens
  // over 32 K 606, 16 parts 72, 32 63; 6 x 100 over 2 K, 1, 2 and 4 parts 48, 41 and 29.
  while (n < 64 && wgs * 2 * n <= most && T / (2 * n) >= (wgs * n < full ? 192 : longer)) n *= 2;
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
