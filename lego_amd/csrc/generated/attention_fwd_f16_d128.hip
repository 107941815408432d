// generated by lego_amd (python -m lego_amd.build) -- do not edit; edit the generator
//
// Attention, forward: O = softmax(score(Q K^T)) V over the keys that a query sees, f16, up to 128 head elements.
// One pass over the keys with a running maximum and sum.  A workgroup of 4 wavefronts owns 128 queries of a head, a wavefront 32 of them, one to a
// lane of each half: the scores are computed transposed, S^T = K Q^T, so that a query's scores lie in two lanes, its maximum and sum cost one exchange between
// the halves, and its factors are a lane's own.  P^T is the second operand of O^T = V^T P^T as it lies in the registers.  Tiles of 64 keys go from memory into LDS
// without passing registers, the next one while the present one is computed.
// Bound by the matrix cores and, level with them, by the vector unit, which has an exponential and five more instructions a score to issue and with a cap another exponential and a reciprocal: 2 x 32
// bf16 heads of 128, 8192 tokens, causal with prefixes, in 1.25 ms, 1.0 PFLOP/s of what is seen, both pipes 58 % busy; with a cap and 2 x 16 heads of 4096, 0.20 ms, 680 TFLOP/s, MFMA 32 %, vector 62 %.
// Wavefronts of 32 queries: LDS then delivers as many operands as the matrix cores take.  Two wavefronts a SIMD, one's softmax beside the other's products.
// P is rounded to the operands' type for the product with V, as is everything that MFMAs of 16-bit operands take; its sum is of the unrounded values, in fp32.
// Index expressions printed from LEGO layouts:
//   LDS tile   OrderBy(GenP((64, 16), row*16 + (chunk ^ key(row)))).TileBy([64, 16])
//   launch     Row(blocks, heads).inv(wg) = block, turn; head = OrderBy(Col(per_xcd, 8)).TileBy([per_xcd, 8])[Row(per_xcd, 8).inv(turn)]

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_args.h"

namespace {

typedef _Float16 elt_t;
typedef elt_t elt2 __attribute__((ext_vector_type(2)));
typedef elt_t elt8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v lds_short4;
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef int int4v __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr unsigned DC = 128;               // head elements that are computed; elements from the head's size on are zeros
constexpr unsigned KS = DC / 16, DB = DC / 32;   // MFMA steps along the head, blocks of 32 head elements
constexpr unsigned PITCH = 128;           // elements between the rows of a tile in LDS
constexpr unsigned ROWS = 64;                   // rows of a tile in LDS
constexpr unsigned TILE = ROWS * PITCH * 2;     // bytes
constexpr unsigned WAVES = 4;
constexpr unsigned COPIES = TILE / 1024 / WAVES; // memory->LDS instructions of a wave for a tile
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float16v mfma(elt8 a, elt8 b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float16v zeros()
{
  float16v z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.0f;
  return z;
}

// Two fp32 values as a pair of the operands' type, rounded to nearest.
__device__ __forceinline__ unsigned pack(float a, float b) { return __builtin_bit_cast(unsigned, __builtin_convertvector(float2v{a, b}, elt2)); }

// The sixteen values that a lane holds of a 32 x 32 accumulator block (column lane % 32; value r is row 8 (r / 4) + 4 (lane / 32) + r % 4)
// as the second operand of two MFMA steps over the block's rows.  The steps sum over the rows in the order in which a lane holds them:
// rows 16 s + 4 (lane / 32) + 0..3 and 16 s + 8 + 4 (lane / 32) + 0..3, and the first operand is read in that order (transposed()).
struct Operands { elt8 step[2]; };
__device__ __forceinline__ Operands as_operands(const float16v& x)
{
  Operands o;
#pragma unroll
  for (int s = 0; s < 2; ++s)
    o.step[s] = __builtin_bit_cast(elt8, u32x4{pack(x[8 * s], x[8 * s + 1]), pack(x[8 * s + 2], x[8 * s + 3]), pack(x[8 * s + 4], x[8 * s + 5]), pack(x[8 * s + 6], x[8 * s + 7])});
  return o;
}

// A tile in LDS: OrderBy(GenP((64, 16), row*16 + (chunk ^ key(row)))).TileBy([64, 16])
// with chunks of 16 bytes; the key makes both kinds of reads, 16 bytes of 16 rows in a row and transposing ones of 64 bytes of four rows, free of bank
// conflicts.  rows(): the first operand whose rows are the tile's (block of 32 rows, step of 16 head elements); transposed(): the first operand whose rows
// are 32 head elements (block `db`) and whose sum goes over 16 of the tile's rows, in as_operands()'s order.
struct Reader {
  unsigned row_at, tr_at;       // bytes within a tile
  __device__ __forceinline__ explicit Reader(unsigned lane)
  {
    const unsigned l32 = lane % 32, lhi = lane / 32, l16 = lane % 16, lgrp = lane / 16;
    row_at = 16 * (16*l32 + ((lhi) ^ (4*(l32 % 4) + ((l32)/(4)) % 4)));
    tr_at = 16 * (64*lhi + ((2*(lgrp % 2) + ((l16 % 4)/(2))) ^ (lhi + 4*((l16)/(4)))) + 16*((l16)/(4))) + 8 * (l16 % 2);
    (void)lgrp;
  }
  __device__ __forceinline__ elt8 rows(const char* tile, unsigned block, unsigned ks) const
  {
    return *reinterpret_cast<const elt8*>(tile + (row_at ^ (32 * ks)) + block * (32 * PITCH * 2));
  }
  // rows 16 * step .. of the tile
  __device__ __forceinline__ elt8 transposed(const char* tile, unsigned step, unsigned db) const
  {
    const char* const at = tile + step * (16 * PITCH * 2);
    const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + (tr_at ^ (64 * db))));
    const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + (tr_at ^ (64 * db) ^ 32) + 8 * PITCH * 2));
    return __builtin_bit_cast(elt8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// Fills a tile from rows of memory: lane l of copy `it` of wave w fetches the 16-byte chunk that belongs into slot 64 (WAVES it + w) + l.  Chunks past
// the head's size, rows past the last one and rows that `skip` names lie outside the descriptor, for which zeros are written (rows that share their memory with others, tokens
// no elements apart, are read as those).  Inline assembly, as the compiler orders
// every LDS read after all outstanding memory->LDS loads it knows of; a scalar write of M0 needs one wait state before the instruction that reads it.
constexpr unsigned kOutside = 0x80000000u;
struct Filler {
  const char* base;
  unsigned stride, bytes;       // of a row
  __device__ __forceinline__ Filler(const elt_t* base_, long long token, unsigned head)
      : base(reinterpret_cast<const char*>(base_)), stride(2 * (unsigned)token), bytes(2 * head) {}
  // from row `first` on, `rows` of which there are, at least one
  template <class Skip>
  __device__ __forceinline__ void operator()(unsigned lane, unsigned wave, unsigned first, unsigned rows, unsigned lds, const Skip& skip) const
  {
    const uintptr_t at = reinterpret_cast<uintptr_t>(base) + (size_t)first * stride;
    const u32x4 rsrc = {(unsigned)at, (unsigned)(at >> 32), (min(rows, ROWS) - 1) * stride + bytes, 0x00020000u};
    asm volatile("" : "+v"(lane));      // what follows from it is a few operations, and not to be kept in registers from tile to tile
    const unsigned row0 = 4*wave + ((lane)/(16)), chunk = ((lane % 16) ^ (wave + 4*((lane)/(16))));
    const unsigned offset = 16 * chunk < bytes ? row0 * stride + 16 * chunk : kOutside;
#pragma unroll
    for (unsigned it = 0; it < COPIES; ++it) {
      unsigned off = offset + it * ((ROWS / COPIES) * stride);
      if (skip(row0 + it * (ROWS / COPIES))) off = kOutside;
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc), "s"(lds + it * (WAVES * 1024)) : "memory", "m0");
    }
  }
};

// 64 words, a statistic or a number of each row, into LDS by one wavefront; rows past the last one read as zeros
__device__ __forceinline__ void fill_words(const void* base, unsigned rows, unsigned lane, unsigned lds)
{
  const uintptr_t at = reinterpret_cast<uintptr_t>(base);
  const u32x4 rsrc = {(unsigned)__builtin_amdgcn_readfirstlane((unsigned)at), (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(at >> 32)),
                      (unsigned)__builtin_amdgcn_readfirstlane(4 * min(rows, ROWS)), 0x00020000u};
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(4 * lane), "s"(rsrc), "s"(lds) : "memory", "m0");
}
// The scheduler's next instructions of a kind: it would read an operand from LDS only when the one before is used, and wait for each.
#define LEGO_MFMAS(N) __builtin_amdgcn_sched_group_barrier(0x008, N, 0)
#define LEGO_READS(N) __builtin_amdgcn_sched_group_barrier(0x100, N, 0)

__device__ __forceinline__ void wait_for_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Score function, in units of log2 e: what the exponential takes.  CAP: cap * tanh(scale q.k / cap) as cap (1 - 2 / (e^(2x) + 1)); its derivative by
// scale q.k is 1 - tanh^2.  BIAS: less slope * |distance|.
template <bool CAP>
__device__ __forceinline__ float score(float qk, const Scores& f)
{
  if (!CAP) return f.scale_log2 * qk;
  const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(f.cap_in * qk) + 1.0f);
  return __builtin_fmaf(-2.0f * f.cap_log2, r, f.cap_log2);
}

// For the backward pass with a cap: the score with `less`, which holds the cap too, added, and a quarter of its derivative by scale q.k.
template <bool CAP>
__device__ __forceinline__ float score(float qk, const Scores& f, float less, float& bend)
{
  const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(f.cap_in * qk) + 1.0f);
  bend = __builtin_fmaf(-r, r, r);
  return __builtin_fmaf(-2.0f * f.cap_log2, r, less);
}

// The head of a workgroup's turn among `all`: turns go round the XCDs, heads stay on one where that comes out even.
__device__ __forceinline__ unsigned place(unsigned turn, unsigned all)
{
  const unsigned per_xcd = all / 8;
  return all % 8 ? turn : per_xcd*(turn % 8) + ((turn)/(8));
}

// What of the keys the queries of a block see.  Query i stands at position i + shift; it sees keys below limit(i), of its own document.
struct Seen {
  int keys, shift, prefix;      // prefix: -1 where queries see all keys
  __device__ __forceinline__ int limit(int i) const { return prefix < 0 ? keys : min(keys, max(max(i + shift + 1, prefix), 0)); }
};

// Documents of a tile of 64 positions: the lowest and highest number (negative: padding).  Tiles that share no document with the others need no look at all; where
// both hold one and the same document, nothing has to be compared.
__device__ __forceinline__ bool apart(int2 a, int2 b) { return a.y < 0 || b.y < 0 || a.y < b.x || b.y < a.x; }
__device__ __forceinline__ bool same(int2 a, int2 b) { return a.x == a.y && b.x == b.y && a.x == b.x; }

// What a look at the documents of a tile (t) tells beside those of the workgroup's own rows.
constexpr unsigned kNeeded = 1, kCompare = 2, kPadded = 4;
__device__ __forceinline__ unsigned look_at(int2 t, int2 own) { return apart(t, own) ? 0u : same(t, own) ? kNeeded : kNeeded | kCompare | (t.x < 0 ? kPadded : 0u); }

// The tiles that a workgroup goes through, in order.  With documents 64 of them are looked at at a time, a lane each.
struct Step {
  unsigned tile;                // ~0u: none is left
  bool compare, padded;         // documents have to be compared; some rows of the tile are padding
  __device__ __forceinline__ bool there() const { return tile != ~0u; }
};
template <bool DOCS, class Look>
struct Walk {
  const Look& look;             // (tile) -> kNeeded, kCompare, kPadded
  unsigned lane, base, end;     // base: the next tile, or the first of the 64
  unsigned long long need = 0, compare = 0, padded = 0;
  __device__ __forceinline__ Walk(const Look& look_, unsigned lane_, unsigned begin, unsigned end_) : look(look_), lane(lane_), end(end_) { restart(begin); }
  __device__ __forceinline__ void restart(unsigned begin)
  {
    base = begin;
    if (DOCS) fetch();
  }
  __device__ __forceinline__ void fetch()
  {
    const unsigned tile = base + lane;
    const unsigned bits = tile < end ? look(tile) : 0u;
    need = __builtin_amdgcn_ballot_w64((bits & kNeeded) != 0);
    compare = __builtin_amdgcn_ballot_w64((bits & kCompare) != 0);
    padded = __builtin_amdgcn_ballot_w64((bits & kPadded) != 0);
  }
  __device__ __forceinline__ Step next()
  {
    if (!DOCS) return {base < end ? base++ : ~0u, false, false};
    while (need == 0) {
      if (base + 64 >= end) return {~0u, false, false};
      base += 64;
      fetch();
    }
    const unsigned at = (unsigned)__builtin_ctzll(need);
    need &= need - 1;
    return {base + at, (compare >> at & 1) != 0, (padded >> at & 1) != 0};
  }
};

// a value and the other half of the wavefront's, joined
typedef unsigned pair_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float across_max(float x)
{
  const pair_t p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
}
__device__ __forceinline__ float across_sum(float x)
{
  const pair_t p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(p.x) + __uint_as_float(p.y);
}

// Stores the columns of a wave's transposed result, blocks of 32 head elements: lane l holds element 8 (r / 4) + 4 (l / 32) + r % 4 of column l % 32.  Neighbouring
// groups of four change places between the halves, so that a lane stores 16 bytes at a time.
template <unsigned BLOCKS>
__device__ __forceinline__ void store_columns(const float16v (&acc)[BLOCKS], elt_t* row, unsigned lane, unsigned head, float factor)
{
  const unsigned lhi = lane / 32;
#pragma unroll
  for (unsigned db = 0; db < BLOCKS; ++db)
#pragma unroll
    for (unsigned g = 0; g < 2; ++g) {
      u32x2 w[2];
#pragma unroll
      for (unsigned e = 0; e < 2; ++e) {
        const unsigned lo = pack(factor * acc[db][8 * g + 2 * e], factor * acc[db][8 * g + 2 * e + 1]);
        const unsigned hi = pack(factor * acc[db][8 * g + 4 + 2 * e], factor * acc[db][8 * g + 4 + 2 * e + 1]);
        const pair_t both = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
        w[0][e] = both.x;
        w[1][e] = both.y;
      }
      const unsigned d = 32 * db + 16 * g + 8 * lhi;
      if (row && d < head) *reinterpret_cast<u32x4*>(row + d) = u32x4{w[0][0], w[0][1], w[1][0], w[1][1]};
    }
}

// A wave's sums into LDS, times a factor, and another wave's added to them.
template <unsigned BLOCKS>
__device__ __forceinline__ void put(const float16v (&acc)[BLOCKS], float4v* to, unsigned lane, float factor)
{
#pragma unroll
  for (unsigned db = 0; db < BLOCKS; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) to[(4 * db + g) * 64 + lane] = factor * float4v{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
}
template <unsigned BLOCKS>
__device__ __forceinline__ void add(float16v (&acc)[BLOCKS], float factor, const float4v* from, unsigned lane, float other)
{
#pragma unroll
  for (unsigned db = 0; db < BLOCKS; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4v x = from[(4 * db + g) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[db][4 * g + e] = factor * acc[db][4 * g + e] + other * x[e];
    }
}

}  // namespace

namespace {

// A maximum rises by less than this (in units of log2) without the sums being scaled down: P stays below 2^8, which changes no relative rounding.
constexpr float kLazy = 8.0f;
constexpr unsigned RING = 4;      // operands read ahead

template <bool CAP, bool BIAS, bool DOCS, unsigned HALVES>
__global__ void __launch_bounds__(64 * WAVES, 2) lego_attention_fwd_f16_d128_kernel(AttentionArgs a)
{
  constexpr unsigned RW = WAVES / HALVES, OWN = 32 * RW, SLOTS = 2 * HALVES;      // wavefronts of other rows than the others; queries of the workgroup; tiles in LDS
  __shared__ __attribute__((aligned(1024))) char lds[SLOTS * (2 * TILE + 256)];      // K and V, then the keys' documents
  const unsigned lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l32 = lane % 32, lhi = lane / 32, half = wave / RW;
  const unsigned blocks = (a.queries + OWN - 1) / OWN;
  const unsigned all_heads = a.heads * a.batch, turn = blockIdx.x / all_heads;
  const unsigned head = place(blockIdx.x % all_heads, all_heads);
  const unsigned h = head % a.heads, b = head / a.heads;
  const unsigned block = DOCS && a.order_queries ? __builtin_amdgcn_readfirstlane(a.order_queries[b * blocks + turn]) : blocks - 1 - turn;      // later queries may see more keys
  const unsigned hk = h / (a.heads / a.key_heads);
  const int q0 = (int)(OWN * block), q_last = min(q0 + (int)OWN, a.queries) - 1;
  const int w0 = q0 + 32 * (int)(wave % RW);                      // the wavefront's first query
  const int i = w0 + (int)l32;                              // the lane's query
  const Seen seen{a.keys, a.keys - a.queries, a.causal ? (a.prefix ? max(a.prefix[b], 0) : 0) : -1};
  const int limit = seen.limit(i), limit_w0 = seen.limit(w0), limit_w1 = seen.limit(min(w0 + 31, q_last));
  const int* const documents = DOCS ? a.documents + (size_t)b * a.keys : nullptr;
  const int2* const tiles = DOCS ? a.tiles + (size_t)b * ((a.keys + 63) / 64) : nullptr;

  // Without cap and slopes the running maximum is of the products themselves, and the scale comes in with the exponential; a negative one turns the queries round.
  constexpr bool RAW = !CAP && !BIAS;
  const float unit = RAW ? fabsf(a.scores.scale_log2) : 1.0f, lazy = kLazy / unit;
  // a lane's query as the second operand; queries past the last one are computed as the last one is
  elt8 qv[KS];
  {
    const elt_t* const row = static_cast<const elt_t*>(a.q) + (size_t)b * a.sq.batch + (size_t)min(i, a.queries - 1) * a.sq.token + (size_t)h * a.sq.head;
#pragma unroll
    for (unsigned ks = 0; ks < KS; ++ks) {
      const unsigned d = 16 * ks + 8 * lhi;
      qv[ks] = d < (unsigned)a.head ? *reinterpret_cast<const elt8*>(row + d) : elt8{};
      if (RAW && a.scores.scale_log2 < 0.0f) qv[ks] = -qv[ks];
    }
  }
  const int own_document = DOCS ? documents[min(i, a.queries - 1) + seen.shift] : 0;
  int2 own_tiles = {0, 0};
  if (DOCS) {
    own_tiles = tiles[(q0 + seen.shift) / 64];
    for (int t = (q0 + seen.shift) / 64 + 1; t <= (q_last + seen.shift) / 64; ++t) own_tiles = {min(own_tiles.x, tiles[t].x), max(own_tiles.y, tiles[t].y)};
  }
  const float slope = BIAS ? kLog2e * a.slopes[h] : 0.0f;

  const elt_t* const kb = static_cast<const elt_t*>(a.k) + (size_t)b * a.sk.batch + (size_t)hk * a.sk.head;
  const elt_t* const vb = static_cast<const elt_t*>(a.v) + (size_t)b * a.sv.batch + (size_t)hk * a.sv.head;
  const Filler fill_k(kb, a.sk.token, a.head), fill_v(vb, a.sv.token, a.head);
  const Reader read(lane);
  typedef __attribute__((address_space(3))) void* lds_ptr;
  const unsigned lds_at = (unsigned)(uintptr_t)(lds_ptr)lds + wave * 1024;
  const auto fill = [&](const Step& step, unsigned slot) {
    if (!step.there()) return;
    const unsigned first = 64 * step.tile, rows = a.keys - first;
    const unsigned at = lds_at + slot * (2 * TILE);
    if (DOCS && step.compare && wave == 0) fill_words(documents + first, rows, lane, lds_at + SLOTS * (2 * TILE) + slot * 256);
    // padding among the keys is read as zeros, whatever it holds
    const auto skip = [&](unsigned row) { return DOCS && step.padded && documents[min(first + row, (unsigned)a.keys - 1)] < 0; };
    fill_k(lane, wave, first, rows, at, skip);
    fill_v(lane, wave, first, rows, at + TILE, skip);
  };
  const auto look = [&](unsigned tile) { return look_at(tiles[tile], own_tiles); };

  float16v acc[DB];
#pragma unroll
  for (unsigned db = 0; db < DB; ++db) acc[db] = zeros();
  float most = -INFINITY, sum = 0.0f;      // of the lane's own keys; the halves agree on `most`
  Walk<DOCS, decltype(look)> walk(look, lane, 0, (unsigned)(seen.limit(q_last) + 63) / 64);
  // the walk's tiles in turn for the halves of the workgroup
  Step now[HALVES];
  unsigned buffer = 0;
#pragma unroll
  for (unsigned n = 0; n < HALVES; ++n) {
    now[n] = walk.next();
    fill(now[n], n);
  }
  while (now[0].there()) {
    Step next[HALVES];
#pragma unroll
    for (unsigned n = 0; n < HALVES; ++n) next[n] = walk.next();
    wait_for_copies();
    __syncthreads();                       // the tiles are there, and the other buffers are read no more
#pragma unroll
    for (unsigned n = 0; n < HALVES; ++n) fill(next[n], (buffer ^ HALVES) + n);
    const Step own = now[half ? HALVES - 1 : 0];
    const char* const kt = lds + (buffer + half) * (2 * TILE);
    const char* const vt = kt + TILE;
    const int first = (int)(64 * own.tile);
    const int* const document_s = reinterpret_cast<const int*>(lds + SLOTS * (2 * TILE) + (buffer + half) * 256);
    if ((HALVES == 1 || own.there()) && first < limit_w1) {
      float16v s[2] = {zeros(), zeros()};
#pragma unroll
      for (unsigned ks = 0; ks < KS; ++ks)
#pragma unroll
        for (unsigned kb2 = 0; kb2 < 2; ++kb2) s[kb2] = mfma(read.rows(kt, kb2, ks), qv[ks], s[kb2]);
      LEGO_READS(6);
#pragma unroll
      for (unsigned n = 0; n < KS - 3; ++n) {
        LEGO_MFMAS(2);
        LEGO_READS(2);
      }
      LEGO_MFMAS(6);
      __builtin_amdgcn_sched_barrier(0);
      elt8 ahead[RING];      // operands of the second products, on their way meanwhile
#pragma unroll
      for (unsigned j = 0; j < RING; ++j) ahead[j] = read.transposed(vt, j / DB, j % DB);
      __builtin_amdgcn_sched_barrier(0);
      // scores of keys first + 32 kb2 + 8 (r / 4) + 4 lhi + r % 4
      if (!RAW) {
        const float distance0 = (float)(i + seen.shift - first - 4 * (int)lhi);
#pragma unroll
        for (unsigned kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float x = score<CAP>(s[kb2][r], a.scores);
            if (BIAS) x -= slope * fabsf(distance0 - (float)(int)(32 * kb2 + 8 * (r / 4) + r % 4));
            s[kb2][r] = x;
          }
      }
      if (first + 64 > limit_w0) {
        int end = limit - first - 4 * (int)lhi;
        asm volatile("" : "+v"(end));      // a branch, and no comparisons ahead of it: most tiles have nothing to hide
#pragma unroll
        for (unsigned kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb2][r] = (int)(32 * kb2 + 8 * (r / 4) + r % 4) < end ? s[kb2][r] : -INFINITY;
      }
      if (DOCS && own.compare) {
#pragma unroll
        for (unsigned kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int4v d = *reinterpret_cast<const int4v*>(document_s + 32 * kb2 + 8 * g + 4 * lhi);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[kb2][4 * g + e] = own_document >= 0 && d[e] == own_document ? s[kb2][4 * g + e] : -INFINITY;
          }
      }
      float top = s[0][0];
#pragma unroll
      for (unsigned kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb2][r]);
      top = across_max(top);
      if (__builtin_amdgcn_ballot_w64(top > most + lazy) != 0) {
        // (-inf - -inf where a query has seen nothing yet: its sums are zeros, whatever they are multiplied by but not by NaN)
        const float risen = fmaxf(most, top), factor = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(unit * (most - risen));
        most = risen;
        sum *= factor;
#pragma unroll
        for (unsigned db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[db][r] *= factor;
      }
      const float base = most == -INFINITY ? 0.0f : unit * most;
      float sums[4] = {sum, 0.0f, 0.0f, 0.0f};
      const auto exponential = [&](unsigned kb2, int r) {
        s[kb2][r] = __builtin_amdgcn_exp2f(RAW ? __builtin_fmaf(unit, s[kb2][r], -base) : s[kb2][r] - base);
        sums[r % 4] += s[kb2][r];
      };
#pragma unroll
      for (int r = 0; r < 16; ++r) exponential(0, r);
      Operands p = as_operands(s[0]);
      __builtin_amdgcn_sched_barrier(0);
      // every product has its slot, with the operand of the one RING further on and a part of what the second half of the keys needs
#pragma unroll
      for (unsigned j = 0; j < 4 * DB; ++j) {
        if (j == 2 * DB) p = as_operands(s[1]);
        acc[j % DB] = mfma(ahead[j % RING], p.step[j / DB % 2], acc[j % DB]);
        if (j + RING < 4 * DB) ahead[j % RING] = read.transposed(vt, (j + RING) / DB, (j + RING) % DB);
        if (j < 2 * DB) {
#pragma unroll
          for (int r = (int)(16 * j / (2 * DB)); r < (int)(16 * (j + 1) / (2 * DB)); ++r) exponential(1, r);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }
#pragma unroll
    for (unsigned n = 0; n < HALVES; ++n) now[n] = next[n];
    buffer ^= HALVES;
  }
  sum = across_sum(sum);
  most *= unit;      // in units of log2 from here on
  if constexpr (HALVES == 2) {      // the second half's sums through LDS, in the tiles' place
    __syncthreads();
    float4v* const acc_s = reinterpret_cast<float4v*>(lds) + (wave % RW) * (64 * 4 * DB);
    float2* const stat_s = reinterpret_cast<float2*>(lds + RW * (64 * 16 * DB * 4)) + (wave % RW) * 64;
    static_assert(RW * (64 * 16 * DB * 4 + 64 * 8) <= SLOTS * 2 * TILE, "sums of the second half in the tiles' place");
    if (half) {
      put<DB>(acc, acc_s, lane, 1.0f);
      stat_s[lane] = float2{most, sum};
    }
    __syncthreads();
    if (half) return;
    const float2 o = stat_s[lane];
    const float top = fmaxf(most, o.x);
    const float f0 = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(most - top), f1 = o.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(o.x - top);
    most = top;
    sum = f0 * sum + f1 * o.y;
    add<DB>(acc, f0, acc_s, lane, f1);
  }
  const size_t row_at = (size_t)b * a.so.batch + (size_t)min(i, a.queries - 1) * a.so.token + (size_t)h * a.so.head;
  const float factor = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (unsigned db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] *= factor;
  store_columns<DB>(acc, i < a.queries ? static_cast<elt_t*>(a.o) + row_at : nullptr, lane, a.head, 1.0f);
  if (a.o_rest) {
#pragma unroll
    for (unsigned db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] -= static_cast<float>(static_cast<elt_t>(acc[db][r]));
    store_columns<DB>(acc, i < a.queries ? static_cast<elt_t*>(a.o_rest) + row_at : nullptr, lane, a.head, 1.0f);
  }
  if (i < a.queries && lhi == 0) a.lse[((size_t)b * a.heads + h) * a.queries + i] = sum == 0.0f ? -INFINITY : kLn2 * (most + __builtin_amdgcn_logf(sum));
}

}  // namespace

hipError_t lego_attention_fwd_f16_d128_launch(const AttentionArgs& a, hipStream_t stream)
{
  const auto launch = [&](auto whole, auto halves) {
    const unsigned own = a.halve_queries ? 16 * WAVES : 32 * WAVES, blocks = ((unsigned)a.queries + own - 1) / own * (unsigned)(a.heads * a.batch);
    hipLaunchKernelGGL(a.halve_queries ? halves : whole, dim3(blocks), dim3(64 * WAVES), 0, stream, a);
    return hipGetLastError();
  };
  if ((a.capped != 0) == true && (a.slopes != nullptr) == true)
    return a.documents ? launch(lego_attention_fwd_f16_d128_kernel<true, true, true, 1>, lego_attention_fwd_f16_d128_kernel<true, true, true, 2>)
                       : launch(lego_attention_fwd_f16_d128_kernel<true, true, false, 1>, lego_attention_fwd_f16_d128_kernel<true, true, false, 2>);
  if ((a.capped != 0) == true && (a.slopes != nullptr) == false)
    return a.documents ? launch(lego_attention_fwd_f16_d128_kernel<true, false, true, 1>, lego_attention_fwd_f16_d128_kernel<true, false, true, 2>)
                       : launch(lego_attention_fwd_f16_d128_kernel<true, false, false, 1>, lego_attention_fwd_f16_d128_kernel<true, false, false, 2>);
  if ((a.capped != 0) == false && (a.slopes != nullptr) == true)
    return a.documents ? launch(lego_attention_fwd_f16_d128_kernel<false, true, true, 1>, lego_attention_fwd_f16_d128_kernel<false, true, true, 2>)
                       : launch(lego_attention_fwd_f16_d128_kernel<false, true, false, 1>, lego_attention_fwd_f16_d128_kernel<false, true, false, 2>);
  if ((a.capped != 0) == false && (a.slopes != nullptr) == false)
    return a.documents ? launch(lego_attention_fwd_f16_d128_kernel<false, false, true, 1>, lego_attention_fwd_f16_d128_kernel<false, false, true, 2>)
                       : launch(lego_attention_fwd_f16_d128_kernel<false, false, false, 1>, lego_attention_fwd_f16_d128_kernel<false, false, false, 2>);
  return hipErrorInvalidValue;
}
