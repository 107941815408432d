// generated by lego_amd (python -m lego_amd.build) -- do not edit; edit the generator
//
// Attention, backward: dQ, dK and dV from dO, bf16, up to 128 head elements.
//   P = exp(score(Q K^T) - lse),  dS = P * (dO V^T - delta),  dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K
// with delta and lse of the rows.  Two kernels, each of which owns what it writes, so that no sum is shared and none depends on an order of arrival: one
// goes through the queries for 128 keys and sums dK and dV, four products a tile, the other through the keys for 128 queries and sums dQ, three.  A single
// kernel would need five products and not seven, and would add dQ up through memory.
// A lane holds one column of everything, a key in the first kernel and a query in the second; P and dS are the second operands of their products as they lie in the registers.
// P and dS are rounded to the operands' type, which their products take; the sums are fp32.
// Bound by issue and by LDS, whose operands for 32 rows a wavefront keep the matrix cores no busier than it is itself: 2 x 16 bf16 heads of 128 to 4, 4096 tokens, causal and capped, dK and dV in 380 us
// (MFMA 35 % busy, vector unit 41 %), dQ in 225 (49 %, 66 %).  Measured and not taken: 64 keys a wavefront, half the LDS reads, 518 us and not 382 for want of registers; sums in the accumulation
// registers at one wavefront a SIMD, slower still.
// Index expressions printed from LEGO layouts:
//   LDS tile   OrderBy(GenP((64, 16), row*16 + (chunk ^ key(row)))).TileBy([64, 16])
//   launch     Row(blocks, heads).inv(wg) = block, turn; head = OrderBy(Col(per_xcd, 8)).TileBy([per_xcd, 8])[Row(per_xcd, 8).inv(turn)]

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_args.h"

namespace {

typedef __bf16 elt_t;
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

__device__ __forceinline__ float16v mfma(elt8 a, elt8 b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

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

constexpr float kUnshift = 1.0f / (1 << 0);      // P is held as P / kUnshift
template <unsigned V> struct Constant { static constexpr unsigned value = V; };
constexpr unsigned RING = 3;      // operands read ahead

template <bool CAP, bool BIAS, bool DOCS, unsigned HALVES>
__global__ void __launch_bounds__(64 * WAVES, 2) lego_attention_dkv_bf16_d128_kernel(AttentionArgs a)
{
  constexpr unsigned RW = WAVES / HALVES, OWN = 32 * RW, SLOTS = 2 * HALVES;      // wavefronts of other keys than the others; keys of the workgroup; tiles in LDS
  __shared__ __attribute__((aligned(1024))) char lds[SLOTS * (2 * TILE + 768)];      // Q and dO, then lse, delta and documents
  const unsigned lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l32 = lane % 32, lhi = lane / 32, half = wave / RW;
  const unsigned blocks = (a.keys + OWN - 1) / OWN, group = a.heads / a.key_heads, parts = group / a.heads_per_part;
  const unsigned all_parts = parts * a.key_heads * a.batch, turn = blockIdx.x / all_parts;
  const unsigned at_part = place(blockIdx.x % all_parts, all_parts), part = at_part % parts, hk = at_part / parts % a.key_heads, b = at_part / parts / a.key_heads;
  const unsigned block = DOCS && a.order_keys ? __builtin_amdgcn_readfirstlane(a.order_keys[b * blocks + turn]) : turn;      // earlier keys may be seen by more queries
  const int k0 = (int)(OWN * block), k_last = min(k0 + (int)OWN, a.keys) - 1;
  const int w0 = k0 + (int)(32 * (wave % RW)), key = w0 + (int)l32;
  const int shift = a.keys - a.queries, prefix = a.causal ? (a.prefix ? max(a.prefix[b], 0) : 0) : a.keys;
  const int first_row = a.causal && prefix == 0 ? -shift : 0;      // that sees a key
  // a query sees a key from this row on
  const auto from = [&](int j) { return j < prefix ? -(1 << 30) : j - shift; };
  const int from_key = from(key), from_w0 = from(w0), from_w1 = from(min(w0 + 31, a.keys - 1));
  const int* const documents = DOCS ? a.documents + (size_t)b * a.keys : nullptr;
  const int2* const tiles = DOCS ? a.tiles + (size_t)b * ((a.keys + 63) / 64) : nullptr;

  const int own_document = DOCS ? documents[min(key, a.keys - 1)] : 0;
  elt8 kv[KS], vv[KS];      // a key of padding is zeros, whatever it holds
  {
    const int j = min(key, a.keys - 1);
    const elt_t* const krow = static_cast<const elt_t*>(a.k) + (size_t)b * a.sk.batch + (size_t)j * a.sk.token + (size_t)hk * a.sk.head;
    const elt_t* const vrow = static_cast<const elt_t*>(a.v) + (size_t)b * a.sv.batch + (size_t)j * a.sv.token + (size_t)hk * a.sv.head;
#pragma unroll
    for (unsigned ks = 0; ks < KS; ++ks) {
      const unsigned d = 16 * ks + 8 * lhi;
      kv[ks] = d < (unsigned)a.head && own_document >= 0 ? *reinterpret_cast<const elt8*>(krow + d) : elt8{};
      vv[ks] = d < (unsigned)a.head && own_document >= 0 ? *reinterpret_cast<const elt8*>(vrow + d) : elt8{};
    }
  }
  int2 own_tiles = {0, 0};
  if (DOCS) {
    own_tiles = tiles[k0 / 64];
    for (int t = k0 / 64 + 1; t <= k_last / 64; ++t) own_tiles = {min(own_tiles.x, tiles[t].x), max(own_tiles.y, tiles[t].y)};
  }

  Filler fill_q(static_cast<const elt_t*>(a.q) + (size_t)b * a.sq.batch, a.sq.token, a.head), fill_do(static_cast<const elt_t*>(a.dout) + (size_t)b * a.sdo.batch, a.sdo.token, a.head);
  Reader read(lane);
  typedef __attribute__((address_space(3))) void* lds_ptr;
  const unsigned lds_base = (unsigned)(uintptr_t)(lds_ptr)lds, lds_at = lds_base + wave * 1024;
  const auto fill = [&](unsigned h, const Step& step, unsigned slot) {
    if (!step.there()) return;
    const unsigned first = 64 * step.tile, rows = a.queries - first;
    fill_q.base = reinterpret_cast<const char*>(static_cast<const elt_t*>(a.q) + (size_t)b * a.sq.batch + (size_t)h * a.sq.head);
    fill_do.base = reinterpret_cast<const char*>(static_cast<const elt_t*>(a.dout) + (size_t)b * a.sdo.batch + (size_t)h * a.sdo.head);
    const size_t row = ((size_t)b * a.heads + h) * a.queries + first;
    const unsigned at = lds_at + slot * (2 * TILE), words = lds_base + SLOTS * (2 * TILE) + slot * 768;
    if (wave == 0) fill_words(a.less + row, rows, lane, words);
    if (wave == 1) fill_words(a.delta + row, rows, lane, words + 256);
    if (DOCS && wave == 2 && step.compare) fill_words(documents + first + shift, rows, lane, words + 512);
    // rows that see no key, padding and those before the first key, are read as zeros, whatever they hold
    const auto skip = [&](unsigned r) { return DOCS ? step.padded && a.lse[row + min(r, rows - 1)] == -INFINITY : (int)(first + r) < first_row; };
    fill_q(lane, wave, first, rows, at, skip);
    fill_do(lane, wave, first, rows, at + TILE, skip);
  };
  const auto look = [&](unsigned tile) -> unsigned {
    const int first = (int)(64 * tile), t0 = (first + shift) / 64, t1 = (min(first + 63, a.queries - 1) + shift) / 64;
    return look_at(t0 == t1 ? tiles[t0] : int2{min(tiles[t0].x, tiles[t1].x), max(tiles[t0].y, tiles[t1].y)}, own_tiles);
  };

  float16v dk[DB], dv[DB];
#pragma unroll
  for (unsigned db = 0; db < DB; ++db) dk[db] = dv[db] = zeros();
  float up = 0.0f;                 // the power of two that dk carries (fp16)
  const unsigned h0 = hk * group + part * a.heads_per_part, h1 = h0 + a.heads_per_part;
  const unsigned begin = k0 < prefix ? 0u : (unsigned)max(k0 - shift, 0) / 64, end = (unsigned)(a.queries + 63) / 64;
  typedef Walk<DOCS, decltype(look)> Queries;
  Queries walk(look, lane, begin, end);
  unsigned h = h0;
  const auto advance = [&](unsigned& head) {      // the next tile of the heads in turn
    Step step = walk.next();
    while (!step.there() && head + 1 < h1) {
      ++head;
      walk.restart(begin);
      step = walk.next();
    }
    return step;
  };
  // the tiles in turn for the halves of the workgroup
  struct { Step step; unsigned h; } now[HALVES], next[HALVES];
  unsigned buffer = 0;
#pragma unroll
  for (unsigned n = 0; n < HALVES; ++n) {
    now[n].step = advance(h);
    now[n].h = h;
    fill(h, now[n].step, n);
  }
  while (now[0].step.there()) {
#pragma unroll
    for (unsigned n = 0; n < HALVES; ++n) {
      next[n].step = advance(h);
      next[n].h = h;
    }
    wait_for_copies();
    __syncthreads();
#pragma unroll
    for (unsigned n = 0; n < HALVES; ++n) fill(next[n].h, next[n].step, (buffer ^ HALVES) + n);
    const Step own = now[half ? HALVES - 1 : 0].step;
    const unsigned own_h = now[half ? HALVES - 1 : 0].h;
    const char* const qt = lds + (buffer + half) * (2 * TILE);
    const char* const dot = qt + TILE;
    const float* const less_s = reinterpret_cast<const float*>(lds + SLOTS * (2 * TILE) + (buffer + half) * 768);
    const int first = (int)(64 * own.tile);
    const bool any = HALVES == 1 || own.there();
    const float slope = BIAS ? (CAP ? kLog2e : kLog2e * a.scores.unscale) * a.slopes[own_h] : 0.0f;
    if (any && first + 63 >= from_w0) {
#pragma unroll 1
      for (unsigned qb = 0; qb < 2; ++qb) {
        asm volatile("" : "+v"(read.row_at), "+v"(read.tr_at));      // the offsets of a step are one operation from these: they are not to be kept in registers
        // The operands that the products read from LDS, in their order: rows of Q, of dO, then columns of dO and of Q
        const auto operand = [&](unsigned j) {
          if (j < 2 * KS) return read.rows(j < KS ? qt : dot, qb, j % KS);
          const unsigned i = j - 2 * KS;
          return read.transposed(i < 2 * DB ? dot : qt, 2 * qb + i / DB % 2, i % DB);
        };
        // rows first + 32 qb + 8 (r / 4) + 4 lhi + r % 4
        const int row0 = first + 32 * (int)qb + 4 * (int)lhi;
        const bool edge = first + 32 * (int)qb < from_w1 || first + 32 * (int)qb + 32 > a.queries;
        // The sums start at what is added to them: a score at -lse (and its slope) over the scale, where no cap is in between, and dP at -delta.
        const auto lessened = [&](int g) { return *reinterpret_cast<const float4v*>(less_s + 32 * qb + 8 * g + 4 * lhi); };
        float16v s, dp;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4v x = CAP ? float4v{0.0f, 0.0f, 0.0f, 0.0f} : lessened(g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * g + e] = BIAS && !CAP ? x[e] - slope * fabsf((float)(row0 + 8 * g + e + shift - key)) : x[e];
        }
        elt8 ahead[RING];
#pragma unroll
        for (unsigned j = 0; j < RING; ++j) ahead[j] = operand(j);
        __builtin_amdgcn_sched_barrier(0);
        // every product has its slot, with the operand of the one RING further on and a part of the arithmetic that the products after these need
#pragma unroll
        for (unsigned j = 0; j < KS; ++j) {
          s = mfma(ahead[j % RING], kv[j], s);
          ahead[j % RING] = operand(j + RING);
          if (j == KS - 2) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float4v d = *reinterpret_cast<const float4v*>(less_s + 64 + 32 * qb + 8 * g + 4 * lhi);
#pragma unroll
              for (int e = 0; e < 4; ++e) dp[4 * g + e] = d[e];
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        unsigned p_pairs[8], ds_pairs[8];      // as operands: steps of eight values
        float4v less = CAP ? lessened(0) : float4v{};
        float p_even = 0.0f;
        const auto exponential = [&](int r) {
          float x = a.scores.scale_log2 * s[r], bend = 1.0f;
          if (CAP) {
            x = score<CAP>(s[r], a.scores, less[r % 4], bend);
            if (BIAS) x -= slope * fabsf((float)(row0 + 8 * (r / 4) + r % 4 + shift - key));
            if (r % 4 == 3 && r < 15) less = lessened(r / 4 + 1);
          }
          const float p = __builtin_amdgcn_exp2f(x);
          if (r % 2) p_pairs[r / 2] = pack(p_even, p);
          else p_even = p;
          s[r] = CAP ? p * bend : p;
        };
        const auto hide = [&](int r, bool seen0, bool seen1) {      // of rows r and r + 1
          p_pairs[r / 2] &= (seen0 ? 0xffffu : 0u) | (seen1 ? 0xffff0000u : 0u);
          s[r] = seen0 ? s[r] : 0.0f;
          s[r + 1] = seen1 ? s[r + 1] : 0.0f;
        };
        const auto derivative = [&](int r) {
          dp[r] *= s[r];
          if (r % 2) ds_pairs[r / 2] = pack(dp[r - 1], dp[r]);
        };
        const auto step_of = [](const unsigned (&x)[8], unsigned st) { return __builtin_bit_cast(elt8, u32x4{x[4 * st], x[4 * st + 1], x[4 * st + 2], x[4 * st + 3]}); };
#pragma unroll
        for (unsigned j = KS; j < 2 * KS; ++j) {
          dp = mfma(ahead[j % RING], vv[j - KS], dp);
          ahead[j % RING] = operand(j + RING);
#pragma unroll
          for (int r = (int)(16 * (j - KS) / KS); r < (int)(16 * (j - KS + 1) / KS); ++r) exponential(r);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (edge) {
          int begin = from_key - row0, end = a.queries - row0;
          asm volatile("" : "+v"(begin), "+v"(end));      // a branch, and no comparisons ahead of it: most tiles have nothing to hide
          const auto seen = [&](int r) { return 8 * (r / 4) + r % 4 >= begin && 8 * (r / 4) + r % 4 < end; };
#pragma unroll
          for (int r = 0; r < 16; r += 2) hide(r, seen(r), seen(r + 1));
        }
        if (DOCS && own.compare) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int4v d = *reinterpret_cast<const int4v*>(reinterpret_cast<const int*>(less_s) + 128 + 32 * qb + 8 * g + 4 * lhi);
            const auto seen = [&](int e) { return own_document >= 0 && d[e] == own_document; };
#pragma unroll
            for (int e = 0; e < 4; e += 2) hide(4 * g + e, seen(e), seen(e + 1));
          }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (unsigned j = 2 * KS; j < 2 * KS + 2 * DB; ++j) {
          const unsigned i = j - 2 * KS;
          dv[i % DB] = mfma(ahead[j % RING], step_of(p_pairs, i / DB), dv[i % DB]);
          ahead[j % RING] = operand(j + RING);
#pragma unroll
          for (int r = (int)(16 * i / (2 * DB)); r < (int)(16 * (i + 1) / (2 * DB)); ++r) derivative(r);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (unsigned j = 2 * KS + 2 * DB; j < 2 * KS + 4 * DB; ++j) {
          const unsigned i = j - 2 * KS - 2 * DB;
          dk[i % DB] = mfma(ahead[j % RING], step_of(ds_pairs, i / DB), dk[i % DB]);
          if (j + RING < 2 * KS + 4 * DB) ahead[j % RING] = operand(j + RING);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
#pragma unroll
    for (unsigned n = 0; n < HALVES; ++n) now[n] = next[n];
    buffer ^= HALVES;
  }
  float k_factor = (CAP ? 4.0f : 1.0f) * a.scores.scale, v_factor = kUnshift;
  if constexpr (HALVES == 2) {      // the second half's sums through LDS, in the tiles' place
    __syncthreads();
    float4v* const sums_s = reinterpret_cast<float4v*>(lds) + (wave % RW) * (2 * 64 * 4 * DB);
    static_assert(RW * 2 * 64 * 16 * DB * 4 <= SLOTS * 2 * TILE, "sums of the second half in the tiles' place");
    if (half) {
      put<DB>(dk, sums_s, lane, k_factor);
      put<DB>(dv, sums_s + 64 * 4 * DB, lane, v_factor);
    }
    __syncthreads();
    if (half) return;
    add<DB>(dk, k_factor, sums_s, lane, 1.0f);
    add<DB>(dv, v_factor, sums_s + 64 * 4 * DB, lane, 1.0f);
    k_factor = v_factor = 1.0f;
  }
  {
    const int j = key;
    const bool mine = j < a.keys;
    if (!a.parts) {
      store_columns<DB>(dk, mine ? static_cast<elt_t*>(a.dk) + (size_t)b * a.sdk.batch + (size_t)j * a.sdk.token + (size_t)hk * a.sdk.head : nullptr, lane, a.head, k_factor);
      store_columns<DB>(dv, mine ? static_cast<elt_t*>(a.dv) + (size_t)b * a.sdv.batch + (size_t)j * a.sdv.token + (size_t)hk * a.sdv.head : nullptr, lane, a.head, v_factor);
    } else if (mine) {
      const size_t rows = (size_t)a.batch * a.key_heads * a.keys, row = ((size_t)b * a.key_heads + hk) * a.keys + j;
      float* const dk_at = a.parts + ((size_t)(2 * part) * rows + row) * a.head;
      float* const dv_at = dk_at + rows * a.head;
#pragma unroll
      for (unsigned db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const unsigned d = 32 * db + 8 * g + 4 * lhi;
          if (d >= (unsigned)a.head) continue;
          *reinterpret_cast<float4v*>(dk_at + d) = float4v{k_factor * dk[db][4 * g], k_factor * dk[db][4 * g + 1], k_factor * dk[db][4 * g + 2], k_factor * dk[db][4 * g + 3]};
          *reinterpret_cast<float4v*>(dv_at + d) = float4v{v_factor * dv[db][4 * g], v_factor * dv[db][4 * g + 1], v_factor * dv[db][4 * g + 2], v_factor * dv[db][4 * g + 3]};
        }
    }
  }
}

template <bool CAP, bool BIAS, bool DOCS, unsigned HALVES>
__global__ void __launch_bounds__(64 * WAVES, 2) lego_attention_dq_bf16_d128_kernel(AttentionArgs a)
{
  constexpr unsigned RW = WAVES / HALVES, OWN = 32 * RW, SLOTS = 2 * HALVES;      // as in the forward kernel
  __shared__ __attribute__((aligned(1024))) char lds[SLOTS * (2 * TILE + 256)];      // K and V, then the keys' documents
  const unsigned lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l32 = lane % 32, lhi = lane / 32, half = wave / RW;
  const unsigned blocks = (a.queries + OWN - 1) / OWN;
  const unsigned all_heads = a.heads * a.batch, turn = blockIdx.x / all_heads;
  const unsigned head = place(blockIdx.x % all_heads, all_heads);
  const unsigned h = head % a.heads, b = head / a.heads;
  const unsigned block = DOCS && a.order_queries ? __builtin_amdgcn_readfirstlane(a.order_queries[b * blocks + turn]) : blocks - 1 - turn;      // later queries may see more keys
  const unsigned hk = h / (a.heads / a.key_heads);
  const int q0 = (int)(OWN * block), q_last = min(q0 + (int)OWN, a.queries) - 1;
  const int w0 = q0 + 32 * (int)(wave % RW), i = w0 + (int)l32;
  const Seen seen{a.keys, a.keys - a.queries, a.causal ? (a.prefix ? max(a.prefix[b], 0) : 0) : -1};
  const int limit = seen.limit(i), limit_w0 = seen.limit(w0), limit_w1 = seen.limit(min(w0 + 31, q_last));
  const int* const documents = DOCS ? a.documents + (size_t)b * a.keys : nullptr;
  const int2* const tiles = DOCS ? a.tiles + (size_t)b * ((a.keys + 63) / 64) : nullptr;
  const size_t stat = ((size_t)b * a.heads + h) * a.queries + min(i, a.queries - 1);
  const bool nothing = a.lse[stat] == -INFINITY;      // a query that sees no key is zeros, whatever it holds
  const float less = nothing ? 0.0f : a.less[stat], delta = nothing ? 0.0f : a.delta[stat];

  elt8 qv[KS], dov[KS];
  {
    const elt_t* const qrow = static_cast<const elt_t*>(a.q) + (size_t)b * a.sq.batch + (size_t)min(i, a.queries - 1) * a.sq.token + (size_t)h * a.sq.head;
    const elt_t* const dorow = static_cast<const elt_t*>(a.dout) + (size_t)b * a.sdo.batch + (size_t)min(i, a.queries - 1) * a.sdo.token + (size_t)h * a.sdo.head;
#pragma unroll
    for (unsigned ks = 0; ks < KS; ++ks) {
      const unsigned d = 16 * ks + 8 * lhi;
      qv[ks] = d < (unsigned)a.head && !nothing ? *reinterpret_cast<const elt8*>(qrow + d) : elt8{};
      dov[ks] = d < (unsigned)a.head && !nothing ? *reinterpret_cast<const elt8*>(dorow + d) : elt8{};
    }
  }
  const int own_document = DOCS ? documents[min(i, a.queries - 1) + seen.shift] : 0;
  int2 own_tiles = {0, 0};
  if (DOCS) {
    own_tiles = tiles[(q0 + seen.shift) / 64];
    for (int t = (q0 + seen.shift) / 64 + 1; t <= (q_last + seen.shift) / 64; ++t) own_tiles = {min(own_tiles.x, tiles[t].x), max(own_tiles.y, tiles[t].y)};
  }
  const float slope = BIAS ? (CAP ? kLog2e : kLog2e * a.scores.unscale) * a.slopes[h] : 0.0f;

  const elt_t* const kb = static_cast<const elt_t*>(a.k) + (size_t)b * a.sk.batch + (size_t)hk * a.sk.head;
  const elt_t* const vb = static_cast<const elt_t*>(a.v) + (size_t)b * a.sv.batch + (size_t)hk * a.sv.head;
  const Filler fill_k(kb, a.sk.token, a.head), fill_v(vb, a.sv.token, a.head);
  Reader read(lane);
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

  float16v dq[DB];
#pragma unroll
  for (unsigned db = 0; db < DB; ++db) dq[db] = zeros();
  Walk<DOCS, decltype(look)> walk(look, lane, 0, (unsigned)(seen.limit(q_last) + 63) / 64);
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
    __syncthreads();
#pragma unroll
    for (unsigned n = 0; n < HALVES; ++n) fill(next[n], (buffer ^ HALVES) + n);
    const Step own = now[half ? HALVES - 1 : 0];
    const char* const kt = lds + (buffer + half) * (2 * TILE);
    const char* const vt = kt + TILE;
    const int first = (int)(64 * own.tile);
    const int* const document_s = reinterpret_cast<const int*>(lds + SLOTS * (2 * TILE) + (buffer + half) * 256);
    if ((HALVES == 1 || own.there()) && first < limit_w1) {
      asm volatile("" : "+v"(read.row_at), "+v"(read.tr_at));      // the offsets of a step are one operation from these: they are not to be kept in registers
      // The operands that the products read from LDS, in their order: rows of K and of V for either half of the keys, then columns of K
      const auto operand = [&](unsigned j) {
        if (j < 4 * KS) return read.rows(j / KS % 2 ? vt : kt, j / (2 * KS), j % KS);
        const unsigned i = j - 4 * KS;
        return read.transposed(kt, i / DB, i % DB);
      };
      float16v s[2], dp[2];      // they start at what is added to them, as in the other kernel
      const auto start = [&](int kb2, bool scores) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (!scores) dp[kb2][r] = delta;
          else s[kb2][r] = CAP ? 0.0f : BIAS ? less - slope * fabsf((float)(i + seen.shift - first - 4 * (int)lhi - (32 * kb2 + 8 * (r / 4) + r % 4))) : less;
        }
      };
      elt8 ahead[RING];
#pragma unroll
      for (unsigned j = 0; j < RING; ++j) ahead[j] = operand(j);
      __builtin_amdgcn_sched_barrier(0);
      const auto exponential = [&](int kb2, int r) {
        float x = a.scores.scale_log2 * s[kb2][r], bend = 1.0f;
        if (CAP) {
          x = score<CAP>(s[kb2][r], a.scores, less, bend);
          if (BIAS) x -= slope * fabsf((float)(i + seen.shift - first - 4 * (int)lhi - (32 * kb2 + 8 * (r / 4) + r % 4)));
        }
        s[kb2][r] = __builtin_amdgcn_exp2f(x);
        if (CAP) s[kb2][r] *= bend;
      };
      unsigned ds_pairs[2][8];      // as operands: steps of eight values
      const auto derivative = [&](int kb2, int r) {
        dp[kb2][r] *= s[kb2][r];
        if (r % 2) ds_pairs[kb2][r / 2] = pack(dp[kb2][r - 1], dp[kb2][r]);
      };
      const auto step_of = [](const unsigned (&x)[8], unsigned st) { return __builtin_bit_cast(elt8, u32x4{x[4 * st], x[4 * st + 1], x[4 * st + 2], x[4 * st + 3]}); };
      const auto hide = [&](int kb2) {
        if (first + 32 * kb2 + 32 > limit_w0) {
          int end = limit - first - 32 * kb2 - 4 * (int)lhi;
          asm volatile("" : "+v"(end));      // a branch, and no comparisons ahead of it: most tiles have nothing to hide
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb2][r] = 8 * (r / 4) + r % 4 < end ? s[kb2][r] : 0.0f;
        }
        if (DOCS && own.compare) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int4v d = *reinterpret_cast<const int4v*>(document_s + 32 * kb2 + 8 * g + 4 * lhi);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[kb2][4 * g + e] = own_document >= 0 && d[e] == own_document ? s[kb2][4 * g + e] : 0.0f;
          }
        }
      };
      // every product has its slot, with the operand of the one RING further on and a part of the arithmetic that the products after these need
      const auto products = [&](auto which) {      // scores of a half of the keys, or dP of it
        constexpr unsigned PART = decltype(which)::value, HALF = PART / 2;
        start(HALF, PART % 2 == 0);
#pragma unroll
        for (unsigned ks = 0; ks < KS; ++ks) {
          constexpr unsigned j0 = PART * KS;
          if (PART % 2 == 0) s[HALF] = mfma(ahead[(j0 + ks) % RING], qv[ks], s[HALF]);
          else dp[HALF] = mfma(ahead[(j0 + ks) % RING], dov[ks], dp[HALF]);
          ahead[(j0 + ks) % RING] = operand(j0 + ks + RING);
#pragma unroll
          for (int r = (int)(16 * ks / KS); r < (int)(16 * (ks + 1) / KS); ++r) {
            if (PART == 2) derivative(0, r);
            else if (PART % 2) exponential(HALF, r);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      products(Constant<0>{});
      products(Constant<1>{});
      hide(0);
      products(Constant<2>{});
      products(Constant<3>{});
      hide(1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (unsigned j = 4 * KS; j < 4 * KS + 4 * DB; ++j) {
        const unsigned i = j - 4 * KS;
        dq[i % DB] = mfma(ahead[j % RING], step_of(ds_pairs[i / (2 * DB)], i / DB % 2), dq[i % DB]);
        if (j + RING < 4 * KS + 4 * DB) ahead[j % RING] = operand(j + RING);
        if (i < 2 * DB) {
#pragma unroll
          for (int r = (int)(16 * i / (2 * DB)); r < (int)(16 * (i + 1) / (2 * DB)); ++r) derivative(1, r);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (unsigned n = 0; n < HALVES; ++n) now[n] = next[n];
    buffer ^= HALVES;
  }
  if constexpr (HALVES == 2) {      // the second half's sums through LDS, in the tiles' place
    __syncthreads();
    float4v* const sums_s = reinterpret_cast<float4v*>(lds) + (wave % RW) * (64 * 4 * DB);
    if (half) put<DB>(dq, sums_s, lane, 1.0f);
    __syncthreads();
    if (half) return;
    add<DB>(dq, 1.0f, sums_s, lane, 1.0f);
  }
  elt_t* const row = i < a.queries ? static_cast<elt_t*>(a.dq) + (size_t)b * a.sdq.batch + (size_t)i * a.sdq.token + (size_t)h * a.sdq.head : nullptr;
  store_columns<DB>(dq, row, lane, a.head, (CAP ? 4.0f : 1.0f) * a.scores.scale);
}

}  // namespace

hipError_t lego_attention_bwd_bf16_d128_launch(const AttentionArgs& a, hipStream_t stream)
{
  const auto launch = [&](auto whole, auto halves, bool halve, int rows, unsigned of) {
    const unsigned own = halve ? 16 * WAVES : 32 * WAVES;
    hipLaunchKernelGGL(halve ? halves : whole, dim3(((unsigned)rows + own - 1) / own * of), dim3(64 * WAVES), 0, stream, a);
    return hipGetLastError();
  };
  const auto both = [&](auto dkv, auto dkv_halves, auto dq, auto dq_halves) {
    const hipError_t e = launch(dkv, dkv_halves, a.halve_keys != 0, a.keys, (unsigned)(a.heads / a.heads_per_part) * (unsigned)a.batch);
    return e != hipSuccess ? e : launch(dq, dq_halves, a.halve_queries != 0, a.queries, (unsigned)(a.heads * a.batch));
  };
  if ((a.capped != 0) == true && (a.slopes != nullptr) == true && (a.documents != nullptr) == true)
    return both(lego_attention_dkv_bf16_d128_kernel<true, true, true, 1>, lego_attention_dkv_bf16_d128_kernel<true, true, true, 2>,
                lego_attention_dq_bf16_d128_kernel<true, true, true, 1>, lego_attention_dq_bf16_d128_kernel<true, true, true, 2>);
  if ((a.capped != 0) == true && (a.slopes != nullptr) == true && (a.documents != nullptr) == false)
    return both(lego_attention_dkv_bf16_d128_kernel<true, true, false, 1>, lego_attention_dkv_bf16_d128_kernel<true, true, false, 2>,
                lego_attention_dq_bf16_d128_kernel<true, true, false, 1>, lego_attention_dq_bf16_d128_kernel<true, true, false, 2>);
  if ((a.capped != 0) == true && (a.slopes != nullptr) == false && (a.documents != nullptr) == true)
    return both(lego_attention_dkv_bf16_d128_kernel<true, false, true, 1>, lego_attention_dkv_bf16_d128_kernel<true, false, true, 2>,
                lego_attention_dq_bf16_d128_kernel<true, false, true, 1>, lego_attention_dq_bf16_d128_kernel<true, false, true, 2>);
  if ((a.capped != 0) == true && (a.slopes != nullptr) == false && (a.documents != nullptr) == false)
    return both(lego_attention_dkv_bf16_d128_kernel<true, false, false, 1>, lego_attention_dkv_bf16_d128_kernel<true, false, false, 2>,
                lego_attention_dq_bf16_d128_kernel<true, false, false, 1>, lego_attention_dq_bf16_d128_kernel<true, false, false, 2>);
  if ((a.capped != 0) == false && (a.slopes != nullptr) == true && (a.documents != nullptr) == true)
    return both(lego_attention_dkv_bf16_d128_kernel<false, true, true, 1>, lego_attention_dkv_bf16_d128_kernel<false, true, true, 2>,
                lego_attention_dq_bf16_d128_kernel<false, true, true, 1>, lego_attention_dq_bf16_d128_kernel<false, true, true, 2>);
  if ((a.capped != 0) == false && (a.slopes != nullptr) == true && (a.documents != nullptr) == false)
    return both(lego_attention_dkv_bf16_d128_kernel<false, true, false, 1>, lego_attention_dkv_bf16_d128_kernel<false, true, false, 2>,
                lego_attention_dq_bf16_d128_kernel<false, true, false, 1>, lego_attention_dq_bf16_d128_kernel<false, true, false, 2>);
  if ((a.capped != 0) == false && (a.slopes != nullptr) == false && (a.documents != nullptr) == true)
    return both(lego_attention_dkv_bf16_d128_kernel<false, false, true, 1>, lego_attention_dkv_bf16_d128_kernel<false, false, true, 2>,
                lego_attention_dq_bf16_d128_kernel<false, false, true, 1>, lego_attention_dq_bf16_d128_kernel<false, false, true, 2>);
  if ((a.capped != 0) == false && (a.slopes != nullptr) == false && (a.documents != nullptr) == false)
    return both(lego_attention_dkv_bf16_d128_kernel<false, false, false, 1>, lego_attention_dkv_bf16_d128_kernel<false, false, false, 2>,
                lego_attention_dq_bf16_d128_kernel<false, false, false, 1>, lego_attention_dq_bf16_d128_kernel<false, false, false, 2>);
  return hipErrorInvalidValue;
}
