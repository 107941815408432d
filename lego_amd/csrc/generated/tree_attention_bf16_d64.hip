// generated by lego_amd (python -m lego_amd.build) -- do not edit; edit the generator
//
// Attention of drafted tokens over a paged cache, bf16, up to 64 head elements: a draft sees all cached keys of its sequence and the drafts that the tree shows
// it.  One draft a sequence is ordinary decoding.
// Bound by memory where drafts are few: every cached key and value is read once for all drafts and all query heads that share its head.  Those are the rows of an item, 32 to a
// wavefront; up to 32 rows leave the keys of a tile to two wavefronts, up to 64 to two pairs, more share the tile.  Sequences have any length, so the tiles of
// all items, one after another, are dealt to the workgroups in equal runs, whatever item they belong to; an item in one run is done there, sums of one in several are joined by a second kernel,
// in their order.  With few tiles an item a workgroup takes an item, in one launch.
// Scores are transposed as in the forward kernel: a row to a lane of each half.  Tiles of 64 keys go from memory into LDS without passing registers, the next one on its way
// while one is computed, the pages of the one after that looked up meanwhile.
// Index expressions printed from LEGO layouts:
//   LDS tile   OrderBy(GenP((64, 8), row*8 + (chunk ^ key(row)))).TileBy([64, 8])

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

constexpr unsigned DC = 64;               // head elements that are computed; elements from the head's size on are zeros
constexpr unsigned KS = DC / 16, DB = DC / 32;   // MFMA steps along the head, blocks of 32 head elements
constexpr unsigned PITCH = 64;           // elements between the rows of a tile in LDS
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

// A tile in LDS: OrderBy(GenP((64, 8), row*8 + (chunk ^ key(row)))).TileBy([64, 8])
// with chunks of 16 bytes; the key makes both kinds of reads, 16 bytes of 16 rows in a row and transposing ones of 64 bytes of four rows, free of bank
// conflicts.  rows(): the first operand whose rows are the tile's (block of 32 rows, step of 16 head elements); transposed(): the first operand whose rows
// are 32 head elements (block `db`) and whose sum goes over 16 of the tile's rows, in as_operands()'s order.
struct Reader {
  unsigned row_at, tr_at;       // bytes within a tile
  __device__ __forceinline__ explicit Reader(unsigned lane)
  {
    const unsigned l32 = lane % 32, lhi = lane / 32, l16 = lane % 16, lgrp = lane / 16;
    row_at = 16 * (8*l32 + ((lhi) ^ (((l32)/(4)) % 4 + 4*(((l32)/(2)) % 2))));
    tr_at = 16 * (32*lhi + ((2*(lgrp % 2) + ((l16 % 4)/(2))) ^ (lhi + 4*((l16)/(8)))) + 8*((l16)/(4))) + 8 * (l16 % 2);
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
    const unsigned row0 = 8*wave + ((lane)/(8)), chunk = ((lane % 8) ^ ((2*wave + ((lane)/(32))) % 4 + 4*(((lane)/(16)) % 2)));
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
#define LEGO_ARITHMETIC(N) __builtin_amdgcn_sched_group_barrier(0x402, N, 0)

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

}  // namespace

namespace {

constexpr float kLazy = 8.0f;

// Tiles of a sequence's items
struct Sequence { unsigned b, length, cached, tiles; };

__device__ __forceinline__ Sequence sequence_of(const TreeArgs& a, unsigned b)
{
  const unsigned most = (unsigned)a.width * (unsigned)a.page;
  const unsigned length = (unsigned)min((unsigned)max(a.lengths[b], 0), most), cached = (length + 63) / 64;
  return {b, length, cached, cached + (a.k ? ((unsigned)a.drafts + 63) / 64 : 0u)};
}

__device__ __forceinline__ unsigned scan_of_wave(unsigned x, unsigned lane)      // sum over lanes up to this one
{
#pragma unroll
  for (unsigned d = 1; d < 64; d *= 2) {
    const unsigned y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// All items' tiles, and the first sequence whose tiles end behind tile `at` with the tiles before it (wave-uniform).
__device__ __forceinline__ unsigned total_tiles(const TreeArgs& a, unsigned lane, unsigned items)
{
  unsigned sum = 0;
  for (unsigned b0 = 0; b0 < (unsigned)a.batch; b0 += 64) sum += b0 + lane < (unsigned)a.batch ? sequence_of(a, b0 + lane).tiles * items : 0u;
#pragma unroll
  for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
  return __builtin_amdgcn_readfirstlane(sum);
}
__device__ __forceinline__ unsigned find_sequence(const TreeArgs& a, unsigned lane, unsigned items, unsigned at, unsigned& before)
{
  before = 0;
  for (unsigned b0 = 0; b0 < (unsigned)a.batch; b0 += 64) {
    const unsigned n = b0 + lane < (unsigned)a.batch ? sequence_of(a, b0 + lane).tiles * items : 0u;
    const unsigned upto = scan_of_wave(n, lane);
    const unsigned long long behind = __builtin_amdgcn_ballot_w64(before + upto > at);
    if (behind) {
      const unsigned l = (unsigned)__builtin_ctzll(behind);
      before += __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l);
      return b0 + l;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return a.batch;
}
__device__ __forceinline__ unsigned tiles_before(const TreeArgs& a, unsigned lane, unsigned items, unsigned b)
{
  unsigned sum = 0;
  for (unsigned b0 = 0; b0 < b; b0 += 64) sum += b0 + lane < b ? sequence_of(a, b0 + lane).tiles * items : 0u;
#pragma unroll
  for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
  return __builtin_amdgcn_readfirstlane(sum);
}

__device__ __forceinline__ unsigned run_of(const TreeArgs& a, unsigned total) { return max(2u, (total + a.workgroups - 1) / a.workgroups); }

template <bool CAP, bool BIAS, unsigned RW>
__global__ void __launch_bounds__(RW == 1 ? 128 : 256, RW == 1 ? 1 : 2) lego_tree_bf16_d64_kernel(TreeArgs a)
{
  constexpr unsigned NW = RW == 1 ? 2 : 4, KW = NW / RW, NB = 2 / KW, FILLS = TILE / 1024 / NW;
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];      // K and V, twice
  const unsigned lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l32 = lane % 32, lhi = lane / 32;
  const unsigned rw = wave % RW, kw = wave / RW;
  const unsigned group = a.heads / a.key_heads, rows = group * a.drafts, items = a.key_heads * a.row_blocks;
  const Reader read(lane);
  typedef __attribute__((address_space(3))) void* lds_ptr;
  const unsigned lds_at = (unsigned)(uintptr_t)(lds_ptr)lds;

  unsigned b, item, tile, left;      // the present sequence, item of it, tile of that; tiles of the run that are left
  Sequence seq;
  if (a.whole) {
    b = blockIdx.x / items;
    item = blockIdx.x % items;
    seq = sequence_of(a, b);
    tile = 0;
    left = seq.tiles;
  } else {
    const unsigned total = total_tiles(a, lane, items), run = run_of(a, total), first = blockIdx.x * run;
    if (first >= total) return;
    left = min(run, total - first);
    unsigned before;
    b = find_sequence(a, lane, items, first, before);
    seq = sequence_of(a, b);
    item = (first - before) / seq.tiles;
    tile = (first - before) % seq.tiles;
  }
  do {
    const unsigned hk = item / a.row_blocks, rb = item % a.row_blocks;
    const unsigned count = min(left, seq.tiles - tile);      // tiles of this item
    const unsigned r = 32 * (rb * RW + rw) + l32;             // the lane's row
    const bool mine = r < rows;
    const unsigned t = min(r, rows - 1) / group, h = hk * group + min(r, rows - 1) % group;
    elt8 qv[KS];
    {
      const elt_t* const row = static_cast<const elt_t*>(a.q) + (size_t)b * a.sq.batch + (size_t)t * a.sq.token + (size_t)h * a.sq.head;
#pragma unroll
      for (unsigned ks = 0; ks < KS; ++ks) {
        const unsigned d = 16 * ks + 8 * lhi;
        qv[ks] = d < (unsigned)a.head ? *reinterpret_cast<const elt8*>(row + d) : elt8{};
      }
    }
    const int* const pages = a.pages + (size_t)b * a.width;
    const float slope = BIAS ? kLog2e * a.slopes[h] : 0.0f;
    const int position = BIAS ? (a.positions ? a.positions[(size_t)b * a.drafts + t] : (int)(seq.length + t)) : 0;
    const unsigned char* const shown = a.tree ? a.tree + (size_t)b * a.tree_batch + (size_t)t * a.drafts : nullptr;

    // Where the rows of a tile lie, a row to a lane: 16-byte chunks from the base, ~0 for none.  One division a tile; the lanes that copy a row ask the lane that knows it.
    struct Rows { unsigned k, v; };
    const auto look_up = [&](unsigned n) {
      Rows p = {~0u, ~0u};
      if (n < seq.cached) {
        const unsigned key = 64 * n + lane;
        const int at = page_of(pages, a.width, a.page, a.count, seq.length, key);
        const unsigned slot = key % (unsigned)a.page;
        if (at >= 0)
          p = {(unsigned)(((size_t)at * a.skc.batch + (size_t)slot * a.skc.token + (size_t)hk * a.skc.head) / 8), (unsigned)(((size_t)at * a.svc.batch + (size_t)slot * a.svc.token + (size_t)hk * a.svc.head) / 8)};
      } else {
        const unsigned j = 64 * (n - seq.cached) + lane;
        if (j < (unsigned)a.drafts)
          p = {(unsigned)(((size_t)b * a.sk.batch + (size_t)j * a.sk.token + (size_t)hk * a.sk.head) / 8), (unsigned)(((size_t)b * a.sv.batch + (size_t)j * a.sv.token + (size_t)hk * a.sv.head) / 8)};
      }
      return p;
    };
    const auto fill = [&](unsigned n, const Rows& p, unsigned buffer) {
      const char* const kb = static_cast<const char*>(n < seq.cached ? a.k_cache : a.k);
      const char* const vb = static_cast<const char*>(n < seq.cached ? a.v_cache : a.v);
#pragma unroll
      for (unsigned it = 0; it < FILLS; ++it) {
        const unsigned g = it * NW + wave, row = 8*g + ((lane)/(8)), chunk = ((lane % 8) ^ ((2*g + ((lane)/(32))) % 4 + 4*(((lane)/(16)) % 2)));
        const unsigned k_at = __shfl(p.k, row), v_at = __shfl(p.v, row);
        const unsigned to = buffer * (2 * TILE) + g * 1024;
        if (k_at != ~0u && 8 * chunk < (unsigned)a.head) {
          asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(kb + ((size_t)k_at + chunk) * 16), "s"(lds_at + to) : "memory", "m0");
          asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(vb + ((size_t)v_at + chunk) * 16), "s"(lds_at + to + TILE) : "memory", "m0");
        } else if (8 * chunk < DC) {      // whatever another sequence left there
          *reinterpret_cast<u32x4*>(lds + to + lane * 16) = u32x4{0u, 0u, 0u, 0u};
          *reinterpret_cast<u32x4*>(lds + to + TILE + lane * 16) = u32x4{0u, 0u, 0u, 0u};
        }
      }
    };

    float16v acc[DB];
#pragma unroll
    for (unsigned db = 0; db < DB; ++db) acc[db] = zeros();
    float most = -INFINITY, sum = 0.0f;
    unsigned buffer = 0;
    Rows next_rows = look_up(tile);
    unsigned long long here = 0, here_next = __builtin_amdgcn_ballot_w64(next_rows.k != ~0u);
    if (count) {
      const Rows rows_now = next_rows;
      if (count > 1) next_rows = look_up(tile + 1);
      fill(tile, rows_now, 0);
    }
    for (unsigned n = tile; n < tile + count; ++n) {
      here = here_next;
      wait_for_copies();
      __syncthreads();
      if (n + 1 < tile + count) {
        const Rows rows_now = next_rows;
        here_next = __builtin_amdgcn_ballot_w64(rows_now.k != ~0u);
        if (n + 2 < tile + count) next_rows = look_up(n + 2);
        fill(n + 1, rows_now, buffer ^ 1);
      }
      const char* const kt = lds + buffer * (2 * TILE);
      const char* const vt = kt + TILE;
      const bool cached = n < seq.cached;
      const int first = (int)(64 * (cached ? n : n - seq.cached)) + (int)(32 * NB * kw);      // of this wavefront's keys
      float16v s[NB];
#pragma unroll
      for (unsigned i = 0; i < NB; ++i) s[i] = zeros();
#pragma unroll
      for (unsigned ks = 0; ks < KS; ++ks)
#pragma unroll
        for (unsigned i = 0; i < NB; ++i) s[i] = mfma(read.rows(kt, NB * kw + i, ks), qv[ks], s[i]);
      const float distance0 = (float)(position - first - 4 * (int)lhi);
#pragma unroll
      for (unsigned i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x = score<CAP>(s[i][e], a.scores);
          if (BIAS && cached) x -= slope * fabsf(distance0 - (float)(int)(32 * i + 8 * (e / 4) + e % 4));
          s[i][e] = x;
        }
      // what of the cache's tile is not there
      if (cached) {
        if (here != ~0ull) {
          const unsigned long long own = here >> (32 * NB * kw + 4 * lhi);
#pragma unroll
          for (unsigned i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[i][e] = own >> (32 * i + 8 * (e / 4) + e % 4) & 1 ? s[i][e] : -INFINITY;
        }
      } else {
#pragma unroll
        for (unsigned i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int j = first + (int)(32 * i + 8 * (e / 4) + 4 * lhi) + e % 4;
            const bool inside = j < a.drafts;
            const bool seen = inside && (shown ? shown[inside ? j : 0] != 0 : j <= (int)t);
            float x = s[i][e];
            if (BIAS) x -= slope * fabsf((float)(position - (a.positions ? a.positions[(size_t)b * a.drafts + (inside ? j : 0)] : (int)seq.length + j)));
            s[i][e] = seen ? x : -INFINITY;
          }
      }
      float top = s[0][0];
#pragma unroll
      for (unsigned i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[i][e]);
      top = across_max(top);
      if (__builtin_amdgcn_ballot_w64(top > most + kLazy) != 0) {
        const float risen = fmaxf(most, top), factor = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(most - risen);
        most = risen;
        sum *= factor;
#pragma unroll
        for (unsigned db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[db][e] *= factor;
      }
      const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll
      for (unsigned i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[i][e] = __builtin_amdgcn_exp2f(s[i][e] - base);
          sum += s[i][e];
        }
#pragma unroll
      for (unsigned i = 0; i < NB; ++i) {
        const Operands p = as_operands(s[i]);
#pragma unroll
        for (unsigned st = 0; st < 2; ++st)
#pragma unroll
          for (unsigned db = 0; db < DB; ++db) acc[db] = mfma(read.transposed(vt, 2 * (NB * kw + i) + st, db), p.step[st], acc[db]);
      }
      buffer ^= 1;
    }
    sum = across_sum(sum);
    if constexpr (KW == 2) {      // the second wavefront's sums through LDS, past its tiles
      __syncthreads();
      float4v* const acc_s = reinterpret_cast<float4v*>(lds) + rw * (64 * 4 * DB);
      float2* const stat_s = reinterpret_cast<float2*>(lds + 3 * TILE) + rw * 64;
      static_assert(RW * 64 * 16 * DB * 4 <= 3 * TILE && RW * 64 * 8 <= TILE, "sums of the second wavefronts in the tiles' place");
      if (kw == 1) {
#pragma unroll
        for (unsigned db = 0; db < DB; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g) acc_s[(4 * db + g) * 64 + lane] = float4v{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
        stat_s[lane] = float2{most, sum};
      }
      __syncthreads();
      if (kw == 0) {
        const float2 o = stat_s[lane];
        const float top = fmaxf(most, o.x);
        const float f0 = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(most - top), f1 = o.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(o.x - top);
        most = top;
        sum = f0 * sum + f1 * o.y;
#pragma unroll
        for (unsigned db = 0; db < DB; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4v x = acc_s[(4 * db + g) * 64 + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[db][4 * g + e] = f0 * acc[db][4 * g + e] + f1 * x[e];
          }
      }
    }
    if (kw == 0) {
      if (count == seq.tiles) {
        elt_t* const row = mine ? static_cast<elt_t*>(a.o) + (size_t)b * a.so.batch + (size_t)t * a.so.token + (size_t)h * a.so.head : nullptr;
        store_columns<DB>(acc, row, lane, a.head, sum == 0.0f ? 0.0f : 1.0f / sum);
      } else {      // slot: the workgroup's number and the item's, which no two parts share
        const size_t slot = (size_t)blockIdx.x + (size_t)b * items + item;
        const size_t at = slot * (32 * RW) + 32 * rw + l32;
        if (lhi == 0) a.stats[at] = float2{most, sum};
        float* const to = a.sums + at * DC;
#pragma unroll
        for (unsigned db = 0; db < DB; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4v*>(to + 32 * db + 8 * g + 4 * lhi) = float4v{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
      }
    }
    left -= count;
    if (left == 0) break;
    __syncthreads();      // the tiles' place is free again
    tile = 0;
    if (++item == items) {
      item = 0;
      do seq = sequence_of(a, ++b);
      while (seq.tiles == 0);
    }
  } while (true);
}

// The rows of items in several runs, and of those that have no tile: a workgroup a row, DC / 4 lanes a part of its sums, the parts in turn.
__global__ void __launch_bounds__(256) lego_tree_join_bf16_d64_kernel(TreeArgs a, unsigned block_rows)
{
  constexpr unsigned LANES = DC / 4 > 16 ? 32 : 16, TEAMS = 256 / LANES;
  __shared__ float4v sums_s[TEAMS][LANES];
  __shared__ float2 stats_s[4];
  const unsigned lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const unsigned group = a.heads / a.key_heads, rows = group * a.drafts, items = a.key_heads * a.row_blocks;
  const unsigned b = blockIdx.x / (a.key_heads * rows), hk = blockIdx.x / rows % a.key_heads, r = blockIdx.x % rows;
  const unsigned total = total_tiles(a, lane, items), run = run_of(a, total);
  const unsigned item = hk * a.row_blocks + r / block_rows;
  const unsigned tiles = sequence_of(a, b).tiles, first = tiles_before(a, lane, items, b) + item * tiles;
  const unsigned t = r / group, h = hk * group + r % group;
  elt_t* const row = static_cast<elt_t*>(a.o) + (size_t)b * a.so.batch + (size_t)t * a.so.token + (size_t)h * a.so.head;
  if (tiles == 0) {
    if (threadIdx.x < (unsigned)a.head / 8) *reinterpret_cast<u32x4*>(row + 8 * threadIdx.x) = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  const unsigned w0 = first / run, parts = (first + tiles - 1) / run - w0 + 1;
  if (parts == 1) return;
  const size_t place0 = ((size_t)w0 + (size_t)b * items + item) * block_rows + r % block_rows;      // parts are block_rows apart
  float most = -INFINITY;
  for (unsigned p = threadIdx.x; p < parts; p += 256) most = fmaxf(most, a.stats[place0 + (size_t)p * block_rows].x);
#pragma unroll
  for (int d = 32; d; d /= 2) most = fmaxf(most, __shfl_xor(most, d));
  if (lane == 0) stats_s[wave].x = most;
  __syncthreads();
  most = fmaxf(fmaxf(stats_s[0].x, stats_s[1].x), fmaxf(stats_s[2].x, stats_s[3].x));
  float sum = 0.0f;      // the same in every lane of a team
  float4v x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (unsigned p = team; p < parts; p += TEAMS) {
    const size_t place = place0 + (size_t)p * block_rows;
    const float2 stat = a.stats[place];
    const float f = stat.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(stat.x - most);
    sum += f * stat.y;
    if (4 * c < DC) x += f * *reinterpret_cast<const float4v*>(a.sums + place * DC + 4 * c);
  }
  sums_s[team][c] = x;
  __shared__ float sum_s[TEAMS];
  if (c == 0) sum_s[team] = sum;
  __syncthreads();
  if (team) return;
#pragma unroll
  for (unsigned i = 1; i < TEAMS; ++i) {
    x += sums_s[i][c];
    sum += sum_s[i];
  }
  const float factor = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (4 * c < (unsigned)a.head) *reinterpret_cast<u32x2*>(row + 4 * c) = u32x2{pack(factor * x[0], factor * x[1]), pack(factor * x[2], factor * x[3])};
}

template <unsigned RW>
hipError_t launch_rows(const TreeArgs& a, hipStream_t stream)
{
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(a.whole ? (unsigned)(a.batch * a.key_heads) * a.row_blocks : a.workgroups), dim3(RW == 1 ? 128 : 256), 0, stream, a);
    return hipGetLastError();
  };
  hipError_t e;
  if (a.capped) e = a.slopes ? launch(lego_tree_bf16_d64_kernel<true, true, RW>) : launch(lego_tree_bf16_d64_kernel<true, false, RW>);
  else e = a.slopes ? launch(lego_tree_bf16_d64_kernel<false, true, RW>) : launch(lego_tree_bf16_d64_kernel<false, false, RW>);
  if (e != hipSuccess || a.whole) return e;
  const unsigned all = (unsigned)(a.batch * a.heads * a.drafts);
  hipLaunchKernelGGL(lego_tree_join_bf16_d64_kernel, dim3(all), dim3(256), 0, stream, a, 32 * RW);
  return hipGetLastError();
}

}  // namespace

// row_waves: wavefronts of 32 rows that share a tile, 1, 2 or 4
hipError_t lego_tree_bf16_d64_launch(const TreeArgs& a, int row_waves, hipStream_t stream)
{
  return row_waves == 1 ? launch_rows<1>(a, stream) : row_waves == 2 ? launch_rows<2>(a, stream) : launch_rows<4>(a, stream);
}
