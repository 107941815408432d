// generated by lego_amd (python -m lego_amd.build) -- do not edit; edit the generator
//
// Attention of drafted tokens over a paged cache, bf16, up to 64 head elements: a draft sees all cached keys of its sequence and the drafts that the tree shows
// it.  One draft a sequence is ordinary decoding.
// Bound by memory where drafts are few: every cached key and value is read once for all drafts and all query heads that share its head.  Those are the rows of an item, 32 to a
// wavefront.  Sequences have any length, so the tiles of all items, one after another, are dealt out in equal runs, whatever item they belong to; an item within one run is done there, the sums of one
// in several are joined by a second kernel, in their order.  With few tiles an item a workgroup takes an item, in one launch.
// Scores are transposed as in the forward kernel: a row to a lane of each half.  Tiles go from memory into LDS without passing registers; a piece of the sequence's table of pages is kept there too.
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

constexpr float kLazy = 8.0f;
constexpr unsigned RING = 4;      // operands read ahead

// Tiles of a sequence's items
struct Sequence { unsigned length, cached, tiles; };      // (its keys, tiles of them, and with the drafts')

__device__ __forceinline__ Sequence sequence_of(const TreeArgs& a, unsigned b)
{
  const unsigned most = (unsigned)a.width * (unsigned)a.page, keys = a.tile;
  const unsigned length = (unsigned)min((unsigned)max(a.lengths[b], 0), most), cached = (length + keys - 1) / keys;
  return {length, cached, cached + (a.k ? ((unsigned)a.drafts + keys - 1) / keys : 0u)};
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

__device__ __forceinline__ unsigned run_of(const TreeArgs& a, unsigned total) { return max(a.least, (total + a.runs - 1) / a.runs); }

// N memory->LDS instructions of this wavefront may be on their way
template <unsigned N>
__device__ __forceinline__ void wait_for_copies_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// what this wavefront has asked of LDS is done: a copy may go where it was read
__device__ __forceinline__ void wait_for_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

constexpr unsigned NW = 4;                     // wavefronts of a workgroup
constexpr unsigned PIECE = 1024;               // entries of a page table in LDS

// Where keys and values lie, in 16-byte chunks: 32 bits of every product are enough, they are all that is left of the sum, which lies in what the strides reach.  Read once and held: as fields of the
// arguments they are fetched one after the other at every tile (a first token 7.5 -> 7.0 us, a decoding step of 32 sequences 108 -> 106).
struct Rows {
  unsigned outer, row, head;      // from a page (a sequence) to the next one, from a token, from a head
  __device__ __forceinline__ Rows(const Strides& by) : outer((unsigned)(by.batch >> 3)), row((unsigned)(by.token >> 3)), head((unsigned)(by.head >> 3))
  {
    asm volatile("" : "+s"(outer), "+s"(row), "+s"(head));
  }
};

// A row of a tile, as the lane knows it that looks it up: 16-byte chunks from the base of what it lies in.
struct Place { unsigned k, v; bool there; };
__device__ __forceinline__ Place place_of(const TreeArgs& a, const Rows& k, const Rows& v, const Rows& dk, const Rows& dv, unsigned b, unsigned hk, const Sequence& seq, const int* table, unsigned piece,
                                          unsigned entries, bool cached, unsigned key)
{
  if (!cached) {
    const bool there = key < (unsigned)a.drafts;
    const unsigned row = there ? key : 0u;
    return {there ? b * dk.outer + row * dk.row + hk * dk.head : 0u, there ? b * dv.outer + row * dv.row + hk * dv.head : 0u, there};
  }
  const unsigned at = quotient(key, a.page_factor, a.page_shift), row = key - at * (unsigned)a.page;
  const int page = page_of(table, entries, a.count, key < seq.length, at - piece);
  const bool there = page >= 0;
  return {there ? (unsigned)page * k.outer + row * k.row + hk * k.head : 0u, there ? (unsigned)page * v.outer + row * v.row + hk * v.head : 0u, there};
}

// Copy number g of a tile: 1 KiB of the rows' chunks.  Every instruction has all its lanes, so that each counts for one: a row that is not there reads the base's first one, and a chunk past
// the head its row's last one, which meets zeros of Q and gives columns that nobody stores.  The lane's row of the copy is asked for (row_of_copy) well before its place is used.
__device__ __forceinline__ unsigned row_of_copy(unsigned own, unsigned g, unsigned lane) { return __shfl(own, 8*g + ((lane)/(8))); }
__device__ __forceinline__ void copy_row(const void* base, unsigned at, unsigned g, unsigned lane, unsigned head, unsigned lds)
{
  const unsigned chunk = ((lane % 8) ^ ((2*g + ((lane)/(32))) % 4 + 4*(((lane)/(16)) % 2)));
  const char* const from = static_cast<const char*>(base) + (size_t)at * 16 + min(16 * chunk, 2 * head - 16);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds + g * 1024) : "memory", "m0");
}

// Up to 32 rows: a workgroup's tiles of an item are shared out among its wavefronts, and each goes through its own by itself, with no other one to wait for, in tiles of 32 keys; eight of them and more
// on a CU keep the memory busy.  The keys of the next tile come while the products with the present values are formed, its values while those with the keys are.  The sums meet in LDS at the end.
// A step of 32 sequences of 37 to 8192 tokens, 32 bf16 heads of 128 to 8 (537 MB of keys and values): 107 us, 5.0 TB/s, and 7 us for the join; with wavefronts that share tiles behind barriers 135 us.
template <bool CAP, bool BIAS>
__global__ void __launch_bounds__(64 * NW, 2) lego_tree_few_bf16_d64_kernel(TreeArgs a)
{
  constexpr unsigned HALF = TILE / 2, FILLS = HALF / 1024;      // bytes of 32 rows; copies
  __shared__ __attribute__((aligned(1024))) char lds[NW][2 * HALF];
  __shared__ int pages_s[NW][PIECE / NW];
  __shared__ float2 stats_s[NW][64];
  const unsigned lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l32 = lane % 32, lhi = lane / 32;
  const unsigned group = a.heads / a.key_heads, rows = group * a.drafts, items = a.key_heads;
  const Reader read(lane);
  typedef __attribute__((address_space(3))) void* lds_ptr;
  char *const kt = lds[wave], *const vt = kt + HALF;
  const unsigned lds_at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr)lds + wave * (2 * HALF));
  int* const table = pages_s[wave];
  constexpr bool RAW = !CAP && !BIAS;
  const float unit = RAW ? fabsf(a.scores.scale_log2) : 1.0f, lazy = kLazy / unit;

  const Rows cache_k(a.skc), cache_v(a.svc), draft_k(a.sk), draft_v(a.sv);
  const void *k_cache = a.k_cache, *v_cache = a.v_cache;
  asm volatile("" : "+s"(k_cache), "+s"(v_cache));
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

  while (true) {
    const unsigned hk = item, count = min(left, seq.tiles - tile), share = (count + NW - 1) / NW;      // tiles of this item, and of a wavefront
    const unsigned own_first = tile + min(wave * share, count), last = tile + min((wave + 1) * share, count);
    const bool mine = l32 < rows;
    const unsigned t = min(l32, rows - 1) / group, h = hk * group + min(l32, rows - 1) % group;
    elt8 qv[KS];
    {
      const elt_t* const row = static_cast<const elt_t*>(a.q) + (size_t)b * a.sq.batch + (size_t)t * a.sq.token + (size_t)h * a.sq.head;
#pragma unroll
      for (unsigned ks = 0; ks < KS; ++ks) {
        const unsigned d = 16 * ks + 8 * lhi;
        qv[ks] = d < (unsigned)a.head ? *reinterpret_cast<const elt8*>(row + d) : elt8{};
        if (RAW && a.scores.scale_log2 < 0.0f) qv[ks] = -qv[ks];
      }
    }
    const int* const pages = a.pages + (size_t)b * a.width;
    const float slope = BIAS ? kLog2e * a.slopes[h] : 0.0f;
    const int position = BIAS ? (a.positions ? a.positions[(size_t)b * a.drafts + t] : (int)(seq.length + t)) : 0;
    const unsigned char* const shown = a.tree ? a.tree + (size_t)b * a.tree_batch + (size_t)t * a.drafts : nullptr;

    unsigned piece = 0, piece_end = 0;      // entries of the table in LDS
    unsigned next_k[FILLS], next_v[FILLS], next_here = 0;      // of the next tile: the lane's rows, and which there are
    const auto look_up = [&](unsigned n) __attribute__((always_inline)) {
      const bool cached = n < seq.cached;
      if (cached) {
        const unsigned after = quotient(min(32 * n + 31, seq.length - 1), a.page_factor, a.page_shift) + 1;
        if (after > piece_end) {
          piece = quotient(32 * n, a.page_factor, a.page_shift);
          piece_end = min(piece + PIECE / NW, (unsigned)a.width);
          wait_for_reads();
          for (unsigned i = lane; i < piece_end - piece; i += 64) table[i] = pages[piece + i];
          __builtin_amdgcn_wave_barrier();
        }
      }
      const Place place = place_of(a, cache_k, cache_v, draft_k, draft_v, b, hk, seq, table, piece, piece_end - piece, cached, 32 * (cached ? n : n - seq.cached) + l32);
      next_here = (unsigned)__builtin_amdgcn_ballot_w64(place.there);
#pragma unroll
      for (unsigned g = 0; g < FILLS; ++g) next_k[g] = row_of_copy(place.k, g, lane), next_v[g] = row_of_copy(place.v, g, lane);
    };
    const auto fill = [&](unsigned n, const unsigned* from, bool values) __attribute__((always_inline)) {
      const void* const base = n < seq.cached ? (values ? v_cache : k_cache) : (values ? a.v : a.k);
#pragma unroll
      for (unsigned g = 0; g < FILLS; ++g) copy_row(base, from[g], g, lane, a.head, lds_at + (values ? HALF : 0));
    };

    float16v acc[DB];
#pragma unroll
    for (unsigned db = 0; db < DB; ++db) acc[db] = zeros();
    float most = -INFINITY, sum = 0.0f;
    wait_for_copies();      // nothing of what came before is counted
    if (own_first < last) {
      look_up(own_first);
      fill(own_first, next_k, false);
      fill(own_first, next_v, true);
    }
    for (unsigned n = own_first; n < last; ++n) {
      const unsigned here = next_here;
      const bool more = n + 1 < last, cached = n < seq.cached;
      if (more) look_up(n + 1);
      wait_for_copies_but<FILLS>();
      float16v s = zeros();
#pragma unroll
      for (unsigned ks = 0; ks < KS; ++ks) s = mfma(read.rows(kt, 0, ks), qv[ks], s);
      LEGO_READS(4);
#pragma unroll
      for (unsigned i = 0; i < KS - 4; ++i) {
        LEGO_MFMAS(1);
        LEGO_READS(1);
      }
      LEGO_MFMAS(4);
      __builtin_amdgcn_sched_barrier(0);
      wait_for_reads();
      if (more) fill(n + 1, next_k, false);
      const int first = (int)(32 * (cached ? n : n - seq.cached));
      if (!RAW) {
        const float distance0 = (float)(position - first - 4 * (int)lhi);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x = score<CAP>(s[e], a.scores);
          if (BIAS && cached) x -= slope * fabsf(distance0 - (float)(8 * (e / 4) + e % 4));
          s[e] = x;
        }
      }
      // what of the cache's tile is not there, and what the tree hides
      if (!cached) {
        int j0 = first + 4 * (int)lhi;
        asm volatile("" : "+v"(j0));      // nothing of this is made ahead of the branch
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = j0 + 8 * (e / 4) + e % 4;
          const bool inside = j < a.drafts;
          const bool seen = inside && (shown ? shown[inside ? j : 0] != 0 : j <= (int)t);
          float x = s[e];
          if (BIAS) x -= slope * fabsf((float)(position - (a.positions ? a.positions[(size_t)b * a.drafts + (inside ? j : 0)] : (int)seq.length + j)));
          s[e] = seen ? x : -INFINITY;
        }
      } else if (here != ~0u) {
        const unsigned own = here >> (4 * lhi);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = own >> (8 * (e / 4) + e % 4) & 1 ? s[e] : -INFINITY;
      }
      float top = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
      top = across_max(top);
      if (__builtin_amdgcn_ballot_w64(top > most + lazy) != 0) {
        const float risen = fmaxf(most, top), factor = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(unit * (most - risen));
        most = risen;
        sum *= factor;
#pragma unroll
        for (unsigned db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[db][e] *= factor;
      }
      const float base = most == -INFINITY ? 0.0f : unit * most;
      float sums[4] = {sum, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(RAW ? __builtin_fmaf(unit, s[e], -base) : s[e] - base);
        sums[e % 4] += s[e];
      }
      sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
      const Operands p = as_operands(s);
      if (more) wait_for_copies_but<FILLS>();
      else wait_for_copies();
      if (here != ~0u) {      // values that are not there are zeros: whatever was read in their place, times a P of zero
#pragma unroll
        for (unsigned at = lane; at < HALF / 16; at += 64)
          if (!(here >> (at / (PITCH / 8)) & 1)) reinterpret_cast<u32x4*>(vt)[at] = u32x4{0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (unsigned j = 0; j < 2 * DB; ++j) acc[j % DB] = mfma(read.transposed(vt, j / DB, j % DB), p.step[j / DB], acc[j % DB]);
      LEGO_READS(6);
#pragma unroll
      for (unsigned j = 0; j < 2 * DB - 3; ++j) {
        LEGO_MFMAS(1);
        LEGO_READS(2);
      }
      LEGO_MFMAS(3);
      __builtin_amdgcn_sched_barrier(0);
      wait_for_reads();
      if (more) fill(n + 1, next_v, true);
    }
    sum = across_sum(sum);
    most *= unit;      // in units of log2 from here on
    // every wavefront's sums into its own place, then each joins blocks of 32 elements of the head
    float4v* const own = reinterpret_cast<float4v*>(lds[wave]);
    static_assert(64 * 16 * DB * 4 <= 2 * HALF, "a wavefront's sums in its tiles' place");
#pragma unroll
    for (unsigned db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) own[(4 * db + g) * 64 + lane] = float4v{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
    stats_s[wave][lane] = float2{most, sum};
    __syncthreads();
    if (wave < DB) {
      float all = 0.0f, factor[NW];
      most = -INFINITY;
#pragma unroll
      for (unsigned w = 0; w < NW; ++w) most = fmaxf(most, stats_s[w][lane].x);
#pragma unroll
      for (unsigned w = 0; w < NW; ++w) {
        const float2 o = stats_s[w][lane];
        factor[w] = o.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(o.x - most);
        all += factor[w] * o.y;
      }
      float16v joined[1] = {zeros()};
#pragma unroll
      for (unsigned w = 0; w < NW; ++w)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4v x = reinterpret_cast<const float4v*>(lds[w])[(4 * wave + g) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) joined[0][4 * g + e] += factor[w] * x[e];
        }
      if (count == seq.tiles) {
        elt_t* const row = static_cast<elt_t*>(a.o) + (size_t)b * a.so.batch + (size_t)t * a.so.token + (size_t)h * a.so.head + 32 * wave;
        store_columns<1>(joined, mine && 32 * wave < (unsigned)a.head ? row : nullptr, lane, a.head - min(32 * wave, (unsigned)a.head), all == 0.0f ? 0.0f : 1.0f / all);
      } else if (mine) {      // slot: the workgroup's number and the item's, which no two parts share
        const size_t at = ((size_t)blockIdx.x + (size_t)b * items + item) * 32 + l32;
        if (lhi == 0 && wave == 0) a.stats[at] = float2{most, all};
        float* const to = a.sums + at * DC + 32 * wave;
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4v*>(to + 8 * g + 4 * lhi) = float4v{joined[0][4 * g], joined[0][4 * g + 1], joined[0][4 * g + 2], joined[0][4 * g + 3]};
      }
    }
    left -= count;
    if (left == 0) return;
    __syncthreads();      // the tiles' places are free again
    tile = 0;
    if (++item == items) {
      item = 0;
      do seq = sequence_of(a, ++b);
      while (seq.tiles == 0);
    }
  }
}

// More rows: wavefronts of 32 rows share tiles of 64 keys, two pairs of them or four.
// 8 sequences of 1021 to 16384 tokens, trees of 48 drafts, 32 bf16 heads of 128 to 8, capped (285 MB of keys and values, 55 GFLOP): 167 us and 19 for the join, MFMA 22 % busy, vector unit 53 %.  The
// forward kernel takes nearly as long for dense tensors that come from memory as these do (32 x 256 rows of 8 heads, 8192 keys: 470 us, and 546 here).  Two blocks of 128 rows for 192: three of 64, which
// waste none, take 240 us, as they have each tile of keys brought to LDS for half as many rows.
template <bool CAP, bool BIAS, unsigned RW>
__global__ void __launch_bounds__(64 * NW, 2) lego_tree_many_bf16_d64_kernel(TreeArgs a)
{
  constexpr unsigned STAGES = 2, KW = RW == 4 ? 1 : 2, NB = 2 / KW, FILLS = TILE / 1024 / NW;
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * 2 * TILE];      // K and V, STAGES times
  __shared__ int pages_s[PIECE];
  const unsigned lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l32 = lane % 32, lhi = lane / 32;
  const unsigned rw = wave % RW, kw = wave / RW;
  const unsigned group = a.heads / a.key_heads, rows = group * a.drafts, items = a.key_heads;
  const Reader read(lane);
  typedef __attribute__((address_space(3))) void* lds_ptr;
  const unsigned lds_at = (unsigned)(uintptr_t)(lds_ptr)lds;

  const Rows cache_k(a.skc), cache_v(a.svc), draft_k(a.sk), draft_v(a.sv);
  const void *k_cache = a.k_cache, *v_cache = a.v_cache;
  asm volatile("" : "+s"(k_cache), "+s"(v_cache));
  unsigned b, item, tile, left;      // the present sequence, item of it, tile of that; tiles of the run that are left
  Sequence seq;
  // the workgroups of a run, one for each block of its rows, are 8 apart: they go over its tiles side by side on one XCD, whose L2 the later ones find them in
  const unsigned at8 = blockIdx.x / 8, worker = at8 / a.row_blocks * 8 + blockIdx.x % 8, rb = at8 % a.row_blocks;
  if (a.whole) {
    if (worker >= (unsigned)a.batch * items) return;
    b = worker / items;
    item = worker % items;
    seq = sequence_of(a, b);
    tile = 0;
    left = seq.tiles;
  } else {
    const unsigned total = total_tiles(a, lane, items), run = run_of(a, total), first = worker * run;
    if (worker >= a.runs || first >= total) return;
    left = min(run, total - first);
    unsigned before;
    b = find_sequence(a, lane, items, first, before);
    seq = sequence_of(a, b);
    item = (first - before) / seq.tiles;
    tile = (first - before) % seq.tiles;
  }

  do {
    const unsigned hk = item;
    const unsigned count = min(left, seq.tiles - tile), last = tile + count;      // tiles of this item
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
        if (!CAP && !BIAS && a.scores.scale_log2 < 0.0f) qv[ks] = -qv[ks];
      }
    }
    const int* const pages = a.pages + (size_t)b * a.width;
    const float slope = BIAS ? kLog2e * a.slopes[h] : 0.0f;
    const int position = BIAS ? (a.positions ? a.positions[(size_t)b * a.drafts + t] : (int)(seq.length + t)) : 0;
    const unsigned char* const shown = a.tree ? a.tree + (size_t)b * a.tree_batch + (size_t)t * a.drafts : nullptr;

    unsigned piece = 0, piece_end = 0;      // entries of the table that pages_s holds
    unsigned next_k[FILLS], next_v[FILLS];      // of the tile that is copied next: the lane's rows, and which there are
    unsigned long long next_here = 0;
    const auto look_up = [&](unsigned n) __attribute__((always_inline)) {
      const bool cached = n < seq.cached;
      if (cached) {
        const unsigned after = quotient(min(64 * n + 63, seq.length - 1), a.page_factor, a.page_shift) + 1;
        if (after > piece_end) {      // the table's next piece (uniform: all wavefronts come here together)
          __syncthreads();
          piece = quotient(64 * n, a.page_factor, a.page_shift);
          piece_end = min(piece + PIECE, (unsigned)a.width);
          for (unsigned i = threadIdx.x; i < piece_end - piece; i += 64 * NW) pages_s[i] = pages[piece + i];
          __syncthreads();
        }
      }
      const Place place = place_of(a, cache_k, cache_v, draft_k, draft_v, b, hk, seq, pages_s, piece, piece_end - piece, cached, 64 * (cached ? n : n - seq.cached) + lane);
      next_here = __builtin_amdgcn_ballot_w64(place.there);
#pragma unroll
      for (unsigned it = 0; it < FILLS; ++it) next_k[it] = row_of_copy(place.k, it * NW + wave, lane), next_v[it] = row_of_copy(place.v, it * NW + wave, lane);
    };
    const auto fill = [&](unsigned n, unsigned stage, bool values) __attribute__((always_inline)) {
      const void* const base = n < seq.cached ? (values ? v_cache : k_cache) : (values ? a.v : a.k);
#pragma unroll
      for (unsigned it = 0; it < FILLS; ++it)
        copy_row(base, values ? next_v[it] : next_k[it], it * NW + wave, lane, a.head, lds_at + stage * (2 * TILE) + (values ? TILE : 0));
    };

    // as in the forward kernel: the running maximum is of the products themselves where nothing but the scale comes in between
    constexpr bool RAW = !CAP && !BIAS;
    const float unit = RAW ? fabsf(a.scores.scale_log2) : 1.0f, lazy = kLazy / unit;
    float16v acc[DB];
#pragma unroll
    for (unsigned db = 0; db < DB; ++db) acc[db] = zeros();
    float most = -INFINITY, sum = 0.0f;
    unsigned stage = 0;
    // Copies are asked for in the order K(n), V(n), K(n + 1), V(n + 1): the keys of the tile after the next one when those of this tile have been read, the values of the next tile when those of
    // the last one have.  So two of them are on their way behind the one that is waited for, and each has one and a half tiles' time.
    unsigned long long here = 0, here1 = 0;      // rows that are there, of this tile and of the next one
    wait_for_copies();
    if (tile < last) {
      look_up(tile);
      fill(tile, 0, false);
      fill(tile, 0, true);
      here = next_here;
      if (tile + 1 < last) {
        look_up(tile + 1);
        fill(tile + 1, 1, false);
      }
    }
    for (unsigned n = tile; n < last; ++n) {
      if (n + 1 < last) wait_for_copies_but<2 * FILLS>();
      else wait_for_copies_but<FILLS>();
      __syncthreads();      // the keys are there, and the values before these have been read
      here1 = next_here;
      if (n + 1 < last) fill(n + 1, stage ^ 1, true);
      if (n + 2 < last) look_up(n + 2);
      __builtin_amdgcn_sched_barrier(0);
      char* const kt = lds + stage * (2 * TILE);
      char* const vt = kt + TILE;
      const bool cached = n < seq.cached;
      const int first = (int)(64 * (cached ? n : n - seq.cached)) + (int)(32 * NB * kw);      // of this wavefront's keys
      float16v s[NB];
#pragma unroll
      for (unsigned i = 0; i < NB; ++i) s[i] = zeros();
#pragma unroll
      for (unsigned ks = 0; ks < KS; ++ks)
#pragma unroll
        for (unsigned i = 0; i < NB; ++i) s[i] = mfma(read.rows(kt, NB * kw + i, ks), qv[ks], s[i]);
      constexpr unsigned ROW_READS = KS * NB, FIRST_READS = ROW_READS < 6 ? ROW_READS : 6;
      LEGO_READS(FIRST_READS);
#pragma unroll
      for (unsigned i = 0; i < (ROW_READS - FIRST_READS) / 2; ++i) {
        LEGO_MFMAS(2);
        LEGO_READS(2);
      }
      LEGO_MFMAS(FIRST_READS);
      __builtin_amdgcn_sched_barrier(0);
      if (n + 1 < last) wait_for_copies_but<2 * FILLS>();
      else wait_for_copies();
      __syncthreads();      // the values are there, and the keys have been read
      if (n + 2 < last) fill(n + 2, stage, false);
      stage ^= 1;
      if (here != ~0ull) {      // values that are not there are zeros: whatever was read in their place, times a P of zero
#pragma unroll
        for (unsigned at = threadIdx.x; at < TILE / 16; at += 64 * NW)
          if (!(here >> (at / (PITCH / 8)) & 1)) reinterpret_cast<u32x4*>(vt)[at] = u32x4{0u, 0u, 0u, 0u};
        __syncthreads();
      }
      const auto operand = [&](unsigned j) { return read.transposed(vt, 2 * NB * kw + j / DB, j % DB); };
      elt8 ahead[RING];      // operands of the second products, on their way meanwhile
#pragma unroll
      for (unsigned j = 0; j < RING; ++j) ahead[j] = operand(j);
      __builtin_amdgcn_sched_barrier(0);
      if (!RAW) {
        const float distance0 = (float)(position - first - 4 * (int)lhi);
#pragma unroll
        for (unsigned i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x = score<CAP>(s[i][e], a.scores);
            if (BIAS && cached) x -= slope * fabsf(distance0 - (float)(int)(32 * i + 8 * (e / 4) + e % 4));
            s[i][e] = x;
          }
      }
      // what of the cache's tile is not there, and what the tree hides
      if (!cached) {
        int j0 = first + 4 * (int)lhi;
        asm volatile("" : "+v"(j0));      // nothing of this is made ahead of the branch
#pragma unroll
        for (unsigned i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int j = j0 + (int)(32 * i + 8 * (e / 4)) + e % 4;
            const bool inside = j < a.drafts;
            const bool seen = inside && (shown ? shown[inside ? j : 0] != 0 : j <= (int)t);
            float x = s[i][e];
            if (BIAS) x -= slope * fabsf((float)(position - (a.positions ? a.positions[(size_t)b * a.drafts + (inside ? j : 0)] : (int)seq.length + j)));
            s[i][e] = seen ? x : -INFINITY;
          }
      } else if (here != ~0ull) {
        const unsigned long long own = here >> (32 * NB * kw + 4 * lhi);
#pragma unroll
        for (unsigned i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[i][e] = own >> (32 * i + 8 * (e / 4) + e % 4) & 1 ? s[i][e] : -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (unsigned i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[i][e]);
      top = across_max(top);
      if (__builtin_amdgcn_ballot_w64(top > most + lazy) != 0) {
        const float risen = fmaxf(most, top), factor = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(unit * (most - risen));
        most = risen;
        sum *= factor;
#pragma unroll
        for (unsigned db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[db][e] *= factor;
      }
      const float base = most == -INFINITY ? 0.0f : unit * most;
      float sums[4] = {sum, 0.0f, 0.0f, 0.0f};
      const auto exponential = [&](unsigned i, int e) {
        s[i][e] = __builtin_amdgcn_exp2f(RAW ? __builtin_fmaf(unit, s[i][e], -base) : s[i][e] - base);
        sums[e % 4] += s[i][e];
      };
#pragma unroll
      for (int e = 0; e < 16; ++e) exponential(0, e);
      Operands p = as_operands(s[0]);
      __builtin_amdgcn_sched_barrier(0);
      // every product has its slot, with the operand of the one RING further on and a part of what the second half of the keys needs
#pragma unroll
      for (unsigned j = 0; j < 2 * NB * DB; ++j) {
        if (j == 2 * DB) p = as_operands(s[NB - 1]);
        acc[j % DB] = mfma(ahead[j % RING], p.step[j / DB % 2], acc[j % DB]);
        if (j + RING < 2 * NB * DB) ahead[j % RING] = operand(j + RING);
        if (NB == 2 && j < 2 * DB) {
#pragma unroll
          for (int e = (int)(16 * j / (2 * DB)); e < (int)(16 * (j + 1) / (2 * DB)); ++e) exponential(NB - 1, e);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
      here = here1;
    }
    sum = across_sum(sum);
    most *= unit;      // in units of log2 from here on
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
      } else {      // slot: the run's number and the item's, which no two parts share
        const size_t slot = (size_t)worker + (size_t)b * items + item;
        const size_t at = (slot * a.row_blocks + rb) * (32 * RW) + 32 * rw + l32;
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
    __syncthreads();      // the tiles' place and the table's are free again
    tile = 0;
    if (++item == items) {
      item = 0;
      do seq = sequence_of(a, ++b);
      while (seq.tiles == 0);
    }
  } while (true);
}

// The rows of items in several runs, and of those that have no tile, `share` rows of an item a workgroup: a few parts of several rows are gone through by the lanes of each row, others by teams of lanes, a row
// after the other.  Either order is the same whenever the lengths are.
__global__ void __launch_bounds__(256) lego_tree_join_bf16_d64_kernel(TreeArgs a, unsigned held_rows, unsigned share, unsigned chunks)
{
  constexpr unsigned LANES = DC / 4 > 16 ? 32 : 16, TEAMS = 256 / LANES;
  __shared__ float4v sums_s[TEAMS][LANES];
  __shared__ float sum_s[TEAMS], most_s[4];
  const unsigned lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const unsigned group = a.heads / a.key_heads, rows = group * a.drafts, items = a.key_heads;
  const unsigned chunk = blockIdx.x % chunks, item = blockIdx.x / chunks % items, b = blockIdx.x / chunks / items;
  const unsigned begin = chunk * share, end = min(begin + share, rows);
  const unsigned tiles = sequence_of(a, b).tiles, total = total_tiles(a, lane, items), run = run_of(a, total), first = tiles_before(a, lane, items, b) + item * tiles;
  const auto row_at = [&](unsigned i) {
    const unsigned t = i / group, h = item * group + i % group;
    return static_cast<elt_t*>(a.o) + (size_t)b * a.so.batch + (size_t)t * a.so.token + (size_t)h * a.so.head + 4 * c;
  };
  const unsigned w0 = tiles ? first / run : 0, parts = tiles ? (first + tiles - 1) / run - w0 + 1 : 0;
  if (parts == 1) return;
  const size_t place0 = ((size_t)w0 + (size_t)b * items + item) * held_rows;      // parts are held_rows apart
  const auto store = [&](unsigned i, float sum, const float4v& x) {
    const float factor = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (4 * c < (unsigned)a.head) *reinterpret_cast<u32x2*>(row_at(i)) = u32x2{pack(factor * x[0], factor * x[1]), pack(factor * x[2], factor * x[3])};
  };
  const auto add = [&](size_t place, float most, float& sum, float4v& x) {
    const float2 stat = a.stats[place];
    const float f = stat.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(stat.x - most);
    sum += f * stat.y;
    if (4 * c < DC) x += f * *reinterpret_cast<const float4v*>(a.sums + place * DC + 4 * c);
  };
  if (share > 1 && parts <= 8) {
    for (unsigned i = begin + team; i < end; i += TEAMS) {
      float most = -INFINITY, sum = 0.0f;
      float4v x = {0.0f, 0.0f, 0.0f, 0.0f};
      for (unsigned p = 0; p < parts; ++p) most = fmaxf(most, a.stats[place0 + i + (size_t)p * held_rows].x);
#pragma unroll 2
      for (unsigned p = 0; p < parts; ++p) add(place0 + i + (size_t)p * held_rows, most, sum, x);
      store(i, sum, x);
    }
    return;
  }
  for (unsigned i = begin; i < end; ++i) {
    float most = -INFINITY, sum = 0.0f;
    float4v x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (unsigned p = threadIdx.x; p < parts; p += 256) most = fmaxf(most, a.stats[place0 + i + (size_t)p * held_rows].x);
#pragma unroll
    for (int d = 32; d; d /= 2) most = fmaxf(most, __shfl_xor(most, d));
    if (lane == 0) most_s[wave] = most;
    __syncthreads();
    most = fmaxf(fmaxf(most_s[0], most_s[1]), fmaxf(most_s[2], most_s[3]));
#pragma unroll 4
    for (unsigned p = team; p < parts; p += TEAMS) add(place0 + i + (size_t)p * held_rows, most, sum, x);
    sums_s[team][c] = x;
    if (c == 0) sum_s[team] = sum;
    __syncthreads();
    if (team == 0) {
#pragma unroll
      for (unsigned o = 1; o < TEAMS; ++o) {
        x += sums_s[o][c];
        sum += sum_s[o];
      }
      store(i, sum, x);
    }
  }
}

}  // namespace

// row_waves: wavefronts of 32 rows that share a tile, 1, 2 or 4
hipError_t lego_tree_bf16_d64_launch(const TreeArgs& a, int row_waves, hipStream_t stream)
{
  const auto launch = [&](auto kernel) {
    const unsigned workers = a.whole ? (unsigned)(a.batch * a.key_heads) : a.runs, grid = a.row_blocks == 1 ? workers : (workers + 7) / 8 * 8 * a.row_blocks;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * NW), 0, stream, a);
    return hipGetLastError();
  };
  hipError_t e = hipErrorInvalidValue;
  if ((a.capped != 0) == true && (a.slopes != nullptr) == true)
    e = row_waves == 1 ? launch(lego_tree_few_bf16_d64_kernel<true, true>)
        : row_waves == 2 ? launch(lego_tree_many_bf16_d64_kernel<true, true, 2>) : launch(lego_tree_many_bf16_d64_kernel<true, true, 4>);
  if ((a.capped != 0) == true && (a.slopes != nullptr) == false)
    e = row_waves == 1 ? launch(lego_tree_few_bf16_d64_kernel<true, false>)
        : row_waves == 2 ? launch(lego_tree_many_bf16_d64_kernel<true, false, 2>) : launch(lego_tree_many_bf16_d64_kernel<true, false, 4>);
  if ((a.capped != 0) == false && (a.slopes != nullptr) == true)
    e = row_waves == 1 ? launch(lego_tree_few_bf16_d64_kernel<false, true>)
        : row_waves == 2 ? launch(lego_tree_many_bf16_d64_kernel<false, true, 2>) : launch(lego_tree_many_bf16_d64_kernel<false, true, 4>);
  if ((a.capped != 0) == false && (a.slopes != nullptr) == false)
    e = row_waves == 1 ? launch(lego_tree_few_bf16_d64_kernel<false, false>)
        : row_waves == 2 ? launch(lego_tree_many_bf16_d64_kernel<false, false, 2>) : launch(lego_tree_many_bf16_d64_kernel<false, false, 4>);
  if (e != hipSuccess || a.whole) return e;
  // One row a workgroup while they are few, and have many parts each; 8 of many rows share the search for their parts.
  const unsigned rows = (unsigned)(a.drafts * (a.heads / a.key_heads)), share = (unsigned)(a.batch * a.key_heads) * rows <= 4096 ? 1 : 8, chunks = (rows + share - 1) / share;
  hipLaunchKernelGGL(lego_tree_join_bf16_d64_kernel, dim3((unsigned)(a.batch * a.key_heads) * chunks), dim3(256), 0, stream, a, 32u * (unsigned)row_waves * a.row_blocks, share, chunks);
  return hipGetLastError();
}
