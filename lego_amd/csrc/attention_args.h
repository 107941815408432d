// What the attention kernels' launchers take from the entry points.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// rows of one tensor: elements between batches, tokens and heads
struct Strides { long long batch, token, head; };

// the score function's constants
struct Scores {
  float scale, scale_log2;      // of q.k; times log2 e
  float unscale;                // 1 / scale_log2
  float cap_in, cap_log2;       // 2 scale log2(e) / cap; cap log2(e)
};

struct AttentionArgs {
  const void *q, *k, *v, *out, *rest, *dout;
  void *o, *o_rest, *dq, *dk, *dv;      // rest: what rounding took from out, laid out as out, or null
  float* lse;                   // [batch][head][query], natural logarithm
  float* delta;                 // the same, of the backward pass: - sum of out * dout
  float* less;                  // what the backward pass adds to a score: a power's exponent less log2(e) lse; with a cap that too, without one over scale_log2, as a sum starts at it
  float* ups;                   // [batch][head][tile of 64 queries]: power of two that brings the tile's largest dout to 1..2
  const float* slopes;          // [head], or null
  const int* documents;         // [batch][key], or null
  int2* tiles;                  // [batch][tile of 64 keys]: lowest and highest document
  int *order_queries, *order_keys;      // [batch][block of 128]: the blocks with the most work first, or null: as they come
  const int* prefix;            // [batch], or null
  float* parts;                 // dk and dv of parts of the query heads that share a key head: [part][dk, dv][batch][key head][key][head element], or null
  Strides sq, sk, sv, so, sdo, sdq, sdk, sdv;
  Scores scores;
  int batch, queries, keys, heads, key_heads, head;
  int causal, capped;
  int heads_per_part;           // query heads whose sums one workgroup forms
  int halve_queries, halve_keys;      // workgroups of 64 and not 128 of them, whose wavefronts share the tiles out in halves
};

struct RotaryArgs {
  const void *q, *k;
  void *qo, *ko;
  const void* positions;        // 32 or 64 bits
  const double* frequencies;    // radians a position, [part / 2]
  long long position_batch, position_token;      // elements between positions
  Strides sq, sk, sqo, sko;
  unsigned batch, tokens, heads, key_heads, head, part;
  float magnitude;
  int inverse;
};

// Attention of drafted tokens over a paged cache.
struct TreeArgs {
  const void *q, *k, *v;        // the drafts; k and v may be null
  const void *k_cache, *v_cache;
  void* o;
  const int* pages;             // [batch][width]
  const int* lengths;           // [batch]
  const unsigned char* tree;    // [batch][draft][draft], or null: a draft sees itself and the earlier ones
  const float* slopes;          // [head], or null
  const int* positions;         // [batch][draft], or null: length + draft
  float* sums;                  // of parts of rows: [slot][row][head element]
  float2* stats;                // [slot][row]: maximum (log2) and sum
  Strides sq, sk, sv, so, skc, svc;      // of the caches: between pages, slots of a page and heads
  long long tree_batch;
  Scores scores;
  int batch, drafts, heads, key_heads, head, page, count, width;
  int capped, whole;            // whole: a workgroup goes through all keys of an item
  unsigned row_blocks;          // of a key head's rows, drafts * (heads / key_heads)
  unsigned tile;                // keys of a tile
  unsigned runs, least;         // runs at most; tiles of a run at least
  unsigned page_factor, page_shift;
};

#ifdef __HIPCC__
#define LEGO_HOST_DEVICE __host__ __device__
#else
#define LEGO_HOST_DEVICE
#endif

// Quotients by the page's tokens, of whole numbers below 2^31, as one product and a shift: with 2^l the first power of two that is not below the divisor, the factor ceil(2^(31 + l) / divisor) is off by
// less than 2^l / divisor ulps of 2^-31, which below 2^31 never reaches the next whole quotient; and it is below 2^32.
static inline void quotients_by(unsigned divisor, unsigned& factor, unsigned& shift)
{
  shift = 31;
  while ((1ull << (shift - 31)) < divisor) ++shift;
  factor = (unsigned)(((unsigned __int128)1 << shift) / divisor + ((((unsigned __int128)1 << shift) % divisor) != 0));
}
static inline LEGO_HOST_DEVICE unsigned quotient(unsigned x, unsigned factor, unsigned shift) { return (unsigned)(((unsigned long long)x * factor) >> shift); }

// The page of a cached key by entry `at` of a piece of `entries` of its sequence's table: -1 where the key is not there, or the table names no page of the cache.
static inline LEGO_HOST_DEVICE int page_of(const int* table, unsigned entries, unsigned count, bool within, unsigned at)
{
  if (!within || at >= entries) return -1;
  const int page = table[at];
  return page >= 0 && (unsigned)page < count ? page : -1;
}
