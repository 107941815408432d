// C-ABI entry points of the attention operators (declared in include/lego_hip.h).  Written by hand, as lego_hip_abi.hip is: an entry point checks what
// the generated kernels assume and enqueues them on the caller's stream.  It allocates nothing and never synchronises.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "attention_args.h"
#include "generated/launchers.h"
#include "lego_hip.h"

namespace {

constexpr int kInvalid = static_cast<int>(hipErrorInvalidValue);
constexpr long long kMostTokens = 1ll << 28;
// bytes between tokens: a tile of 64 lies within a descriptor's 2 GiB
constexpr long long kMostPitch = (1ll << 31) / 2 / 64 - LEGO_ATTENTION_MAX_HEAD;

inline bool aligned16(const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }
inline size_t up16(size_t n) { return (n + 15) / 16 * 16; }

// strides of one tensor: whole 16-byte chunks
inline bool take(Strides& s, const long long* three)
{
  s = {three[0], three[1], three[2]};
  for (int i = 0; i < 3; ++i)
    if (three[i] < 0 || three[i] % 8) return false;
  return s.token <= kMostPitch;
}

inline bool take_sizes(AttentionArgs& a, const long long* sizes)
{
  if (!sizes) return false;
  for (int i = 0; i < 6; ++i)
    if (sizes[i] < 1 || sizes[i] > kMostTokens) return false;
  a.batch = (int)sizes[0], a.queries = (int)sizes[1], a.keys = (int)sizes[2], a.heads = (int)sizes[3], a.key_heads = (int)sizes[4], a.head = (int)sizes[5];
  if (a.heads % a.key_heads || a.head % 8 || a.head > LEGO_ATTENTION_MAX_HEAD) return false;
  // workgroups of a launch, the finest being 64 queries of a head
  const unsigned __int128 tiles = ((unsigned __int128)(a.queries > a.keys ? a.queries : a.keys) + 63) / 64;
  return tiles * a.heads * a.batch < (1u << 30) && (unsigned __int128)a.batch * a.key_heads * a.keys * a.head < ((unsigned __int128)1 << 38);
}

inline Scores scores_of(float scale, float softcap)
{
  const float log2e = 1.4426950408889634f;
  const float steep = fabsf(scale * log2e) < 1e-30f ? copysignf(1e-30f, scale) : scale * log2e;      // a scale of nothing: differences of nothing
  return {scale, steep, 1.0f / steep, softcap > 0.0f ? 2.0f * scale * log2e / softcap : 0.0f, softcap * log2e};
}

inline bool take_mask(AttentionArgs& a, float scale, float softcap, const float* slopes, const int* documents, const int* prefix, int causal)
{
  if (!(fabsf(scale) < INFINITY) || !(softcap >= 0.0f && softcap < INFINITY) || (causal != 0 && causal != 1)) return false;
  if (!aligned4(slopes) || !aligned4(documents) || !aligned4(prefix) || (prefix && !causal) || (documents && a.keys < a.queries)) return false;
  a.scores = scores_of(scale, softcap);
  a.capped = softcap > 0.0f;
  a.slopes = slopes, a.documents = documents, a.prefix = prefix, a.causal = causal;
  return true;
}

inline size_t tiles_bytes(const AttentionArgs& a) { return up16((size_t)a.batch * ((a.keys + 63) / 64) * sizeof(int2)); }

// Query heads of a group whose dk and dv one workgroup sums.  All of them where that leaves enough workgroups; else fewer, whose sums go through memory: the more so the shorter the sequences are.
// Enough are 1024 or, up to 1024 keys, 256.  Backward pass, bf16 heads of 128, 32 of them to 8: one sequence of 4096 tokens 559 us with 1024, 589 with 256; one of 5000 783 and 1083; four of 1024 227 and 184.
inline int heads_per_part(const AttentionArgs& a)
{
  const int group = a.heads / a.key_heads;
  const long long blocks = (long long)((a.keys + 127) / 128) * a.key_heads * a.batch, enough = a.keys <= 1024 ? 256 : 1024;
  for (int parts = 1; parts <= group; ++parts)
    if (group % parts == 0 && blocks * parts >= enough) return group / parts;
  return 1;
}

// As many workgroups of 128 rows as the chip holds with twice the tiles in LDS, or fewer: half of the rows each, and the tiles in turn for the halves of the wavefronts, so that a row's way through the
// other side is half as long.  Measured, causal with slopes, forward + backward, us.  fp16 heads of 64: 4 of 1531 tokens, 48 workgroups, 30.5 + 82 -> 19.8 + 54; 36 of them, 432, 39 + 97 -> 33 + 86; 64
// of them, 768, 43 + 118 -> 47 + 128, not cut.  bf16 heads of 128: 4 of 1531 tokens, 39 + 122 -> 28 + 74; 4 of 8192, 256 workgroups, 232 + 592 -> 154 + 378; 36 of 1531, 432, 51 + 158 -> 68 + 172, not cut.
inline bool halve(const AttentionArgs& a, int rows, long long heads) { return (rows + 127) / 128 * heads <= (a.head <= 64 ? 512 : 256); }

// With documents the blocks' work follows no rule: where there are several rounds of workgroups, but not so many that the last one counts for little, they are ordered by it.
inline bool ordered(int rows) { return (rows + 127) / 128 <= LEGO_ATTENTION_ORDERED; }

inline void plan_attention(AttentionArgs& a)
{
  a.heads_per_part = heads_per_part(a);
  a.halve_queries = halve(a, a.queries, (long long)a.heads * a.batch);
  a.halve_keys = halve(a, a.keys, (long long)(a.heads / a.heads_per_part) * a.batch);
}

struct Room { size_t order_queries, order_keys, delta, less, ups, parts, all; };
inline Room room_of(const AttentionArgs& a, bool documents, bool backward)
{
  Room r = {};
  const bool queries = documents && !a.halve_queries && ordered(a.queries), keys = documents && backward && !a.halve_keys && ordered(a.keys);
  r.order_queries = documents ? tiles_bytes(a) : 0;
  r.order_keys = r.order_queries + (queries ? up16((size_t)a.batch * ((a.queries + 127) / 128) * sizeof(int)) : 0);
  r.delta = r.all = r.order_keys + (keys ? up16((size_t)a.batch * ((a.keys + 127) / 128) * sizeof(int)) : 0);
  if (!backward) return r;
  const size_t rows = (size_t)a.batch * a.heads;
  r.less = r.delta + up16(rows * a.queries * sizeof(float));
  r.ups = r.less + up16(rows * a.queries * sizeof(float));
  r.parts = r.ups + up16(rows * ((a.queries + 63) / 64) * sizeof(float));
  const int parts = a.heads / a.key_heads / a.heads_per_part;
  r.all = r.parts + (parts > 1 ? (size_t)parts * 2 * a.batch * a.key_heads * a.keys * a.head * sizeof(float) : 0);
  return r;
}

// The passes over the documents, before the kernels that use them.
inline hipError_t look_at_documents(AttentionArgs& a, const Room& room, void* workspace, hipStream_t stream)
{
  char* const at = static_cast<char*>(workspace);
  a.tiles = reinterpret_cast<int2*>(at);
  a.order_queries = room.order_keys > room.order_queries ? reinterpret_cast<int*>(at + room.order_queries) : nullptr;
  a.order_keys = room.delta > room.order_keys ? reinterpret_cast<int*>(at + room.order_keys) : nullptr;
  const hipError_t e = lego_attention_tiles_launch(a.documents, a.tiles, a.batch, a.keys, stream);
  return e != hipSuccess || !(a.order_queries || a.order_keys) ? e : lego_attention_order_launch(a, stream);
}

inline hipError_t forward(const AttentionArgs& a, int element, hipStream_t stream)
{
  const int which = a.head <= 64 ? 0 : a.head <= 96 ? 1 : 2;
  static hipError_t (*const launch[2][3])(const AttentionArgs&, hipStream_t) = {
    {lego_attention_fwd_f16_d64_launch, lego_attention_fwd_f16_d96_launch, lego_attention_fwd_f16_d128_launch},
    {lego_attention_fwd_bf16_d64_launch, lego_attention_fwd_bf16_d96_launch, lego_attention_fwd_bf16_d128_launch}};
  return launch[element][which](a, stream);
}

inline hipError_t backward(const AttentionArgs& a, int element, hipStream_t stream)
{
  const int which = a.head <= 64 ? 0 : a.head <= 96 ? 1 : 2;
  static hipError_t (*const launch[2][3])(const AttentionArgs&, hipStream_t) = {
    {lego_attention_bwd_f16_d64_launch, lego_attention_bwd_f16_d96_launch, lego_attention_bwd_f16_d128_launch},
    {lego_attention_bwd_bf16_d64_launch, lego_attention_bwd_bf16_d96_launch, lego_attention_bwd_bf16_d128_launch}};
  return launch[element][which](a, stream);
}

// Launch of attention over a cache: wavefronts of 32 rows that share a tile, and what a launch in runs needs.
struct TreePlan { int row_waves; size_t stats, all; };
inline bool plan_of(TreeArgs& a, const long long* sizes, TreePlan& plan)
{
  if (!sizes) return false;
  for (int i = 0; i < 8; ++i)
    if (sizes[i] < 1 || sizes[i] > kMostTokens) return false;
  a.batch = (int)sizes[0], a.drafts = (int)sizes[1], a.heads = (int)sizes[2], a.key_heads = (int)sizes[3], a.head = (int)sizes[4];
  a.page = (int)sizes[5], a.count = (int)sizes[6], a.width = (int)sizes[7];
  if (a.heads % a.key_heads || a.head % 8 || a.head > LEGO_ATTENTION_MAX_HEAD) return false;
  const unsigned __int128 keys = (unsigned __int128)a.page * a.width + a.drafts, all_rows = (unsigned __int128)a.batch * a.heads * a.drafts;
  if (keys > (unsigned)kMostTokens || all_rows > (1u << 30)) return false;
  const unsigned rows = (unsigned)a.drafts * (unsigned)(a.heads / a.key_heads);
  plan.row_waves = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  const unsigned block = 32 * plan.row_waves;
  a.row_blocks = (rows + block - 1) / block;
  a.tile = plan.row_waves == 1 ? 32 : 64;
  const unsigned long long items = (unsigned long long)a.batch * a.key_heads;
  const unsigned long long most = ((unsigned long long)a.page * a.width + a.tile - 1) / a.tile + ((unsigned)a.drafts + a.tile - 1) / a.tile;
  if (items * most >= (1ull << 31)) return false;
  // An item of few tiles is one workgroup's, and there is nothing to join; of more, where there are enough items.  Else the tiles are dealt in equal runs to as many workgroups as the chip holds at a time,
  // but no run is shorter than a tile or two a wavefront.  One launch / runs and join, fp16 heads of 64, four to a key head, us: one token, 4 items of 1000 keys 12.2 / 13.2, of 1500 15.4 / 10.7, 256 items
  // of 2000 keys 26 / 36; 24 drafts, 4 items of 375 16.3 / 17.2, of 500 19.1 / 17.2, 64 of 750 25 / 27, of 1000 31 / 29, 256 of 2000 58 / 62.
  a.least = plan.row_waves == 1 ? 2 * LEGO_TREE_LEAST : LEGO_TREE_LEAST;
  const unsigned long long blocks = items * a.row_blocks;
  a.whole = most <= (plan.row_waves == 1 ? (blocks >= 256 ? 65 : 33) : blocks >= 256 ? 33 : blocks >= 64 ? 13 : 7);
  const unsigned long long chip = plan.row_waves == 1 && a.head <= 64 ? 768 : 512, held = chip > a.row_blocks ? chip / a.row_blocks : 1, runs = (items * most + a.least - 1) / a.least;
  a.runs = (unsigned)(runs < held ? runs : held);
  quotients_by((unsigned)a.page, a.page_factor, a.page_shift);
  plan.stats = plan.all = 0;
  if (a.whole) return true;
  const unsigned pitch = a.head <= 64 ? 64 : a.head <= 96 ? 96 : 128;
  const size_t slots = (size_t)a.runs + items;
  plan.stats = slots * a.row_blocks * block * pitch * sizeof(float);
  plan.all = plan.stats + slots * a.row_blocks * block * sizeof(float2);
  return true;
}

}  // namespace

extern "C" {

int lego_hip_tree_attention_workspace_bytes(const long long* sizes, unsigned long long* bytes)
{
  TreeArgs a = {};
  TreePlan plan;
  if (!bytes || !plan_of(a, sizes, plan)) return kInvalid;
  *bytes = plan.all;
  return 0;
}

int lego_hip_tree_attention(const void* q, const void* k, const void* v, const void* k_cache, const void* v_cache, void* out, const int* pages, const int* lengths,
                            const unsigned char* tree, const float* slopes, const int* positions, const long long* sizes, const long long* strides, float scale,
                            float softcap, int element, void* workspace, unsigned long long workspace_bytes, void* stream)
{
  TreeArgs a = {};
  TreePlan plan;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) || !pages || !lengths || !strides || element < 0 || element > 1) return kInvalid;
  if ((k == nullptr) != (v == nullptr) || (k && (!aligned16(k) || !aligned16(v))) || (!k && tree)) return kInvalid;
  if (!aligned4(pages) || !aligned4(lengths) || !aligned4(slopes) || !aligned4(positions) || (positions && !slopes) || !plan_of(a, sizes, plan)) return kInvalid;
  if (!(fabsf(scale) < INFINITY) || !(softcap >= 0.0f && softcap < INFINITY)) return kInvalid;
  Strides* const into[6] = {&a.sq, &a.sk, &a.sv, &a.skc, &a.svc, &a.so};
  const long long count[6][3] = {{a.batch, a.drafts, a.heads}, {a.batch, a.drafts, a.key_heads}, {a.batch, a.drafts, a.key_heads}, {a.count, a.page, a.key_heads},
                                 {a.count, a.page, a.key_heads}, {a.batch, a.drafts, a.heads}};
  for (int t = 0; t < 6; ++t) {
    *into[t] = {strides[3 * t], strides[3 * t + 1], strides[3 * t + 2]};
    unsigned __int128 extent = 0;
    for (int i = 0; i < 3; ++i) {
      if (strides[3 * t + i] < 0 || strides[3 * t + i] % 8) return kInvalid;
      extent += (unsigned __int128)strides[3 * t + i] * (count[t][i] - 1);
    }
    if (extent / 8 + LEGO_ATTENTION_MAX_HEAD / 8 >= 0xffffffffu && t > 0 && t < 5) return kInvalid;      // rows are told apart by 32 bits of 16-byte chunks
  }
  a.tree_batch = strides[18];
  if (a.tree_batch < 0) return kInvalid;
  if (plan.all && (!aligned16(workspace) || workspace_bytes < plan.all)) return kInvalid;
  const float log2e = 1.4426950408889634f;
  const float steep = fabsf(scale * log2e) < 1e-30f ? copysignf(1e-30f, scale) : scale * log2e;      // a scale of nothing: differences of nothing
  a.scores = {scale, steep, 1.0f / steep, softcap > 0.0f ? 2.0f * scale * log2e / softcap : 0.0f, softcap * log2e};
  a.capped = softcap > 0.0f;
  a.q = q, a.k = k, a.v = v, a.k_cache = k_cache, a.v_cache = v_cache, a.o = out, a.pages = pages, a.lengths = lengths, a.tree = tree, a.slopes = slopes, a.positions = positions;
  a.sums = static_cast<float*>(workspace);
  a.stats = reinterpret_cast<float2*>(static_cast<char*>(workspace) + plan.stats);
  static hipError_t (*const launch[2][3])(const TreeArgs&, int, hipStream_t) = {{lego_tree_f16_d64_launch, lego_tree_f16_d96_launch, lego_tree_f16_d128_launch},
                                                                               {lego_tree_bf16_d64_launch, lego_tree_bf16_d96_launch, lego_tree_bf16_d128_launch}};
  return (int)launch[element][a.head <= 64 ? 0 : a.head <= 96 ? 1 : 2](a, plan.row_waves, as_stream(stream));
}

int lego_hip_attention_workspace_bytes(const long long* sizes, int documents, int backward, unsigned long long* bytes)
{
  AttentionArgs a = {};
  if (!bytes || !take_sizes(a, sizes)) return kInvalid;
  plan_attention(a);
  *bytes = room_of(a, documents != 0, backward != 0).all;
  return 0;
}

int lego_hip_attention_fwd(const void* q, const void* k, const void* v, void* out, void* rest, float* lse, const long long* sizes, const long long* strides, float scale,
                           float softcap, const float* slopes, const int* documents, const int* prefix, int causal, int element, void* workspace,
                           unsigned long long workspace_bytes, void* stream)
{
  AttentionArgs a = {};
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || (rest && !aligned16(rest)) || !lse || !aligned4(lse) || !strides || element < 0 || element > 1) return kInvalid;
  if (!take_sizes(a, sizes) || !take(a.sq, strides) || !take(a.sk, strides + 3) || !take(a.sv, strides + 6) || !take(a.so, strides + 9)) return kInvalid;
  if (!take_mask(a, scale, softcap, slopes, documents, prefix, causal)) return kInvalid;
  plan_attention(a);
  const Room room = room_of(a, documents != nullptr, false);
  if (documents && (!aligned16(workspace) || workspace_bytes < room.all)) return kInvalid;
  a.q = q, a.k = k, a.v = v, a.o = out, a.o_rest = rest, a.lse = lse;
  const hipError_t e = documents ? look_at_documents(a, room, workspace, as_stream(stream)) : hipSuccess;
  return e != hipSuccess ? (int)e : (int)forward(a, element, as_stream(stream));
}

int lego_hip_attention_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out, const void* rest, const float* lse, void* dq, void* dk, void* dv,
                           const long long* sizes, const long long* strides, float scale, float softcap, const float* slopes, const int* documents, const int* prefix,
                           int causal, int element, void* workspace, unsigned long long workspace_bytes, void* stream)
{
  AttentionArgs a = {};
  for (const void* p : {dout, q, k, v, out, (const void*)dq, (const void*)dk, (const void*)dv})
    if (!aligned16(p)) return kInvalid;
  if ((rest && !aligned16(rest)) || !lse || !aligned4(lse) || !strides || element < 0 || element > 1 || !take_sizes(a, sizes)) return kInvalid;
  Strides* const into[8] = {&a.sq, &a.sk, &a.sv, &a.so, &a.sdo, &a.sdq, &a.sdk, &a.sdv};
  for (int t = 0; t < 8; ++t)
    if (!take(*into[t], strides + 3 * t)) return kInvalid;
  if (!take_mask(a, scale, softcap, slopes, documents, prefix, causal)) return kInvalid;
  plan_attention(a);
  const Room room = room_of(a, documents != nullptr, true);
  if (!aligned16(workspace) || workspace_bytes < room.all) return kInvalid;
  char* const at = static_cast<char*>(workspace);
  a.q = q, a.k = k, a.v = v, a.out = out, a.rest = rest, a.dout = dout, a.lse = const_cast<float*>(lse), a.dq = dq, a.dk = dk, a.dv = dv;
  a.delta = reinterpret_cast<float*>(at + room.delta), a.less = reinterpret_cast<float*>(at + room.less), a.ups = reinterpret_cast<float*>(at + room.ups);
  a.parts = room.all > room.parts ? reinterpret_cast<float*>(at + room.parts) : nullptr;
  hipError_t e = documents ? look_at_documents(a, room, workspace, as_stream(stream)) : hipSuccess;
  if (e == hipSuccess) e = lego_attention_delta_launch(a, element, as_stream(stream));
  if (e == hipSuccess) e = backward(a, element, as_stream(stream));
  if (e == hipSuccess && a.parts) e = lego_attention_join_launch(a, element, as_stream(stream));
  return (int)e;
}

int lego_hip_rotary(const void* q, const void* k, void* q_out, void* k_out, const void* positions, const double* frequencies, const long long* sizes,
                    const long long* strides, int interleaved, float magnitude, int inverse, int element, int wide_positions, void* stream)
{
  if (!q || !q_out || !positions || !frequencies || !sizes || !strides || element < 0 || element > 2 || (interleaved | inverse | wide_positions) & ~1) return kInvalid;
  const long long key_heads = sizes[3], head = sizes[4], part = sizes[5];
  if (key_heads < 0 || (key_heads > 0) != (k != nullptr) || (k != nullptr) != (k_out != nullptr)) return kInvalid;
  for (int i : {0, 1, 2, 4, 5})
    if (sizes[i] < 1) return kInvalid;
  for (int i = 0; i < 5; ++i)
    if (sizes[i] > kMostTokens) return kInvalid;
  if (part % 2 || part > head || part > LEGO_ROTARY_MAX_PART) return kInvalid;
  for (int i = 0; i < 14; ++i)
    if (strides[i] < 0) return kInvalid;
  // tokens are workgroups; a token's elements are counted in 32 bits
  if ((unsigned __int128)sizes[0] * sizes[1] > (1u << 30) || (unsigned __int128)(sizes[2] + key_heads) * head > (1u << 30)) return kInvalid;
  const unsigned bytes = element == 2 ? 4 : 2, n = 16 / bytes;
  const auto at = [](const void* p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1u)) == 0; };
  bool vectors = head % n == 0 && (interleaved ? part : part / 2) % n == 0;
  for (const void* p : {q, k, (const void*)q_out, (const void*)k_out}) {
    if (!at(p, bytes)) return kInvalid;
    vectors = vectors && at(p, 16);
  }
  if (!at(positions, wide_positions ? 8 : 4) || !at(frequencies, 8)) return kInvalid;
  for (int i = 0; i < 12; ++i) vectors = vectors && (strides[i] % n == 0 || (!k && (i / 3) % 2));
  RotaryArgs a = {};
  a.q = q, a.k = k, a.qo = q_out, a.ko = k_out, a.positions = positions, a.frequencies = frequencies;
  Strides* const into[4] = {&a.sq, &a.sk, &a.sqo, &a.sko};
  for (int t = 0; t < 4; ++t) *into[t] = {strides[3 * t], strides[3 * t + 1], strides[3 * t + 2]};
  a.position_batch = strides[12], a.position_token = strides[13];
  a.batch = (unsigned)sizes[0], a.tokens = (unsigned)sizes[1], a.heads = (unsigned)sizes[2], a.key_heads = (unsigned)key_heads, a.head = (unsigned)head, a.part = (unsigned)part;
  a.magnitude = magnitude, a.inverse = inverse;
  return (int)lego_rotary_launch(a, interleaved, vectors, wide_positions, element, as_stream(stream));
}

}  // extern "C"
