// generated by lego_amd (python -m lego_amd.build) -- do not edit; edit the generator
//
// The passes over rows beside the attention kernels: the lowest and highest document of every 64 positions; sum of out * dout of every query, what its scores are lessened by, with
// the power of two that brings the largest dout of 64 queries to 1..2; and the sum of the parts of dk and dv.  Each reads its input once.
// Index expressions printed from LEGO layouts:
//   statistics   OrderBy(Row(batch, heads, queries)).TileBy([batch, heads, queries])[b, h, i]
//   parts        OrderBy(Row(parts, 2, batch, key heads, keys, head))
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_args.h"

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

// One wavefront a tile.
__global__ void __launch_bounds__(256) lego_attention_tiles_kernel(const int* __restrict__ documents, int2* __restrict__ tiles, unsigned batch, unsigned keys)
{
  const unsigned per = (keys + 63) / 64, at = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x % 64;
  if (at >= batch * per) return;
  const unsigned b = at / per, key = min(64 * (at % per) + lane, keys - 1);
  int low = documents[(size_t)b * keys + key], high = low;
#pragma unroll
  for (int d = 32; d; d /= 2) {
    low = min(low, __shfl_xor(low, d));
    high = max(high, __shfl_xor(high, d));
  }
  if (lane == 0) tiles[at] = int2{low, high};
}

// The blocks of 128 queries (blockIdx.y 0) or keys (1) of a batch by the tiles that they share a document with, the most first.  A launch of few rounds of workgroups ends when its last heavy one does: for
// 16 heads of 8192 tokens in 7 documents, 1024 workgroups in two rounds, forward 98 -> 84 us, dk and dv 191 -> 167, dq 146 -> 129 at 6 a launch.
__global__ void __launch_bounds__(1024) lego_attention_order_kernel(AttentionArgs a)
{
  __shared__ unsigned work_s[512];
  const unsigned b = blockIdx.x, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const bool of_keys = blockIdx.y != 0;
  int* const order = of_keys ? a.order_keys : a.order_queries;
  if (!order) return;
  const int rows = of_keys ? a.keys : a.queries, shift = a.keys - a.queries, prefix = a.causal ? (a.prefix ? max(a.prefix[b], 0) : 0) : a.keys;
  const unsigned blocks = (unsigned)(rows + 127) / 128;
  const int tiles = (a.keys + 63) / 64;
  const int2* const at = a.tiles + (size_t)b * tiles;
  for (unsigned block = wave; block < blocks; block += 16) {
    const int r0 = (int)(128 * block), r1 = min(r0 + 128, rows) - 1, p0 = of_keys ? r0 : r0 + shift, p1 = of_keys ? r1 : r1 + shift;      // rows, positions
    int2 own = at[p0 / 64];
    for (int t = p0 / 64 + 1; t <= p1 / 64; ++t) own = int2{min(own.x, at[t].x), max(own.y, at[t].y)};
    const int begin = of_keys ? max(p0 < prefix ? 0 : p0, shift) / 64 : 0, end = of_keys ? tiles : (min(a.keys, max(p1 + 1, prefix)) + 63) / 64;
    unsigned work = 0;
    for (int base = begin; base < end; base += 64) {
      const int t = base + (int)lane;
      const int2 other = t < end ? at[t] : int2{0, -1};
      work += __popcll(__ballot(!(other.y < 0 || own.y < 0 || other.y < own.x || own.y < other.x)));
    }
    if (lane == 0) work_s[block] = work;
  }
  __syncthreads();
  if (threadIdx.x >= blocks) return;
  const unsigned own = work_s[threadIdx.x];
  unsigned rank = 0;
  for (unsigned j = 0; j < blocks; ++j) rank += work_s[j] > own || (work_s[j] == own && j < threadIdx.x);
  order[b * blocks + rank] = (int)threadIdx.x;
}

// 64 queries of a head a workgroup, 16 lanes a query: 100 MB of out, its rest and dout in 18 us (2 x 16 heads of 128, 4096 tokens), 5.6 TB/s.
template <class E>
__global__ void __launch_bounds__(256) lego_attention_delta_kernel(AttentionArgs a, unsigned tiles, float shift)
{
  typedef E elt8 __attribute__((ext_vector_type(8)));
  __shared__ float largest_s[4];
  const unsigned tile = blockIdx.x % tiles, h = blockIdx.x / tiles % a.heads, b = blockIdx.x / tiles / a.heads;
  const unsigned lane = threadIdx.x % 16, team = threadIdx.x / 16;
  const E* const out = static_cast<const E*>(a.out) + (size_t)b * a.so.batch + (size_t)h * a.so.head;
  const E* const rest = a.rest ? static_cast<const E*>(a.rest) + (size_t)b * a.so.batch + (size_t)h * a.so.head : nullptr;
  const E* const dout = static_cast<const E*>(a.dout) + (size_t)b * a.sdo.batch + (size_t)h * a.sdo.head;
  float largest = 0.0f;
#pragma unroll
  for (unsigned it = 0; it < 4; ++it) {
    const unsigned i = 64 * tile + 16 * it + team;
    const bool inside = i < (unsigned)a.queries;
    float sum = 0.0f;
    const size_t stat = a.heads*a.queries*(size_t)b + a.queries*h + i;
    const bool empty = !inside || a.lse[stat] == -INFINITY;      // a query that sees nothing gives no gradient, whatever its dout holds
    if (!empty && 8 * lane < (unsigned)a.head) {
      const elt8 x = *reinterpret_cast<const elt8*>(out + (size_t)i * a.so.token + 8 * lane), y = *reinterpret_cast<const elt8*>(dout + (size_t)i * a.sdo.token + 8 * lane);
      const elt8 less = rest ? *reinterpret_cast<const elt8*>(rest + (size_t)i * a.so.token + 8 * lane) : elt8{};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum += ((float)x[e] + (float)less[e]) * (float)y[e];
        largest = fmaxf(largest, fabsf((float)y[e]));
      }
    }
#pragma unroll
    for (int d = 8; d; d /= 2) sum += __shfl_xor(sum, d);
    if (lane == 0 && inside) {
      a.delta[stat] = -sum;
      const float less = shift - 1.4426950408889634f * a.lse[stat];
      a.less[stat] = a.capped ? less + a.scores.cap_log2 : less * a.scores.unscale;
    }
  }
#pragma unroll
  for (int d = 32; d; d /= 2) largest = fmaxf(largest, __shfl_xor(largest, d));
  if (threadIdx.x % 64 == 0) largest_s[threadIdx.x / 64] = largest;
  __syncthreads();
  if (threadIdx.x == 0) {
    largest = fmaxf(fmaxf(largest_s[0], largest_s[1]), fmaxf(largest_s[2], largest_s[3]));
    a.ups[((size_t)b * a.heads + h) * tiles + tile] = largest > 0.0f && largest < INFINITY ? ldexpf(1.0f, 1 - __builtin_amdgcn_frexp_expf(largest)) : 1.0f;
  }
}

// Eight elements of dk or dv a lane, the parts summed in their order: four of 34 MB in 24 us (2 x 4 key heads of 128, 4096 tokens), 5.9 TB/s with what is written.
template <class E>
__global__ void __launch_bounds__(256) lego_attention_join_kernel(AttentionArgs a, unsigned parts)
{
  typedef E elt8 __attribute__((ext_vector_type(8)));
  const size_t chunks = (size_t)a.batch * a.key_heads * a.keys * (a.head / 8), at = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= 2 * chunks) return;
  const unsigned which = at >= chunks;
  const size_t chunk = at - which * chunks;
  const unsigned per_row = a.head / 8, c = chunk % per_row;
  const size_t row = chunk / per_row;
  float4v lo = {0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
  for (unsigned part = 0; part < parts; ++part) {
    const float* const from = a.parts + ((2 * part + which) * chunks + chunk) * 8;
    lo += *reinterpret_cast<const float4v*>(from);
    hi += *reinterpret_cast<const float4v*>(from + 4);
  }
  const unsigned key = row % a.keys, hk = row / a.keys % a.key_heads, b = row / a.keys / a.key_heads;
  const Strides& s = which ? a.sdv : a.sdk;
  elt8 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = static_cast<E>(lo[e]);
    v[4 + e] = static_cast<E>(hi[e]);
  }
  *reinterpret_cast<elt8*>(static_cast<E*>(which ? a.dv : a.dk) + (size_t)b * s.batch + (size_t)key * s.token + (size_t)hk * s.head + 8 * c) = v;
}

}  // namespace

hipError_t lego_attention_tiles_launch(const int* documents, int2* tiles, int batch, int keys, hipStream_t stream)
{
  const unsigned count = (unsigned)batch * (((unsigned)keys + 63) / 64);
  hipLaunchKernelGGL(lego_attention_tiles_kernel, dim3((count + 3) / 4), dim3(256), 0, stream, documents, tiles, (unsigned)batch, (unsigned)keys);
  return hipGetLastError();
}

hipError_t lego_attention_order_launch(const AttentionArgs& a, hipStream_t stream)
{
  hipLaunchKernelGGL(lego_attention_order_kernel, dim3((unsigned)a.batch, 2), dim3(1024), 0, stream, a);
  return hipGetLastError();
}

hipError_t lego_attention_delta_launch(const AttentionArgs& a, int element, hipStream_t stream)
{
  const unsigned tiles = ((unsigned)a.queries + 63) / 64;
  const dim3 grid(tiles * (unsigned)a.heads * (unsigned)a.batch);
  if (element == 0) hipLaunchKernelGGL(lego_attention_delta_kernel<_Float16>, grid, dim3(256), 0, stream, a, tiles, 8.0f);
  else hipLaunchKernelGGL(lego_attention_delta_kernel<__bf16>, grid, dim3(256), 0, stream, a, tiles, 0.0f);
  return hipGetLastError();
}

hipError_t lego_attention_join_launch(const AttentionArgs& a, int element, hipStream_t stream)
{
  const unsigned parts = (unsigned)(a.heads / a.key_heads / a.heads_per_part);
  const unsigned long long chunks = 2ull * a.batch * a.key_heads * a.keys * (a.head / 8);
  const dim3 grid((unsigned)((chunks + 255) / 256));
  if (element == 0) hipLaunchKernelGGL(lego_attention_join_kernel<_Float16>, grid, dim3(256), 0, stream, a, parts);
  else hipLaunchKernelGGL(lego_attention_join_kernel<__bf16>, grid, dim3(256), 0, stream, a, parts);
  return hipGetLastError();
}
