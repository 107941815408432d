// generated by lego_amd (python -m lego_amd.build) -- do not edit; edit the generator
//
// Rotary positions: pairs (a, b) of the first `part` elements of a head become magnitude * (a cos t - b sin t, b cos t + a sin t) with
// t = position * frequency, the other elements are copied; with -t it is the gradient.  Queries and keys in one launch.
// Bound by memory: every element is read and written once, 16384 tokens of 40 bf16 heads of 128 in 60 us, 5.6 TB/s of reads and writes.  A workgroup takes 1 token with all its heads (four of
// them are 5 % faster on inputs from the caches and 9 % slower on inputs from memory), so that a token's angles are computed once, into LDS: the product in 64 bits and reduced to a part of a turn there (a position of a million has lost all its digits in a 32-bit angle), sine and cosine
// of what remains in 32.  A lane then turns one 16-byte vector at a time, or two where a pair's elements lie half the part apart.
// Index expressions printed from LEGO layouts:
//   unit of a token's heads   OrderBy(Row(1, heads, units)).TileBy([1, heads, units]).inv(u)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_args.h"

namespace {

constexpr unsigned kTokens = 1, kThreads = 256, kMostPairs = 256 / 2;

template <class P>
__device__ __forceinline__ void angles(const RotaryArgs& a, unsigned token0, float2 (*turn_s)[kMostPairs])
{
  const unsigned pairs = a.part / 2;
  for (unsigned u = threadIdx.x; u < kTokens * pairs; u += kThreads) {
    const unsigned slot = u / pairs, i = u % pairs, at = token0 + slot;
    if (at >= a.batch * a.tokens) break;
    const long long position = static_cast<const P*>(a.positions)[(size_t)(at / a.tokens) * a.position_batch + (size_t)(at % a.tokens) * a.position_token];
    const double turns = (double)position * a.frequencies[i] * 0.15915494309189535;      // 1 / (2 pi)
    float sine, cosine;
    sincospif((float)(2.0 * (turns - rint(turns))), &sine, &cosine);
    turn_s[slot][i] = float2{a.magnitude * cosine, a.inverse ? -a.magnitude * sine : a.magnitude * sine};
  }
}

__device__ __forceinline__ float2 turned(float x, float y, float2 t) { return float2{x * t.x - y * t.y, y * t.x + x * t.y}; }

// Whole 16-byte vectors of N elements; `half`: pairs half the part apart, which then is a whole number of vectors.
template <class E, class P, bool HALF>
__global__ void __launch_bounds__(kThreads) lego_rotary_kernel(RotaryArgs a)
{
  constexpr unsigned N = 16 / sizeof(E);
  typedef E vec __attribute__((ext_vector_type(N)));
  __shared__ float2 turn_s[kTokens][kMostPairs];
  const unsigned token0 = blockIdx.x * kTokens;
  angles<P>(a, token0, turn_s);
  __syncthreads();
  const unsigned vectors = a.head / N, turning = a.part / N, apart = turning / 2, heads = a.heads + a.key_heads;
  const unsigned units = HALF ? vectors - apart : vectors;      // of a head
  const unsigned slots = min(kTokens, a.batch * a.tokens - token0);
  for (unsigned u = threadIdx.x; u < slots * heads * units; u += kThreads) {
    const unsigned slot = 0, h = ((u)/(units)), c = u % units;
    const unsigned at = token0 + slot, b = at / a.tokens, t = at % a.tokens;
    const bool key = h >= (unsigned)a.heads;
    const unsigned hh = key ? h - a.heads : h;
    const Strides &from = key ? a.sk : a.sq, &to = key ? a.sko : a.sqo;
    const E* const in = static_cast<const E*>(key ? a.k : a.q) + (size_t)b * from.batch + (size_t)t * from.token + (size_t)hh * from.head;
    E* const out = static_cast<E*>(key ? a.ko : a.qo) + (size_t)b * to.batch + (size_t)t * to.token + (size_t)hh * to.head;
    if (HALF) {
      if (c < apart) {
        const vec x = *reinterpret_cast<const vec*>(in + N * c), y = *reinterpret_cast<const vec*>(in + N * (c + apart));
        vec xo, yo;
#pragma unroll
        for (unsigned e = 0; e < N; ++e) {
          const float2 r = turned((float)x[e], (float)y[e], turn_s[slot][N * c + e]);
          xo[e] = static_cast<E>(r.x);
          yo[e] = static_cast<E>(r.y);
        }
        *reinterpret_cast<vec*>(out + N * c) = xo;
        *reinterpret_cast<vec*>(out + N * (c + apart)) = yo;
      } else {
        *reinterpret_cast<vec*>(out + N * (c + apart)) = *reinterpret_cast<const vec*>(in + N * (c + apart));
      }
    } else {
      vec x = *reinterpret_cast<const vec*>(in + N * c);
      if (c < turning) {
#pragma unroll
        for (unsigned e = 0; e < N / 2; ++e) {
          const float2 r = turned((float)x[2 * e], (float)x[2 * e + 1], turn_s[slot][N / 2 * c + e]);
          x[2 * e] = static_cast<E>(r.x);
          x[2 * e + 1] = static_cast<E>(r.y);
        }
      }
      *reinterpret_cast<vec*>(out + N * c) = x;
    }
  }
}

// Any head size, part and alignment, an element or a pair a lane.
template <class E, class P>
__global__ void __launch_bounds__(kThreads) lego_rotary_any_kernel(RotaryArgs a, int half)
{
  __shared__ float2 turn_s[kTokens][kMostPairs];
  const unsigned token0 = blockIdx.x * kTokens;
  angles<P>(a, token0, turn_s);
  __syncthreads();
  const unsigned pairs = a.part / 2, heads = a.heads + a.key_heads, units = a.head - pairs;
  const unsigned slots = min(kTokens, a.batch * a.tokens - token0);
  for (unsigned u = threadIdx.x; u < slots * heads * units; u += kThreads) {
    const unsigned slot = 0, h = ((u)/(units)), c = u % units;
    const unsigned at = token0 + slot, b = at / a.tokens, t = at % a.tokens;
    const bool key = h >= (unsigned)a.heads;
    const unsigned hh = key ? h - a.heads : h;
    const Strides &from = key ? a.sk : a.sq, &to = key ? a.sko : a.sqo;
    const E* const in = static_cast<const E*>(key ? a.k : a.q) + (size_t)b * from.batch + (size_t)t * from.token + (size_t)hh * from.head;
    E* const out = static_cast<E*>(key ? a.ko : a.qo) + (size_t)b * to.batch + (size_t)t * to.token + (size_t)hh * to.head;
    if (c < pairs) {
      const unsigned x = half ? c : 2 * c, y = half ? c + pairs : 2 * c + 1;
      const float2 r = turned((float)in[x], (float)in[y], turn_s[slot][c]);
      out[x] = static_cast<E>(r.x);
      out[y] = static_cast<E>(r.y);
    } else {
      out[c + pairs] = in[c + pairs];
    }
  }
}

template <class E, class P>
hipError_t launch(const RotaryArgs& a, int interleaved, int vectors, hipStream_t stream)
{
  const dim3 grid(((unsigned)a.batch * (unsigned)a.tokens + kTokens - 1) / kTokens);
  if (!vectors) hipLaunchKernelGGL((lego_rotary_any_kernel<E, P>), grid, dim3(kThreads), 0, stream, a, !interleaved);
  else if (interleaved) hipLaunchKernelGGL((lego_rotary_kernel<E, P, false>), grid, dim3(kThreads), 0, stream, a);
  else hipLaunchKernelGGL((lego_rotary_kernel<E, P, true>), grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

template <class E>
hipError_t launch(const RotaryArgs& a, int interleaved, int vectors, int wide, hipStream_t stream)
{
  return wide ? launch<E, long long>(a, interleaved, vectors, stream) : launch<E, int>(a, interleaved, vectors, stream);
}

}  // namespace

// element: 0 f16, 1 bf16, 2 f32.  vectors: bases, strides and sizes are whole 16-byte vectors, and so is the part, or half of it where pairs lie half the part apart.
hipError_t lego_rotary_launch(const RotaryArgs& a, int interleaved, int vectors, int wide, int element, hipStream_t stream)
{
  switch (element) {
    case 0: return launch<_Float16>(a, interleaved, vectors, wide, stream);
    case 1: return launch<__bf16>(a, interleaved, vectors, wide, stream);
    default: return launch<float>(a, interleaved, vectors, wide, stream);
  }
}
