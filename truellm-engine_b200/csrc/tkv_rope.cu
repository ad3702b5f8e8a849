// tkv_rope.cu -- rotary positions with several axes on queries and keys.
//
// Pair i of a head's first rotary_dim channels is turned by the angle
// positions[axis(i)][token] * theta^(-2 i / rotary_dim).  The product is formed
// and reduced in 64 bits as revolutions (position * turns, minus its whole
// part), so a far position loses nothing to the reduction; sine and cosine of
// the rest are 32-bit, and each output is rounded once to the input's type.
//
// A CTA takes TOK tokens: its threads compute the sines and cosines of the
// tokens' pairs into shared memory, once for all q and k heads and while the
// first vectors are on their way, then each thread turns pieces of 8 pairs (two
// 16-byte vectors), one (token, head) after another with the next one loaded
// ahead.  Bound by memory, a read and a write of every element: 32771 tokens of 40
// heads of 128 channels in 123 us, 5.5 TB/s (one token a CTA: 166 us; loads not
// ahead: 141 us).
#include <math.h>

#include "tkv_int8.cuh"

namespace tkv {
namespace {

constexpr int kRopeThreads = 256;

template <int TOK, bool BF16>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ tkv_rope_plan_t plan,
                                                            const RopeArgs a) {
  __shared__ float4 cs[TOK][TKV_ROPE_MAX_PAIRS / 2];  // two pairs' (cos, sin)
  const int half = plan.rotary_dim / 2, t0 = blockIdx.x * TOK, toks = min(TOK, a.n_tokens - t0);
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, nthr = blockDim.x * blockDim.y;
  // unit u of a row: pairs 8 u .. 8 u + 7 while they last, then 16 channels to copy
  const int u = threadIdx.x, rot_units = half / 8;
  const bool turn = u < rot_units, halves = plan.pairing == TKV_ROPE_HALVES;
  const int lo = turn ? (halves ? 8 * u : 16 * u) : 16 * u;
  const int hi = turn && halves ? half + 8 * u : lo + 8;
  const bool two = hi < a.head_dim;  // an odd number of copied vectors ends with one
  const int heads = a.hq + a.hk;
  auto load = [&](int j, int h, uint4& x, uint4& y) {
    const int t = t0 + j;
    const uint16_t* src =
        h < a.hq ? a.q + t * a.q_t + h * a.q_h : a.k + t * a.k_t + (h - a.hq) * a.k_h;
    x = *reinterpret_cast<const uint4*>(src + lo);
    if (two) y = *reinterpret_cast<const uint4*>(src + hi);
  };
  // a thread's rows: (token j, head h) in steps of blockDim.y heads, the next one's
  // vectors always on their way; the first while the angles are computed
  uint4 nx = make_uint4(0, 0, 0, 0), ny = nx;
  int nj = 0, nh = threadIdx.y;
  while (nh >= heads) nh -= heads, ++nj;
  if (nj < toks) load(nj, nh, nx, ny);
  for (int e = tid; e < half * toks; e += nthr) {
    const int j = e / half, p = e - j * half;
    const double rev =
        __ldg(a.positions + plan.axis[p] * a.axis_stride + t0 + j) * plan.turns[p];
    float sn, cn;
    sincospif(2.f * static_cast<float>(rev - rint(rev)), &sn, &cn);
    reinterpret_cast<float2*>(cs[j])[p] = make_float2(cn, a.inverse ? -sn : sn);
  }
  __syncthreads();
  while (nj < toks) {
    const int j = nj, h = nh;
    uint4 x = nx, y = ny;
    nh += blockDim.y;
    while (nh >= heads) nh -= heads, ++nj;
    if (nj < toks) load(nj, nh, nx, ny);
    if (turn) {
      float2 f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 g = cs[j][4 * u + e];
        f[2 * e] = make_float2(g.x, g.y);
        f[2 * e + 1] = make_float2(g.z, g.w);
      }
      uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (halves) {
          const float2 p = unpack2<BF16>(xw[e]), r = unpack2<BF16>(yw[e]);
          const float2 c0 = f[2 * e], c1 = f[2 * e + 1];
          xw[e] = pack2<BF16>(p.x * c0.x - r.x * c0.y, p.y * c1.x - r.y * c1.y);
          yw[e] = pack2<BF16>(r.x * c0.x + p.x * c0.y, r.y * c1.x + p.y * c1.y);
        } else {
          const float2 p = unpack2<BF16>(xw[e]), r = unpack2<BF16>(yw[e]);
          const float2 c0 = f[e], c1 = f[4 + e];
          xw[e] = pack2<BF16>(p.x * c0.x - p.y * c0.y, p.y * c0.x + p.x * c0.y);
          yw[e] = pack2<BF16>(r.x * c1.x - r.y * c1.y, r.y * c1.x + r.x * c1.y);
        }
      }
      x = make_uint4(xw[0], xw[1], xw[2], xw[3]);
      y = make_uint4(yw[0], yw[1], yw[2], yw[3]);
    }
    const int t = t0 + j;
    uint16_t* dst = h < a.hq ? a.q_out + t * a.qo_t + h * a.qo_h
                             : a.k_out + t * a.ko_t + (h - a.hq) * a.ko_h;
    *reinterpret_cast<uint4*>(dst + lo) = x;
    if (two) *reinterpret_cast<uint4*>(dst + hi) = y;
  }
}

template <int TOK>
void launch_t(const tkv_rope_plan_t& plan, const RopeArgs& a, bool bf16, cudaStream_t stream) {
  const int units = (a.head_dim + 15) / 16;
  const dim3 block(units, kRopeThreads / units);
  const unsigned int grid = (a.n_tokens - 1) / TOK + 1;
  if (bf16)
    rope_kernel<TOK, true><<<grid, block, 0, stream>>>(plan, a);
  else
    rope_kernel<TOK, false><<<grid, block, 0, stream>>>(plan, a);
}

}  // namespace

int launch_rope(const tkv_rope_plan_t& plan, const RopeArgs& a, bool bf16, cudaStream_t stream) {
  // One token a CTA where there are few, four from 1024 on.  Measured, 40 heads of 128,
  // one and four tokens a CTA: 256 tokens 3.6 and 5.0 us, 1024 tokens 7.9 and 6.9, 16384
  // tokens 85.7 and 66.4.
  if (a.n_tokens < 1024)
    launch_t<1>(plan, a, bf16, stream);
  else
    launch_t<4>(plan, a, bf16, stream);
  return cudaGetLastError() == cudaSuccess ? TKV_OK : TKV_BACKEND_ERROR;
}

}  // namespace tkv
