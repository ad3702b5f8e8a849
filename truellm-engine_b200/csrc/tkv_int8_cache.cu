// tkv_int8_cache.cu -- writing the paged int8 cache (quantise on append, the
// reshape_and_cache slot of third_party/vllm_kernels/cache_kernels.cu:202-232)
// and reading it back as dense K/V.
//
// One CTA per (16-token page of a sequence's range, kv head): half of its
// threads take the keys, half the values, one thread per (token, 16 channels).
// Lanes 4 c + i of a warp hold token 4 t + i, chunk c, so the four tokens of a
// V word sit in one quad: a 4 x 4 transpose of words over the quad and of bytes
// within a thread turns four rows into 16-byte units of the V layout (and back).
//
// CTAs are numbered along one axis of page units: sequence s owns the units
// from cu[s] / 16 + 2 s on (a range of n tokens touches at most n / 16 + 2
// pages), so a ragged batch launches (tokens / 16 + 2 sequences) x heads CTAs
// whatever its longest sequence; a CTA finds its sequence by a 32-way search.
#include <limits.h>

#include "tkv_int8.cuh"

namespace tkv {
namespace {

// the last sequence whose first page unit is <= u (all lanes of a warp take part)
__device__ __forceinline__ int find_seq(const int32_t* cu, int num_seqs, long long u) {
  int lo = 0, hi = num_seqs;  // the answer is in [lo, hi)
  const int lane = threadIdx.x & 31;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int s = lo + lane * step;
    const bool le = s < hi && static_cast<long long>(__ldg(cu + s) / kPage) + 2ll * s <= u;
    const unsigned int m = __ballot_sync(0xffffffffu, le);
    // offsets are non-decreasing in a valid call; any answer is in range otherwise
    const int last = m ? 31 - __clz(m) : 0;
    lo += last * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// what a CTA works on: page `page` (index in the sequence) of sequence s, and
// the tokens [t_lo, t_hi) of it, which are rows row + (token - t_lo)
struct PageUnit {
  int s, page, t_lo, t_hi, row;
};

// false: nothing to do.  `lens` holds the first token of each sequence's range.
__device__ __forceinline__ bool page_unit(const int32_t* cu, const int32_t* lens, int num_seqs,
                                          int total, int max_n, int max_blocks, long long u,
                                          PageUnit& p) {
  p.s = find_seq(cu, num_seqs, u);
  const int r0 = __ldg(cu + p.s), n = __ldg(cu + p.s + 1) - r0, pos = __ldg(lens + p.s);
  if (!int8_seq_ok(pos, n, r0, total, max_n, max_blocks)) return false;
  const long long j = u - (static_cast<long long>(r0 / kPage) + 2ll * p.s);
  if (j < 0 || j > INT_MAX / kPage) return false;
  const long long pg = pos / kPage + j;
  if (n == 0 || pg * kPage >= static_cast<long long>(pos) + n) return false;
  p.page = static_cast<int>(pg);
  p.t_lo = max(pos, p.page * kPage);
  p.t_hi = min(pos + n, p.page * kPage + kPage);
  p.row = r0 + (p.t_lo - pos);
  return true;
}

// the length error of every sequence, by the launch's first CTA
__device__ __forceinline__ void flag_lengths(const int32_t* cu, const int32_t* lens, int num_seqs,
                                             int total, int max_n, int max_blocks, int* err) {
  for (int s = threadIdx.x; s < num_seqs; s += blockDim.x)
    if (!int8_seq_ok(lens[s], cu[s + 1] - cu[s], cu[s], total, max_n, max_blocks))
      set_err(err, TKV_ERR_BAD_LENGTH);
}

// Codes (+ 128) of x[0..15] for scale d, packed four to a word.  The sum x/d +
// 1.5 2^23 + 128 rounds to a whole number, halves to even (its bias is even),
// and the low byte of its bits is the stored byte.  x * (1/d) is off by less
// than 2^-15 from x/d, so only a remainder close to one half is checked, in
// exact arithmetic: x - k d is exact in f32 (x has 11 bits or fewer and |x - k
// d| < d, a multiple of d's last bit).
__device__ __forceinline__ void quantise16(const float (&x)[16], float d, float inv,
                                           uint32_t (&w)[4]) {
  constexpr float kMagic = 12582912.f + kInt8Bias;
  float t[16], worst = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    t[e] = __fmaf_rn(x[e], inv, kMagic);
    const float k = __fsub_rn(t[e], kMagic);
    worst = fmaxf(worst, fabsf(__fmaf_rn(x[e], inv, -k)));
  }
  if (worst > 0.4999f) {
    const float h = 0.5f * d;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float k = __fsub_rn(t[e], kMagic);
      const float r = __fmaf_rn(-k, d, x[e]);
      const bool odd = __float_as_uint(t[e]) & 1u;
      if (r > h || (r == h && odd)) t[e] += 1.f;
      if (r < -h || (r == -h && odd)) t[e] -= 1.f;
    }
  }
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const uint32_t lo = __byte_perm(__float_as_uint(t[4 * a]), __float_as_uint(t[4 * a + 1]), 0x0040);
    const uint32_t hi =
        __byte_perm(__float_as_uint(t[4 * a + 2]), __float_as_uint(t[4 * a + 3]), 0x0040);
    w[a] = __byte_perm(lo, hi, 0x5410);
  }
}

// max |x| of 16 packed values; a NaN among them gives NaN
template <bool BF16>
__device__ __forceinline__ float amax16(const uint32_t (&p)[8]) {
  if constexpr (BF16) {
    __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&p[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i)
      m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&p[i])));
    return __bfloat162float(__hmax_nan(m.x, m.y));
  } else {
    __half2 m = __habs2(*reinterpret_cast<const __half2*>(&p[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i)
      m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&p[i])));
    return __half2float(__hmax_nan(m.x, m.y));
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  return a != a ? a : (b != b ? b : fmaxf(a, b));
}

template <int D, bool BF16>
__global__ void __launch_bounds__(2 * D) int8_append_kernel(Int8AppendArgs a) {
  using F = Int8Fmt<D>;
  constexpr int CH = D / 16, HALF = kPage * CH;  // threads per tensor
  const long long u = blockIdx.x / a.n_kv_heads;
  const int h = blockIdx.x % a.n_kv_heads;
  if (blockIdx.x == 0)
    flag_lengths(a.cu, a.lens_old, a.num_seqs, a.total, a.max_new, a.max_blocks, a.err);
  PageUnit p;
  if (!page_unit(a.cu, a.lens_old, a.num_seqs, a.total, a.max_new, a.max_blocks, u, p)) return;
  const int tid = threadIdx.x;
  const bool is_v = tid >= HALF;
  const int r = is_v ? tid - HALF : tid;
  const int i = r & 3, c = (r >> 2) % CH, t4 = r / (4 * CH), tok = 4 * t4 + i;
  const int pid = __ldg(a.block_tables + static_cast<int64_t>(p.s) * a.max_blocks + p.page);
  if (pid < 0 || pid >= a.num_pages) {
    if (tid == 0) set_err(a.err, TKV_ERR_BAD_PAGE);
    return;
  }
  const int pos = p.page * kPage + tok;
  const bool valid = pos >= p.t_lo && pos < p.t_hi;
  uint32_t x2[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x2[e] = 0u;
  if (valid) {
    const int64_t row = p.row + (pos - p.t_lo);
    const uint16_t* src = is_v ? a.v + row * a.v_t + h * a.v_h : a.k + row * a.k_t + h * a.k_h;
    const uint4* s4 = reinterpret_cast<const uint4*>(src + 16 * c);
    const uint4 lo = __ldg(s4), hi = __ldg(s4 + 1);
    x2[0] = lo.x, x2[1] = lo.y, x2[2] = lo.z, x2[3] = lo.w;
    x2[4] = hi.x, x2[5] = hi.y, x2[6] = hi.z, x2[7] = hi.w;
  }
  // the row's largest magnitude: its CH chunks are lanes 4 c + i
  float m = amax16<BF16>(x2);
#pragma unroll
  for (int o = 4; o < 4 * CH; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  float d = __fdiv_rn(m, 127.f);
  const bool finite = m <= FLT_MAX;  // false for NaN too
  const bool some = finite && d >= FLT_MIN;
  const float inv = some ? __fdiv_rn(1.f, d) : 0.f;
  if (!some) d = finite ? 0.f : __uint_as_float(0x7fffffffu);
  float x[16];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 f = unpack2<BF16>(some ? x2[e] : 0u);
    x[2 * e] = f.x;
    x[2 * e + 1] = f.y;
  }
  uint32_t w[4];
  quantise16(x, d, inv, w);
  uint8_t* blk = a.pool + (static_cast<int64_t>(pid) * a.n_kv_heads + h) * F::BYTES;
  if (valid && c == 0)
    reinterpret_cast<float*>(blk + F::SCALE_OFF)[2 * tok + (is_v ? 1 : 0)] = d;
  if (!is_v) {
    if (valid)
      *reinterpret_cast<uint4*>(blk + int8_k_unit(tok, c)) = make_uint4(w[0], w[1], w[2], w[3]);
    return;
  }
  // words (channels 4 a ..) of four tokens -> this thread's unit: channels 16 c
  // + 4 i .., tokens 4 t4 ..
  quad_transpose(w, i);
  byte_transpose(w);
  uint8_t* dst = blk + F::V_OFF + int8_v_unit(c / 2, 4 * (c & 1) + i, t4);
  const int q0 = p.page * kPage + 4 * t4;
  if (q0 >= p.t_lo && q0 + 4 <= p.t_hi) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (q0 + b < p.t_lo || q0 + b >= p.t_hi) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[4 * j + b] = static_cast<uint8_t>(w[j] >> (8 * b));
    }
  }
}

// OUT: TKV_F32, TKV_F16 or TKV_BF16
template <int OUT>
__device__ __forceinline__ void store16(void* out, int64_t at, const uint32_t (&w)[4], float s) {
  float x[16];
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    // 0x4B0000uu is 2^23 + u; the product is the code times the scale, rounded
    // to f32 and then to the output's type
#pragma unroll
    for (int b = 0; b < 4; ++b)
      x[4 * a + b] = __fmul_rn(
          __fsub_rn(__uint_as_float(__byte_perm(w[a], 0x4B000000u, 0x7440u + b)),
                    8388608.f + kInt8Bias),
          s);
  }
  if constexpr (OUT == TKV_F32) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      dst[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
  } else {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      dst[e] = make_uint4(pack2<OUT == TKV_BF16>(x[8 * e], x[8 * e + 1]),
                          pack2<OUT == TKV_BF16>(x[8 * e + 2], x[8 * e + 3]),
                          pack2<OUT == TKV_BF16>(x[8 * e + 4], x[8 * e + 5]),
                          pack2<OUT == TKV_BF16>(x[8 * e + 6], x[8 * e + 7]));
  }
}

template <int D, int OUT>
__global__ void __launch_bounds__(2 * D) int8_read_kernel(Int8ReadArgs a) {
  using F = Int8Fmt<D>;
  constexpr int CH = D / 16, HALF = kPage * CH;
  const long long u = blockIdx.x / a.n_kv_heads;
  const int h = blockIdx.x % a.n_kv_heads;
  if (blockIdx.x == 0)
    flag_lengths(a.cu, a.starts, a.num_seqs, a.total, a.max_tokens, a.max_blocks, a.err);
  PageUnit p;
  if (!page_unit(a.cu, a.starts, a.num_seqs, a.total, a.max_tokens, a.max_blocks, u, p)) return;
  const int tid = threadIdx.x;
  const bool is_v = tid >= HALF;
  void* const out = is_v ? a.v_out : a.k_out;
  if (out == nullptr) return;  // whole warps: HALF is a multiple of 32
  const int r = is_v ? tid - HALF : tid;
  const int i = r & 3, c = (r >> 2) % CH, t4 = r / (4 * CH), tok = 4 * t4 + i;
  const int pid = __ldg(a.block_tables + static_cast<int64_t>(p.s) * a.max_blocks + p.page);
  const bool ok = pid >= 0 && pid < a.num_pages;
  if (!ok && r == 0) set_err(a.err, TKV_ERR_BAD_PAGE);
  const uint8_t* blk =
      a.pool + (static_cast<int64_t>(ok ? pid : 0) * a.n_kv_heads + h) * F::BYTES;
  const uint4 q = __ldg(reinterpret_cast<const uint4*>(
      is_v ? blk + F::V_OFF + int8_v_unit(c / 2, 4 * (c & 1) + i, t4) : blk + int8_k_unit(tok, c)));
  float s = __ldg(reinterpret_cast<const float*>(blk + F::SCALE_OFF) + 2 * tok + (is_v ? 1 : 0));
  uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if (is_v) {
    byte_transpose(w);
    quad_transpose(w, i);
  }
  if (!ok) {
    s = 0.f;
    w[0] = w[1] = w[2] = w[3] = 0x80808080u;
  }
  const int pos = p.page * kPage + tok;
  if (pos < p.t_lo || pos >= p.t_hi) return;
  const int64_t row = p.row + (pos - p.t_lo);
  store16<OUT>(out, (row * a.n_kv_heads + h) * D + 16 * c, w, s);
}

// CTAs of a call over `total` tokens of `num_seqs` sequences; 0: too many
unsigned int grid_of(int total, int num_seqs, int heads) {
  const long long n = (static_cast<long long>(total) / kPage + 2ll * num_seqs) * heads;
  return n > INT_MAX ? 0u : static_cast<unsigned int>(n);
}

}  // namespace

int launch_int8_append(const Int8AppendArgs& a, int head_dim, bool bf16, cudaStream_t stream) {
  const unsigned int grid = grid_of(a.total, a.num_seqs, a.n_kv_heads);
  if (grid == 0) return TKV_INVALID_ARGUMENT;
  if (head_dim == 128) {
    if (bf16)
      int8_append_kernel<128, true><<<grid, 256, 0, stream>>>(a);
    else
      int8_append_kernel<128, false><<<grid, 256, 0, stream>>>(a);
  } else {
    if (bf16)
      int8_append_kernel<64, true><<<grid, 128, 0, stream>>>(a);
    else
      int8_append_kernel<64, false><<<grid, 128, 0, stream>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? TKV_OK : TKV_BACKEND_ERROR;
}

int launch_int8_read(const Int8ReadArgs& a, int head_dim, int out_dtype, cudaStream_t stream) {
  const unsigned int grid = grid_of(a.total, a.num_seqs, a.n_kv_heads);
  if (grid == 0) return TKV_INVALID_ARGUMENT;
#define TKV_READ(D, OUT) int8_read_kernel<D, OUT><<<grid, 2 * D, 0, stream>>>(a)
  if (head_dim == 128) {
    if (out_dtype == TKV_F32) TKV_READ(128, TKV_F32);
    else if (out_dtype == TKV_F16) TKV_READ(128, TKV_F16);
    else TKV_READ(128, TKV_BF16);
  } else {
    if (out_dtype == TKV_F32) TKV_READ(64, TKV_F32);
    else if (out_dtype == TKV_F16) TKV_READ(64, TKV_F16);
    else TKV_READ(64, TKV_BF16);
  }
#undef TKV_READ
  return cudaGetLastError() == cudaSuccess ? TKV_OK : TKV_BACKEND_ERROR;
}

}  // namespace tkv
