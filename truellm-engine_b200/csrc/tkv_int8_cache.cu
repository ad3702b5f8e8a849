// tkv_int8_cache.cu -- writing the paged int8 cache (quantise on append, the
// reshape_and_cache slot of third_party/vllm_kernels/cache_kernels.cu:202-232)
// and reading it back as dense K/V.
//
// One CTA per 16-token page of a sequence's range and run of kv heads: half of
// its threads take the keys, half the values, one thread per (token, 16
// channels), one head after another with the next one's loads in flight.  Lanes 4
// c + i of a warp hold token 4 t + i, chunk c, so the four tokens of a
// V word sit in one quad: a 4 x 4 transpose of words over the quad and of bytes
// within a thread turns four rows into 16-byte units of the V layout (and back).
//
// CTAs are numbered along one axis of page units: sequence s owns the units
// from cu[s] / 16 + 2 s on (a range of n tokens touches at most n / 16 + 2
// pages), so a ragged batch launches (tokens / 16 + 2 sequences) x heads CTAs
// whatever its longest sequence; a CTA finds its sequence by a 32-way search.
// Where that is more than the tokens there are (a decode step), sequence s owns
// the units from cu[s] on: a page that is touched holds a token of the range.
// 256 sequences of one token, 8 heads: append 14.5 us against 19.9.
//
// Both kernels are bound by memory: 2 bytes a channel on the dense side, 1 and a
// scale on the paged one.  64 x 2048 tokens of 8 heads of 128 channels: append
// 167 us (4.9 TB/s), read 139 us (5.9 TB/s).
#include <limits.h>

#include <algorithm>

#include "tkv_int8.cuh"
#include "tkv_umma.cuh"  // packed f32x2 arithmetic

namespace tkv {
namespace {

// first page unit of sequence s
__device__ __forceinline__ long long first_unit(int32_t cu_s, int s, bool per_token) {
  return per_token ? cu_s : static_cast<long long>(cu_s / kPage) + 2ll * s;
}

// the last sequence whose first page unit is <= u (all lanes of a warp take part)
__device__ __forceinline__ int find_seq(const int32_t* cu, int num_seqs, long long u,
                                        bool per_token) {
  int lo = 0, hi = num_seqs;  // the answer is in [lo, hi)
  const int lane = threadIdx.x & 31;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int s = lo + lane * step;
    const bool le = s < hi && first_unit(__ldg(cu + s), s, per_token) <= u;
    const unsigned int m = __ballot_sync(0xffffffffu, le);
    // offsets are non-decreasing in a valid call; any answer is in range otherwise
    const int last = m ? 31 - __clz(m) : 0;
    lo += last * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

constexpr int kAhead = 3;  // heads of the append kernel's rows in shared memory

// How a launch is cut up.  heads: kv heads a CTA takes one after another;
// per_token: the numbering of page units.
struct Plan {
  int heads;
  bool per_token;
};

// what a CTA works on: page `page` (index in the sequence) of sequence s, and
// the tokens [t_lo, t_hi) of it, which are rows row + (token - t_lo)
struct PageUnit {
  int s, page, t_lo, t_hi, row;
};

// false: nothing to do.  `lens` holds the first token of each sequence's range.
__device__ __forceinline__ bool page_unit(const int32_t* cu, const int32_t* lens, int num_seqs,
                                          int total, int max_n, int max_blocks, long long u,
                                          bool per_token, PageUnit& p) {
  p.s = find_seq(cu, num_seqs, u, per_token);
  const int r0 = __ldg(cu + p.s), n = __ldg(cu + p.s + 1) - r0, pos = __ldg(lens + p.s);
  if (!int8_seq_ok(pos, n, r0, total, max_n, max_blocks)) return false;
  const long long j = u - first_unit(r0, p.s, per_token);
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
// and the low byte of its bits is the stored byte.  inv_lo <= 1/d <= inv_hi, so
// where the sums with both agree (each a multiply-add, rounded once), the sum with
// x/d itself, which lies between them, rounds to the same.  The others (x/d within
// 2^-15 of a half; with bf16 values, half of a row's largest is such) are
// corrected in exact arithmetic: x - k d is exact in f32 (x has 11 bits or fewer
// and |x - k d| < 2 d, a multiple of d's last bit).  The correction is right for
// every value, so a warp makes it for the pairs where any of its lanes needs it.
template <bool BF16>
__device__ __forceinline__ void quantise16(const uint32_t (&x2)[8], float d, float inv_lo,
                                           float inv_hi, uint32_t (&w)[4]) {
  constexpr float kMagic = 12582912.f + kInt8Bias;
  const float2 lo2 = make_float2(inv_lo, inv_lo), hi2 = make_float2(inv_hi, inv_hi);
  const float2 up2 = make_float2(kMagic, kMagic), minus2 = make_float2(-1.f, -1.f);
  float2 t[8], differ = make_float2(0.f, 0.f);  // a bit for each pair
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 x = unpack2<BF16>(x2[e]);
    t[e] = ffma2(x, lo2, up2);
    const float2 gap = ffma2(t[e], minus2, ffma2(x, hi2, up2));  // exact: 0, 1 or -1
    const float2 bit = make_float2(1 << e, 1 << e);
    differ = ffma2(ffma2(gap, gap, make_float2(0.f, 0.f)), bit, differ);
  }
  const uint32_t near_half = __reduce_or_sync(
      0xffffffffu, static_cast<uint32_t>(differ.x) | static_cast<uint32_t>(differ.y));
  if (near_half) {
    auto fix = [&](float x, float& v) {
      const float r = __fmaf_rn(__fsub_rn(kMagic, v), d, x);
      // at a remainder of exactly d/2 an odd code gives way (d/2 itself may lack the
      // last bit, twice the remainder has it)
      const float most = __uint_as_float(__float_as_uint(d) - (__float_as_uint(v) & 1u));
      if (fabsf(r + r) > most) v += copysignf(1.f, r);
    };
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (near_half >> e & 1) {
        const float2 x = unpack2<BF16>(x2[e]);
        fix(x.x, t[e].x);
        fix(x.y, t[e].y);
      }
    }
  }
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const uint32_t lo = __byte_perm(__float_as_uint(t[2 * a].x), __float_as_uint(t[2 * a].y), 0x0040);
    const uint32_t hi =
        __byte_perm(__float_as_uint(t[2 * a + 1].x), __float_as_uint(t[2 * a + 1].y), 0x0040);
    w[a] = __byte_perm(lo, hi, 0x5410);
  }
}

// bits of max |x| of 16 packed values as f32; a NaN among them gives a NaN's,
// which as whole numbers are above infinity's
template <bool BF16>
__device__ __forceinline__ uint32_t amax16(const uint32_t (&p)[8]) {
  uint32_t m = p[0];  // signs are left to the last step
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    if constexpr (BF16)
      asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(p[i]));
    else
      asm("max.NaN.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(m) : "r"(p[i]));
  }
  const float2 f = unpack2<BF16>(m & 0x7fff7fffu);
  return max(__float_as_uint(f.x), __float_as_uint(f.y));
}

template <int D, bool BF16>
__global__ void __launch_bounds__(2 * D, 1024 / (2 * D))
    int8_append_kernel(Int8AppendArgs a, Plan plan) {
  using F = Int8Fmt<D>;
  constexpr int CH = D / 16, HALF = kPage * CH;  // threads per tensor
  const int parts = (a.n_kv_heads + plan.heads - 1) / plan.heads;
  const int u = blockIdx.x / parts, h0 = (blockIdx.x - u * parts) * plan.heads;
  const int h1 = min(h0 + plan.heads, a.n_kv_heads);
  if (blockIdx.x == 0)
    flag_lengths(a.cu, a.lens_old, a.num_seqs, a.total, a.max_new, a.max_blocks, a.err);
  PageUnit p;
  if (!page_unit(a.cu, a.lens_old, a.num_seqs, a.total, a.max_new, a.max_blocks, u, plan.per_token, p)) return;
  const int tid = threadIdx.x;
  const bool is_v = tid >= HALF;
  const int r = is_v ? tid - HALF : tid;
  const int i = r & 3, c = (r >> 2) % CH, t4 = r / (4 * CH), tok = 4 * t4 + i;
  const int pos = p.page * kPage + tok;
  const bool valid = pos >= p.t_lo && pos < p.t_hi;
  if (!__any_sync(0xffffffffu, valid)) return;  // a warp whose tokens are others'
  // A warp brings the rows of its 128 / CH tokens to shared memory itself, kAhead
  // heads ahead: 64 pieces of 16 bytes a head, lane l copies pieces l and l + 32.
  // Piece q of token 4 t + i lies at q ^ (i & 1 | (i & 2) << 1), so the eight
  // lanes that read at once are in different banks.
  __shared__ __align__(16) uint4 stage[kAhead][2 * D / 32][64];
  const int warp = tid / 32, lane = tid & 31;
  const uint16_t* src[2];
  uint32_t to[2], bytes[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int piece = lane + 32 * e, t = piece / (2 * CH), q = piece % (2 * CH);
    const int at = p.page * kPage + (r & ~31) / CH + t;
    const bool in = at >= p.t_lo && at < p.t_hi;
    const int64_t row = in ? p.row + (at - p.t_lo) : p.row;
    src[e] = (is_v ? a.v + row * a.v_t + h0 * a.v_h : a.k + row * a.k_t + h0 * a.k_h) + 8 * q;
    to[e] = smem_u32(&stage[0][warp][2 * CH * t + (q ^ ((t & 1) | (t & 2) << 1))]);
    bytes[e] = in ? 16u : 0u;  // the rest is filled with zeros
  }
  const int64_t step = is_v ? a.v_h : a.k_h;
  auto fetch = [&](int h) {  // h heads from the first one
    if (h0 + h < h1) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        cp_async16_or_zero(to[e] + (h % kAhead) * static_cast<uint32_t>(sizeof(stage[0])),
                           src[e] + h * step, bytes[e]);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int h = 0; h < kAhead - 1; ++h) fetch(h);
  const int pid = __ldg(a.block_tables + static_cast<int64_t>(p.s) * a.max_blocks + p.page);
  if (pid < 0 || pid >= a.num_pages) {
    if (valid) set_err(a.err, TKV_ERR_BAD_PAGE);
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }
  uint8_t* blk = a.pool + (static_cast<int64_t>(pid) * a.n_kv_heads + h0) * F::BYTES;
  const int mine = 2 * CH * ((r & 31) / (4 * CH) * 4 + i), turn = (i & 1) | (i & 2) << 1;
  for (int h = 0; h < h1 - h0; ++h, blk += F::BYTES) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 2) : "memory");
    __syncwarp();  // every lane's pieces are there, and the stage before is read
    fetch(h + kAhead - 1);
    const uint4* from = stage[h % kAhead][warp] + mine;
    const uint4 lo = from[(2 * c) ^ turn], hi = from[(2 * c + 1) ^ turn];
    uint32_t x2[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    // the row's largest magnitude: its CH chunks are lanes 4 c + i
    uint32_t bits = amax16<BF16>(x2);
#pragma unroll
    for (int o = 4; o < 4 * CH; o <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    const float m = __uint_as_float(bits);
    float d = __fdiv_rn(m, 127.f);
    const bool finite = m <= FLT_MAX;  // false for NaN too
    const bool some = finite && d >= FLT_MIN;
    // the approximation of 1/d (normal, as d is) is off by one unit in the last
    // place at most, so two either way enclose it
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(some ? d : 1.f));
    const float inv_lo = __uint_as_float(__float_as_uint(inv) - 2u);
    const float inv_hi = __uint_as_float(__float_as_uint(inv) + 2u);
    if (!some) {
      d = finite ? 0.f : __uint_as_float(0x7fffffffu);
#pragma unroll
      for (int e = 0; e < 8; ++e) x2[e] = 0u;
    }
    uint32_t w[4];
    quantise16<BF16>(x2, d, inv_lo, inv_hi, w);
    if (valid && c == 0)
      reinterpret_cast<float*>(blk + F::SCALE_OFF)[2 * tok + (is_v ? 1 : 0)] = d;
    if (!is_v) {
      if (valid)
        *reinterpret_cast<uint4*>(blk + int8_k_unit(tok, c)) = make_uint4(w[0], w[1], w[2], w[3]);
      continue;
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
}

// OUT: TKV_F32, TKV_F16 or TKV_BF16
template <int OUT>
__device__ __forceinline__ void store16(void* out, int64_t at, const uint32_t (&w)[4], float s,
                                        bool wide) {
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
    uint32_t y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = pack2<OUT == TKV_BF16>(x[2 * e], x[2 * e + 1]);
    if (wide) {  // whole 32-byte sectors
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(y[0]),
                   "r"(y[1]), "r"(y[2]), "r"(y[3]), "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7])
                   : "memory");
    } else {
      dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
      dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
    }
  }
}

template <int D, int OUT>
__global__ void __launch_bounds__(2 * D) int8_read_kernel(Int8ReadArgs a, Plan plan, bool wide) {
  using F = Int8Fmt<D>;
  constexpr int CH = D / 16, HALF = kPage * CH;
  const int parts = (a.n_kv_heads + plan.heads - 1) / plan.heads;
  const int u = blockIdx.x / parts, h0 = (blockIdx.x - u * parts) * plan.heads;
  const int h1 = min(h0 + plan.heads, a.n_kv_heads);
  if (blockIdx.x == 0)
    flag_lengths(a.cu, a.starts, a.num_seqs, a.total, a.max_tokens, a.max_blocks, a.err);
  PageUnit p;
  if (!page_unit(a.cu, a.starts, a.num_seqs, a.total, a.max_tokens, a.max_blocks, u, plan.per_token, p)) return;
  const int tid = threadIdx.x;
  const bool is_v = tid >= HALF;
  void* const out = is_v ? a.v_out : a.k_out;
  if (out == nullptr) return;  // whole warps: HALF is a multiple of 32
  const int r = is_v ? tid - HALF : tid;
  const int i = r & 3, c = (r >> 2) % CH, t4 = r / (4 * CH), tok = 4 * t4 + i;
  const int pos = p.page * kPage + tok;
  const bool valid = pos >= p.t_lo && pos < p.t_hi;
  if (!__any_sync(0xffffffffu, valid)) return;  // a warp whose tokens are others'
  const int pid = __ldg(a.block_tables + static_cast<int64_t>(p.s) * a.max_blocks + p.page);
  const bool ok = pid >= 0 && pid < a.num_pages;
  if (!ok && valid) set_err(a.err, TKV_ERR_BAD_PAGE);
  const uint8_t* const blk =
      a.pool + (static_cast<int64_t>(ok ? pid : 0) * a.n_kv_heads + h0) * F::BYTES;
  const uint8_t* src =
      blk + (is_v ? F::V_OFF + int8_v_unit(c / 2, 4 * (c & 1) + i, t4) : int8_k_unit(tok, c));
  const uint8_t* scale = blk + F::SCALE_OFF + 8 * tok + (is_v ? 4 : 0);
  int64_t at = (static_cast<int64_t>(p.row + (pos - p.t_lo)) * a.n_kv_heads + h0) * D + 16 * c;
  uint4 q = __ldcs(reinterpret_cast<const uint4*>(src));
  float s = __ldcs(reinterpret_cast<const float*>(scale));
  for (int h = h0; h < h1; ++h, at += D) {
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
    float sh = s;
    if (h + 1 < h1) {
      src += F::BYTES;
      scale += F::BYTES;
      q = __ldcs(reinterpret_cast<const uint4*>(src));
      s = __ldcs(reinterpret_cast<const float*>(scale));
    }
    if (is_v) {
      byte_transpose(w);
      quad_transpose(w, i);
    }
    if (!ok) {
      sh = 0.f;
      w[0] = w[1] = w[2] = w[3] = 0x80808080u;
    }
    if (valid) store16<OUT>(out, at, w, sh, wide);
  }
}

// CTAs of a call over `total` tokens; 0: more than a grid has.  A CTA takes one
// head while that leaves no more than one round of the append kernel's 4 x 148
// CTAs; beyond, up to 8, which spares the later heads their search for the
// sequence and keeps loads in flight.  64 x 2048 tokens of 8 heads with 1, 2, 4
// and 8 heads a CTA: append 432, 315, 257 and 228 us, read 224, 156, 138 and 140
// us (the loads then went through registers); 8 x 512 tokens with one head and
// with 4: append 13.7 and 10.7 us, read 9.2 and 7.5 us.
unsigned int plan_grid(int total, int num_seqs, int n_heads, Plan& plan) {
  const long long pages = static_cast<long long>(total) / kPage + 2ll * num_seqs;
  plan.per_token = total < pages;
  const long long units = plan.per_token ? total : pages;
  plan.heads = static_cast<int>(
      std::max<long long>(1, std::min<long long>({8ll, n_heads, units * n_heads / 592})));
  const long long n = units * ((n_heads + plan.heads - 1) / plan.heads);
  return n > INT_MAX ? 0u : static_cast<unsigned int>(n);
}

}  // namespace

int launch_int8_append(const Int8AppendArgs& a, int head_dim, bool bf16, cudaStream_t stream) {
  Plan plan;
  const unsigned int grid = plan_grid(a.total, a.num_seqs, a.n_kv_heads, plan);
  if (grid == 0) return TKV_INVALID_ARGUMENT;
  if (head_dim == 128) {
    if (bf16)
      int8_append_kernel<128, true><<<grid, 256, 0, stream>>>(a, plan);
    else
      int8_append_kernel<128, false><<<grid, 256, 0, stream>>>(a, plan);
  } else {
    if (bf16)
      int8_append_kernel<64, true><<<grid, 128, 0, stream>>>(a, plan);
    else
      int8_append_kernel<64, false><<<grid, 128, 0, stream>>>(a, plan);
  }
  return cudaGetLastError() == cudaSuccess ? TKV_OK : TKV_BACKEND_ERROR;
}

int launch_int8_read(const Int8ReadArgs& a, int head_dim, int out_dtype, cudaStream_t stream) {
  Plan plan;
  // both outputs start at multiples of 32 bytes, as their rows then do: 16 channels are
  // one store of a whole sector (ragged prefixes of 16 sequences: 98 -> 88 us)
  const bool wide =
      ((reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out)) & 31) == 0;
  const unsigned int grid = plan_grid(a.total, a.num_seqs, a.n_kv_heads, plan);
  if (grid == 0) return TKV_INVALID_ARGUMENT;
#define TKV_READ(D, OUT) int8_read_kernel<D, OUT><<<grid, 2 * D, 0, stream>>>(a, plan, wide)
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
