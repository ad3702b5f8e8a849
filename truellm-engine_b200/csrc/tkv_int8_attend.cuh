// tkv_int8_attend.cuh -- what the decode and the chunk kernel of the int8 cache
// share: checks, the ranges of the f16 operands, and how a context is split.
#pragma once

#include "tkv_int8.cuh"

namespace tkv {

// Range of the f16 weights.  The weight of a token is p s 2^(5 - e): p = 2^(score - m),
// s its value scale.  A row's softmax reference m is moved only when p outgrows
// 2^kInt8Lazy, so weights stay at 2^15 or below where s <= 2^e, and they lose bits (fp16
// has steps of 2^-24 at the bottom) only below 2^-19 2^e.  e is the E of all rows that a
// warp (decode) or CTA (chunk) works on together, the power of two at the largest scale
// that any of them sees, so that s 2^(5 - E) is formed once a token.  But a row may not
// see that token, or hardly weigh it.  Rows whose largest p s is below 2^(E -
// kInt8Quiet) take an e of their own, from that product: their p is multiplied by 2^c, c =
// E - e, whose inverse multiplies their sum of p.  That product is known from steps
// that computed it and is a lower bound after them, which is the safe side: e only gets
// too small, which a weight past 2^15 shows.  So every weight is within 2^-11 of itself
// or 2^-25 of the row's largest p s.  Where c is more than kInt8Far (p 2^c nears the ends of
// 32 bits), weights are 2^(score - m + log2 s + 5 - e) instead.  Measured with no such
// row, with a loud token that all rows see and hardly weigh, and with one past kInt8Far:
// 8 chunks of 512 tokens behind 4096 339, 349 and 981 us; 8 rows behind 8192 95, 96 and
// 96 us; 16 rows behind 60000 75, 81 and 81 us.
constexpr float kInt8Lazy = 10.f;
constexpr float kInt8LazyWeight = 1024.f;  // 2^kInt8Lazy
constexpr float kInt8WeightUp = 32.f;     // 2^kInt8WeightExp
constexpr float kInt8WeightExp = 5.f;
// The chunk kernel multiplies products of a query and codes (2^15 at most) by the key
// scale (2^121) before the row's factor; 2^-9 of the one and 2^9 of the other keep that in
// 32 bits.  (Key scales below 2^-117 lose up to 9 of their 24 bits.)
constexpr float kInt8KeyDown = 0x1p-9f, kInt8KeyUp = 0x1p9f;
constexpr float kInt8Quiet = 4.f, kInt8Far = 60.f;
constexpr int kInt8DecodeRows = 16;     // most rows of the decode kernel

// Decode kernel: the steps (8 pages of a (sequence, kv head)) of all its sequences
// in one row, cut into ranges of equal length, one CTA each.  A pair whose steps
// lie in several CTAs' ranges is joined by the last of them to finish: partial
// 2 i + 1 is CTA i's last pair, begun there, 2 i its first, begun earlier.
constexpr int kInt8StepPages = 8;
struct Int8Splits {
  int ctas, least;      // CTAs at most; steps of a CTA at least
  int rows;             // the largest row count the launch may meet
  unsigned int* count;  // [ctas], zero between launches: of the pair begun there
  float* part_ml;       // [2 ctas][row block][2]  (m in log2 units, sqrt(l))
  float* part_o;        // [2 ctas][row block][D]  normalised
};

// Chunk kernel: an item is a 256-row tile of a (sequence, kv head).  CTA i < whole
// takes item i; the items from `whole` on are cut into n runs of equal length of
// their contexts, one CTA each, and joined by a second launch.
constexpr int kInt8ChunkRows = 256;
constexpr int kInt8ChunkSMs = 148;  // CTAs at a time: one per SM
struct Int8ChunkSplits {
  int whole, n, row_tiles;
  float* part_ml;  // [item - whole][run][256][2]  (m, sqrt(l))
  float* part_o;   // [item - whole][run][256][D]  normalised
};
struct Int8ChunkItem {
  int item, split, runs;
  __device__ __forceinline__ Int8ChunkItem(const Int8ChunkSplits& sp, int cta) {
    const bool one = cta < sp.whole;
    const int e = cta - sp.whole, q = one ? 0 : e / sp.n;
    item = one ? cta : sp.whole + q;
    split = one ? 0 : e - q * sp.n;
    runs = one ? 1 : sp.n;
  }
  __device__ __forceinline__ int pair(const Int8ChunkSplits& sp) const { return item / sp.row_tiles; }
  // longest contexts first
  __device__ __forceinline__ int row_tile(const Int8ChunkSplits& sp) const {
    return sp.row_tiles - 1 - item % sp.row_tiles;
  }
};

// the lengths of one sequence (see tkv_int8_attend)
__device__ __forceinline__ bool int8_attend_ok(const Int8AttendArgs& a, int len, int q0, int n) {
  return len >= 0 && len <= a.max_len &&
         static_cast<long long>(len) <= static_cast<long long>(a.max_blocks) * kPage && n >= 0 &&
         n <= len && n <= a.max_q && q0 >= 0 && q0 <= a.total_q - n;
}

// A bounded wait without the suspend hint of mbar_wait (whose sleep outlasts the
// few hundred cycles between these kernels' hand-overs): gives up after about
// two seconds of the global timer.
__device__ __forceinline__ bool mbar_wait_near(uint64_t* bar, uint32_t parity, int* err) {
  const uint32_t addr = smem_u32(bar);
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 255u) == 0) {
      const uint64_t now = global_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > 2000000000ull) break;
    }
  }
  set_err(err, TKV_ERR_TIMEOUT);
  return false;
}

// Powers of two that bring a row whose largest magnitude is m into fp16's
// range: down = 2^-e, up = 2^e with m 2^-e in [1, 2), or below 1 where m is below the
// normal range (bf16 has 2^-133 at least, so 2^-7), or up to 2^15 where m is above 2^113
// (which keeps up * kInt8KeyUp finite); 1 for infinities.
__device__ __forceinline__ void int8_row_power(float m, float& up, float& down) {
  const uint32_t e = __float_as_uint(m) >> 23;
  up = down = 1.f;
  if (e < 255) {
    const uint32_t ec = max(1u, min(e, 240u));
    up = __uint_as_float(ec << 23);
    down = __uint_as_float((254u - ec) << 23);
  }
}

// 2^-E with s 2^-E in [1/2, 1), s > 0 a finite scale (at most 2^121); E is raised
// when a scale exceeds 2^E
__device__ __forceinline__ float int8_scale_inverse(float s) {
  const int e = static_cast<int>(__float_as_uint(s) >> 23);  // 2^(e - 127) <= s
  return __uint_as_float(static_cast<uint32_t>(min(253, max(1, 253 - e))) << 23);
}

// E of 2^-E
__device__ __forceinline__ float int8_scale_exponent(float inverse) {
  return static_cast<float>(127 - static_cast<int>(__float_as_uint(inverse) >> 23));
}
// 2^e, e a whole number from -126 to 126
__device__ __forceinline__ float int8_pow2(float e) {
  return __uint_as_float(static_cast<uint32_t>(127 + static_cast<int>(e)) << 23);
}
// log2 of a value scale: -inf for none
__device__ __forceinline__ float int8_log2(float s) {
  float y;
  asm("lg2.approx.f32 %0, %1;\n" : "=f"(y) : "f"(s));
  return y;
}
// The e of a row with reference m whose largest score + log2 s is top (a row that has
// seen nothing has no weights: E).  NaN, from scores that are no numbers, gives -126.
__device__ __forceinline__ float int8_row_exponent(float top, float m, float E) {
  if (m == -INFINITY) return E;
  const float e = fminf(fmaxf(ceilf(top - m), -126.f), 126.f);
  return E - e > kInt8Quiet ? e : E;
}

__device__ __forceinline__ float int8_sqrt(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// A part of a row in a join: its outputs count times u^2, u = sqrt(l) 2^((m - M) / 2), M the
// largest m.  Outputs are multiplied by u twice: a part whose m lies 2^-126 and more below
// may hold values that are louder by as much.  Parts are stored with sqrt(l); its last bit
// does not matter, as the sum of the weights has the same.
__device__ __forceinline__ float int8_part_root(float root_l, float m, float M) {
  return root_l * fast_exp2(0.5f * (m - (M == -INFINITY ? 0.f : M)));
}

// four consecutive channels of an output row, rounded once
__device__ __forceinline__ void int8_store4(const Int8AttendArgs& a, int64_t at, float4 v) {
  uint2 w;
  if (a.out_bf16)
    w = make_uint2(pack2<true>(v.x, v.y), pack2<true>(v.z, v.w));
  else
    w = make_uint2(pack2<false>(v.x, v.y), pack2<false>(v.z, v.w));
  *reinterpret_cast<uint2*>(a.out + at) = w;
}

int launch_int8_decode(const Int8AttendArgs& a, const Int8Splits& sp, int head_dim,
                       cudaStream_t stream);

int launch_int8_chunk(const Int8AttendArgs& a, const Int8ChunkSplits& sp, int head_dim,
                      cudaStream_t stream);

}  // namespace tkv
