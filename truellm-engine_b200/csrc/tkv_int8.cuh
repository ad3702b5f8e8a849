// tkv_int8.cuh -- the paged int8 cache: its block layout, argument blocks and
// the device helpers that its append, read-back and attention kernels share.
#pragma once

#include "tkv_common.cuh"

namespace tkv {

// One (page, kv head) block (see truellm_kivi.h): K codes, V codes, scales.
template <int D>
struct Int8Fmt {
  static_assert(D == 64 || D == 128, "head sizes of the cache");
  static constexpr int CODES = kPage * D;          // bytes of the K (or V) codes
  static constexpr int V_OFF = CODES;
  static constexpr int SCALE_OFF = 2 * CODES;      // [16 tokens][2] f32
  static constexpr int BYTES = 2 * CODES + kPage * 8;
  static_assert(BYTES % 16 == 0, "blocks move by 16-byte copies");
};
constexpr int kInt8Bias = 128;  // a stored byte is code + 128

// byte offset of the 16 channels of chunk c of token t in the K codes
__host__ __device__ constexpr int int8_k_unit(int t, int c) {
  return c * 256 + (t ^ (2 * (c & 3))) * 16;
}
// byte offset of the 4 channels x 4 tokens (channels 32 u + 4 g .., tokens 4 t ..)
// in the V codes
__host__ __device__ constexpr int int8_v_unit(int u, int g, int t) {
  return ((u * 8 + g) * 4 + t) * 16;
}

struct Int8AppendArgs {
  uint8_t* pool;
  int num_pages, n_kv_heads;
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_t, k_h, v_t, v_h;  // token and head strides, elements
  const int32_t* cu;
  const int32_t* lens_old;
  const int32_t* block_tables;
  int max_blocks, num_seqs, total, max_new;
  int* err;
};

struct Int8ReadArgs {
  const uint8_t* pool;
  int num_pages, n_kv_heads;
  void* k_out;
  void* v_out;
  const int32_t* block_tables;
  int max_blocks;
  const int32_t* starts;
  const int32_t* cu;
  int num_seqs, total, max_tokens;
  int* err;
};

struct Int8AttendArgs {
  const uint8_t* pool;
  int num_pages, n_kv_heads;
  const uint16_t* q;
  int64_t q_t, q_h;  // token and head strides, elements
  int q_bf16;
  uint16_t* out;
  int out_bf16;
  const int32_t* cu_q;
  const int32_t* block_tables;
  int max_blocks;
  const int32_t* seq_lens;
  int num_seqs, num_q_heads, grp, total_q, max_q, max_len, window;
  float alpha;  // scale * log2(e)
  int* err;
};

// The tokens [pos, pos + n) of one sequence and their rows [row, row + n) in
// the dense tensors; false (and nothing to do) when any of it is out of range.
__device__ __forceinline__ bool int8_seq_ok(int pos, int n, int row, int total, int max_n,
                                            int max_blocks) {
  return pos >= 0 && n >= 0 && n <= max_n && row >= 0 && row <= total - n &&
         static_cast<long long>(pos) + n <= static_cast<long long>(max_blocks) * kPage;
}

// two packed 16-bit values to floats
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  return BF16 ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u))
              : unpack_h2(x);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_h2(a, b);
  }
}

// 16 bytes global -> shared, of which the first `bytes` are copied, the rest zeros
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst_smem, const void* src_gmem, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst_smem), "l"(src_gmem), "r"(bytes)
               : "memory");
}

// 4 x 4 transpose of 32-bit words over the 4 lanes of a quad (lane bits 0-1 =
// i): word a of lane i goes to word i of lane a.
__device__ __forceinline__ void quad_transpose(uint32_t (&w)[4], int i) {
  const bool b0 = i & 1, b1 = i & 2;
  const uint32_t s0 = __shfl_xor_sync(0xffffffffu, b0 ? w[0] : w[1], 1);
  const uint32_t s1 = __shfl_xor_sync(0xffffffffu, b0 ? w[2] : w[3], 1);
  if (b0) {
    w[0] = s0;
    w[2] = s1;
  } else {
    w[1] = s0;
    w[3] = s1;
  }
  const uint32_t r0 = __shfl_xor_sync(0xffffffffu, b1 ? w[0] : w[2], 2);
  const uint32_t r1 = __shfl_xor_sync(0xffffffffu, b1 ? w[1] : w[3], 2);
  if (b1) {
    w[0] = r0;
    w[1] = r1;
  } else {
    w[2] = r0;
    w[3] = r1;
  }
}
// 4 x 4 transpose of the bytes of four words: byte a of word i to byte i of word a
__device__ __forceinline__ void byte_transpose(uint32_t (&w)[4]) {
  const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[0], w[1], 0x7362);
  const uint32_t c = __byte_perm(w[2], w[3], 0x5140), d = __byte_perm(w[2], w[3], 0x7362);
  w[0] = __byte_perm(a, c, 0x5410);
  w[1] = __byte_perm(a, c, 0x7632);
  w[2] = __byte_perm(b, d, 0x5410);
  w[3] = __byte_perm(b, d, 0x7632);
}

// Four stored bytes to exact f16 pairs of codes (bytes 0, 1 and 2, 3): 0x64uu
// is 1024 + u, and 1152 comes off exactly.
__device__ __forceinline__ void int8_to_h2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(lo) : "r"(a), "r"(0x64806480u));
  asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(hi) : "r"(b), "r"(0x64806480u));
}

int launch_int8_append(const Int8AppendArgs& a, int head_dim, bool bf16, cudaStream_t stream);
int launch_int8_read(const Int8ReadArgs& a, int head_dim, int out_dtype, cudaStream_t stream);
size_t int8_attend_workspace(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                             int max_q, int max_len);
int launch_int8_attend(const Int8AttendArgs& a, int head_dim, void* workspace,
                       size_t workspace_bytes, cudaStream_t stream);

// Rotary positions (tkv_rope.cu)
struct RopeArgs {
  const uint16_t* q;
  const uint16_t* k;
  uint16_t* q_out;
  uint16_t* k_out;
  int64_t q_t, q_h, k_t, k_h, qo_t, qo_h, ko_t, ko_h;  // strides, elements
  int hq, hk, head_dim, n_tokens, inverse;
  const int32_t* positions;
  int64_t axis_stride;
};
int launch_rope(const tkv_rope_plan_t& plan, const RopeArgs& a, bool bf16, cudaStream_t stream);

}  // namespace tkv
