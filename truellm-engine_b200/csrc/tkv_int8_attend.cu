// tkv_int8_attend.cu -- attention of each sequence's last tokens over the paged
// int8 cache.
//
// One warp per (query token, q head): lane l takes the scores of token l % 16
// of a page over half of the channels each, the online softmax runs in the
// exp2 domain once per page, and every lane then owns D / 32 channels of the
// output.
#include <limits.h>

#include <algorithm>

#include "tkv_int8_attend.cuh"

namespace tkv {
namespace {

constexpr int kWarps = 4;

// byte b of word w as the code it stands for
__device__ __forceinline__ float code(uint32_t w, int b) {
  return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440u + b)) - (8388608.f + kInt8Bias);
}

template <int D, bool QBF16, bool OBF16>
__global__ void __launch_bounds__(32 * kWarps) int8_attend_kernel(Int8AttendArgs a) {
  using F = Int8Fmt<D>;
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int s = blockIdx.y;
  const int len = __ldg(a.seq_lens + s), q0 = __ldg(a.cu_q + s), n = __ldg(a.cu_q + s + 1) - q0;
  if (!int8_attend_ok(a, len, q0, n)) return;  // flagged by the decode kernel
  if (static_cast<long long>(n) * a.grp <= kInt8DecodeRows) return;  // the decode kernel's
  const long long r = static_cast<long long>(blockIdx.x) * kWarps + warp;
  if (r >= static_cast<long long>(n) * a.num_q_heads) return;
  const int i = static_cast<int>(r / a.num_q_heads), hq = static_cast<int>(r % a.num_q_heads);
  const int h = hq / a.grp;
  const int pos = len - n + i;
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int tok = lane & 15, hf = lane >> 4;
  float q[D / 2];
  {
    const uint16_t* src = a.q + (q0 + i) * a.q_t + hq * a.q_h + hf * (D / 2);
#pragma unroll
    for (int c = 0; c < D / 2; c += 2) {
      const float2 f = unpack2<QBF16>(*reinterpret_cast<const uint32_t*>(src + c));
      q[c] = f.x;
      q[c + 1] = f.y;
    }
  }
  float m = -INFINITY, l = 0.f, o[D / 32];
#pragma unroll
  for (int j = 0; j < D / 32; ++j) o[j] = 0.f;
  for (int pg = lo / kPage; pg <= pos / kPage; ++pg) {
    int pid = __ldg(a.block_tables + static_cast<int64_t>(s) * a.max_blocks + pg);
    if (pid < 0 || pid >= a.num_pages) {
      if (lane == 0) set_err(a.err, TKV_ERR_BAD_PAGE);
      pid = 0;
    }
    const uint8_t* blk = a.pool + (static_cast<int64_t>(pid) * a.n_kv_heads + h) * F::BYTES;
    const float2 sc = __ldg(reinterpret_cast<const float2*>(blk + F::SCALE_OFF) + tok);
    float x = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(blk + int8_k_unit(tok, hf * (D / 32) + c)));
      const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 16; ++e) x = fmaf(q[16 * c + e], code(ww[e >> 2], e & 3), x);
    }
    x += __shfl_xor_sync(0xffffffffu, x, 16);
    const int t = pg * kPage + tok;
    const bool seen = t >= lo && t <= pos;
    x = seen ? x * sc.x * a.alpha : -INFINITY;
    float mx = x;
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
    mx = fmaxf(mx, m);
    const float ref = mx == -INFINITY ? 0.f : mx;
    const float f = exp2f(m - ref), p = exp2f(x - ref);
    m = mx;
    l = l * f + (hf == 0 ? p : 0.f);
    const float pv = seen ? p * sc.y : 0.f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) o[j] *= f;
    // lane owns channels D/32 lane ..: 4 (one group g) for D = 128, 2 for D = 64
    constexpr int W = D / 32;
    const int c0 = W * lane, uu = c0 / 32, g = c0 % 32 / 4, j0 = c0 % 4;
#pragma unroll
    for (int t4 = 0; t4 < 4; ++t4) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(blk + F::V_OFF + int8_v_unit(uu, g, t4));
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const float pt = __shfl_sync(0xffffffffu, pv, 4 * t4 + b);
#pragma unroll
        for (int j = 0; j < W; ++j) o[j] = fmaf(pt, code(__ldg(w + j0 + j), b), o[j]);
      }
    }
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* dst = a.out + (static_cast<int64_t>(q0 + i) * a.num_q_heads + hq) * D + (D / 32) * lane;
#pragma unroll
  for (int j = 0; j < D / 32; j += 2)
    *reinterpret_cast<uint32_t*>(dst + j) = pack2<OBF16>(o[j] * inv, o[j + 1] * inv);
}

}  // namespace

namespace {

constexpr int kSlots = 148 * 3;  // resident CTAs of the decode kernel
constexpr int kMinRun = 8;       // pages: one step of each of a CTA's warps
constexpr int kMaxRun = 64;
constexpr int kMaxRuns = 512;

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

// How decode contexts of up to these sizes are cut: runs of equal length that
// give every resident CTA one, but not shorter than a step of each warp nor
// longer than kMaxRun pages.
void decode_splits(Int8Splits& sp, int num_seqs, int num_kv_heads, int grp, int max_q, int max_len) {
  const long long pages = (static_cast<long long>(max_len) + kPage - 1) / kPage;
  const long long total = pages * num_seqs * num_kv_heads;
  long long run = (total + kSlots - 1) / kSlots;
  run = std::min<long long>(kMaxRun, std::max<long long>(kMinRun, (run + kMinRun - 1) / kMinRun * kMinRun));
  run = std::max(run, (pages + kMaxRuns - 1) / kMaxRuns);
  sp.pages = static_cast<int>(run);
  sp.n = static_cast<int>(std::max<long long>(1, (pages + run - 1) / run));
  sp.rows = static_cast<int>(std::min<long long>(kInt8DecodeRows, static_cast<long long>(max_q) * grp));
}

// bytes of the decode kernel's share of the workspace
size_t decode_bytes(const Int8Splits& sp, int num_seqs, int num_kv_heads, int head_dim) {
  const size_t pairs = static_cast<size_t>(num_seqs) * num_kv_heads;
  const size_t rb = sp.rows <= 8 ? 8 : 16;
  return round256(pairs * 4) + (sp.n > 1 ? round256(pairs * sp.n * rb * 8) + pairs * sp.n * rb * head_dim * 4 : 0);
}

}  // namespace

size_t int8_attend_workspace(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                             int max_q, int max_len) {
  Int8Splits sp;
  decode_splits(sp, num_seqs, num_kv_heads, num_q_heads / num_kv_heads, max_q, max_len);
  return 256 + decode_bytes(sp, num_seqs, num_kv_heads, head_dim);
}

int launch_int8_attend(const Int8AttendArgs& a, int head_dim, void* workspace, size_t,
                       cudaStream_t stream) {
  Int8Splits sp;
  decode_splits(sp, a.num_seqs, a.n_kv_heads, a.grp, a.max_q, a.max_len);
  const size_t pairs = static_cast<size_t>(a.num_seqs) * a.n_kv_heads;
  uint8_t* ws = static_cast<uint8_t*>(workspace) + 256;
  sp.count = reinterpret_cast<unsigned int*>(ws);
  ws += round256(pairs * 4);
  sp.part_ml = reinterpret_cast<float*>(ws);
  sp.part_o = reinterpret_cast<float*>(ws + round256(pairs * sp.n * (sp.rows <= 8 ? 8 : 16) * 8));
  const int st = launch_int8_decode(a, sp, head_dim, stream);
  if (st != TKV_OK || static_cast<long long>(a.max_q) * a.grp <= kInt8DecodeRows) return st;
  const long long rows = static_cast<long long>(a.max_q) * a.num_q_heads;
  const dim3 grid(static_cast<unsigned int>((rows + kWarps - 1) / kWarps), a.num_seqs);
#define TKV_RUN(D, Q, O) int8_attend_kernel<D, Q, O><<<grid, 32 * kWarps, 0, stream>>>(a)
  if (head_dim == 128) {
    if (a.q_bf16) { if (a.out_bf16) TKV_RUN(128, true, true); else TKV_RUN(128, true, false); }
    else { if (a.out_bf16) TKV_RUN(128, false, true); else TKV_RUN(128, false, false); }
  } else {
    if (a.q_bf16) { if (a.out_bf16) TKV_RUN(64, true, true); else TKV_RUN(64, true, false); }
    else { if (a.out_bf16) TKV_RUN(64, false, true); else TKV_RUN(64, false, false); }
  }
#undef TKV_RUN
  return cudaGetLastError() == cudaSuccess ? TKV_OK : TKV_BACKEND_ERROR;
}

}  // namespace tkv
