// tkv_int8_decode.cu -- attention over the paged int8 cache for few query rows
// (decode steps, draft tokens): up to 16 rows (query token x q head of the kv
// head's group) of a (sequence, kv head).
//
// The steps (8 pages of a pair, i.e. a (sequence, kv head)) of all sequences lie in
// one row that the CTAs share in equal ranges, however long each context is; every
// CTA finds its range in the lengths.  Of each pair in it its four warps take pages
// two at a time in turn, each with a private ring of
// shared-memory stages that 1-D bulk copies (cp.async.bulk, no multicast) fill
// with whole 4224-byte blocks, and no synchronisation between warps until the
// pair ends.  Per page, on mma.sync m16n8k16 (tokens are the M side, query rows
// the N side):
//   S^T = K Q^T   codes become exact f16 integers in registers, the key scale
//                 multiplies the finished 32-bit score
//   O^T += V^T P^T  the value scale multiplies the 32-bit weight before its one
//                 rounding to f16, so codes enter exactly here too
// A masked token's weight is exactly 0 whatever its scales hold (codes are
// always finite numbers), so a NaN reaches only the rows that see it.
//
// The parts of a pair that several CTAs share are joined by the one that finishes
// last (partials in the workspace, a counter that it zeroes again); the order of
// the sum is that of the CTAs, so the result does not depend on who is last.
//
// Bound by memory: 33 bytes a token, head and 16 channels of keys and values.  64
// sequences of 1024 to 8192 tokens, 8 kv heads of 128 channels, 4 q heads each: 97 us,
// 6.0 TB/s.  Equal runs of every context instead of one row of steps: 174, 123, 107,
// 103, 100 and 119 us with runs of 16, 32, 64, 128, 256 and 384 pages, and another
// best length for every call.  More than one range a resident CTA: 101 to 106 us.
// Up to 8 query rows take one column tile of the products and 16 rows two (2 x
// 60000 tokens: 58 and 78 us); the chunk kernel takes 106 us for 20 rows of them.
#include <atomic>

#include "tkv_int8.cuh"
#include "tkv_int8_attend.cuh"
#include "tkv_umma.cuh"  // fence_smem_to_async

namespace tkv {
namespace {

constexpr int kWPC = 4;      // warps per CTA
constexpr int kCtasPerSM = 3;
constexpr int kStages = 2;   // ring stages of a warp
constexpr int kSP = 2;       // pages per stage
constexpr int kThreads = 32 * kWPC;
static_assert(kWPC * kSP == kInt8StepPages, "");

// Pages that some row of a sequence sees, if it is this kernel's: pg0 .., in steps.
struct DecodeSeq {
  int len, q0, n, first, pg0, npg, steps;
};
// false: the lengths are not a valid sequence's
template <int RB>
__device__ __forceinline__ bool decode_seq(const Int8AttendArgs& a, int s, DecodeSeq& d) {
  d.len = __ldg(a.seq_lens + s);
  d.q0 = __ldg(a.cu_q + s);
  d.n = __ldg(a.cu_q + s + 1) - d.q0;
  d.steps = 0;
  if (!int8_attend_ok(a, d.len, d.q0, d.n)) return false;
  // rows of a (sequence, kv head) are below 2^30 (checked on the host)
  const int rows = d.n * a.grp;
  if (rows == 0 || rows > RB) return true;  // nothing, or the chunk kernel's
  d.first = a.window > 0 ? max(0, d.len - d.n - a.window + 1) : 0;
  d.pg0 = d.first / kPage;
  d.npg = (d.len + kPage - 1) / kPage - d.pg0;
  d.steps = (d.npg + kInt8StepPages - 1) / kInt8StepPages;
  return true;
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

template <int D>
constexpr int ring_bytes() {
  return kWPC * kStages * kSP * Int8Fmt<D>::BYTES;
}
// shared memory: the rings (at the end: the warps' results, or the weights of
// the runs), then the stage barriers
template <int D>
constexpr int smem_bytes() {
  return ring_bytes<D>() + kWPC * kStages * 8 + 16;
}

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, kCtasPerSM)
    int8_decode_kernel(const Int8AttendArgs a, const Int8Splits sp) {
  using F = Int8Fmt<D>;
  constexpr int RB = 8 * NT;         // rows of the MMA tiles
  constexpr int CI = D / 64;         // 16-channel chunks of one lane
  constexpr int NU = D / 32;         // 32-channel units of V
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_ml[kWPC][RB][2];
  // of a warp's rows: log2 of the largest product of weight and scale, m included (a lower
  // bound), and c = E - e.  Looked at rarely, so not in registers (16 rows of 128
  // channels have none left).
  __shared__ float2 s_row[kWPC][RB];
  __shared__ int s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // ---- this CTA's range of the steps: each thread counts its share of the
  // sequences, the thread whose share holds the range's first step finds it ----
  __shared__ long long s_sum[kWPC];
  __shared__ int s_seq, s_head, s_step;
  const int per = (a.num_seqs + kThreads - 1) / kThreads;
  const int sq_lo = min(a.num_seqs, static_cast<int>(threadIdx.x) * per);
  const int sq_hi = min(a.num_seqs, sq_lo + per);
  DecodeSeq d;
  long long mine = 0;
  for (int q = sq_lo; q < sq_hi; ++q) {
    if (!decode_seq<RB>(a, q, d) && blockIdx.x == 0) set_err(a.err, TKV_ERR_BAD_LENGTH);
    mine += d.steps;
  }
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) s_sum[warp] = upto;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWPC; ++w) {
    if (w < warp) upto += s_sum[w];
    total += s_sum[w];
  }
  total *= a.n_kv_heads;
  // a CTA's steps: as many as let the grid take them all
  const long long share =
      max(static_cast<long long>(sp.least), (total + gridDim.x - 1) / gridDim.x);
  const int me = blockIdx.x;
  long long at = share * me;
  if (at >= total) return;
  const long long end = min(total, at + share);
  {
    long long skip = at - (upto - mine) * a.n_kv_heads;
    if (skip >= 0 && skip < mine * a.n_kv_heads)
      for (int q = sq_lo; q < sq_hi; ++q) {
        decode_seq<RB>(a, q, d);
        const long long all = static_cast<long long>(d.steps) * a.n_kv_heads;
        if (skip < all) {
          s_seq = q;
          s_head = static_cast<int>(skip / d.steps);
          s_step = static_cast<int>(skip % d.steps);
          break;
        }
        skip -= all;
      }
  }
  __syncthreads();
  int s = s_seq, h = s_head, k0 = s_step;

  uint8_t* const ring = smem + warp * (kStages * kSP * F::BYTES);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + ring_bytes<D>()) + warp * kStages;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  int turns = 0;  // ring stages this warp has filled so far
  bool alive = true;

  for (;;) {  // the pairs of the range
    decode_seq<RB>(a, s, d);
    const int len = d.len, q0 = d.q0, n = d.n, first = d.first, rows = n * a.grp;
    const int k1 = static_cast<int>(min(static_cast<long long>(d.steps), k0 + (end - at)));
    if (k1 <= k0) return;  // lengths that changed during the call
    const int p_lo = d.pg0 + k0 * kInt8StepPages;
    const int p_hi = min(d.pg0 + d.npg, d.pg0 + k1 * kInt8StepPages);
    // this warp's steps k: pages p_lo + kSP (warp + kWPC k) ..
    const int w_lo = p_lo + kSP * warp;
    const int steps = alive && w_lo < p_hi ? (p_hi - w_lo + kSP * kWPC - 1) / (kSP * kWPC) : 0;
    const int32_t* bt = a.block_tables + static_cast<int64_t>(s) * a.max_blocks;
    // lane l holds the page of step 16 w + l / 2, page l % 2 (window w), checked
    // against the pool; the next window is loaded one window ahead
    auto load_ids = [&](int w) {
      const int p = w_lo + kSP * kWPC * (16 * w + (lane >> 1)) + (lane & 1);
      int id = p < p_hi ? __ldg(bt + p) : 0;
      if (id < 0 || id >= a.num_pages) {
        set_err(a.err, TKV_ERR_BAD_PAGE);
        id = 0;  // read in bounds; the sequence's output is not meaningful
      }
      return id;
    };
    int ids = load_ids(0), ids_next = 0;
    const uint8_t* const pool_h = a.pool + static_cast<int64_t>(h) * F::BYTES;
    const int64_t page_stride = static_cast<int64_t>(a.n_kv_heads) * F::BYTES;
    auto issue = [&](int k) {  // all lanes; k < steps
      const int p0 = __shfl_sync(0xffffffffu, ids, 2 * (k & 15));
      const int p1 = __shfl_sync(0xffffffffu, ids, 2 * (k & 15) + 1);
      if (lane == 0) {
        const uint64_t pol = l2_evict_first_policy();
        const bool two = w_lo + kSP * kWPC * k + 1 < p_hi;
        const int slot = (turns + k) % kStages;
        uint8_t* dst = ring + slot * (kSP * F::BYTES);
        uint64_t* bar = &bars[slot];
        mbar_arrive_expect_tx(bar, two ? 2 * F::BYTES : F::BYTES);
        bulk_g2s_hint(dst, pool_h + p0 * page_stride, F::BYTES, bar, pol);
        if (two) bulk_g2s_hint(dst + F::BYTES, pool_h + p1 * page_stride, F::BYTES, bar, pol);
      }
      // the window ends with step 15: its successor is in ids_next by now
      if ((k & 15) == 0) ids_next = load_ids((k >> 4) + 1);
      if ((k & 15) == 15) ids = ids_next;
    };
    int issued = 0;
#pragma unroll
    for (int k = 0; k < kStages; ++k)
      if (k < steps) issue(issued++);

    // ---- the query rows as B operands: lane (g, t) holds row 8 nt + g, channels
    // 16 (t + 4 ci) + 4 wi .. of k-slice 4 ci + wi.  bf16 rows are brought to
    // f16 by a power of two: the row's largest value lands in [1, 2), where steps of
    // 2^-24 keep bf16's 8 bits exact down to 2^-17 of it, and within 2^-25 of it below.
    uint32_t bq[NT][4 * CI][2];
    float ra[NT][2];     // 2^e * scale * log2(e) of rows 8 nt + 2 t, + 1
    int plim[NT][2];     // last position that those rows see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = 8 * nt + g;
      float up = 1.f;
      uint32_t w[CI][8];
#pragma unroll
      for (int ci = 0; ci < CI; ++ci)
#pragma unroll
        for (int e = 0; e < 8; ++e) w[ci][e] = 0u;
      if (r < rows) {
        const uint16_t* src = a.q + (q0 + r / a.grp) * a.q_t + (h * a.grp + r % a.grp) * a.q_h;
#pragma unroll
        for (int ci = 0; ci < CI; ++ci) {
          const uint4* s4 = reinterpret_cast<const uint4*>(src + 16 * (t + 4 * ci));
          const uint4 x = s4[0], y = s4[1];  // (the output may lie where they do)
          w[ci][0] = x.x, w[ci][1] = x.y, w[ci][2] = x.z, w[ci][3] = x.w;
          w[ci][4] = y.x, w[ci][5] = y.y, w[ci][6] = y.z, w[ci][7] = y.w;
        }
      }
      if (a.q_bf16) {
        float m = 0.f;
#pragma unroll
        for (int ci = 0; ci < CI; ++ci)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 f = unpack2<true>(w[ci][e]);
            m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        float down;
        int8_row_power(m, up, down);
#pragma unroll
        for (int ci = 0; ci < CI; ++ci)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 f = unpack2<true>(w[ci][e]);
            w[ci][e] = pack_h2(f.x * down, f.y * down);
          }
      }
#pragma unroll
      for (int ci = 0; ci < CI; ++ci)
#pragma unroll
        for (int wi = 0; wi < 4; ++wi) {
          bq[nt][4 * ci + wi][0] = w[ci][2 * wi];
          bq[nt][4 * ci + wi][1] = w[ci][2 * wi + 1];
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ra[nt][e] = __shfl_sync(0xffffffffu, up, 4 * (2 * t + e)) * a.alpha;
        const int rr = 8 * nt + 2 * t + e;
        plim[nt][e] = rr < rows ? len - n + rr / a.grp : -1;
      }
    }

    float o[2 * NU][NT][4], m[NT][2], l[NT][2];
    float vinv = 0x1p126f;  // 2^-E of the value scales
    bool shifted = false;   // c is not 0 in some row of the warp
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2 * NU; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }
    if (lane < RB) s_row[warp][lane] = make_float2(-INFINITY, 0.f);
    __syncwarp();
    const int tk = 4 * (g >> 1) + (g & 1);  // page token of S row g (row g + 8: tk + 2)
    const int unmasked_hi = len - n;        // positions up to here are seen by every row,
    const int unmasked_lo = a.window > 0 ? len - a.window : 0;  // from here on

    for (int k = 0; k < steps; ++k) {
      const int slot = (turns + k) % kStages;
      if (!mbar_wait_fast(&bars[slot], ((turns + k) / kStages) & 1, a.err)) {
        alive = false;
        break;
      }
      const uint8_t* st = ring + slot * (kSP * F::BYTES);
      const int pg = w_lo + kSP * kWPC * k;
      const bool two = pg + 1 < p_hi;
      // ---- scores ----
      float x[kSP][NT][4], sv[kSP][2];
      const bool masked = !two || (pg + 2) * kPage - 1 > unmasked_hi || pg * kPage < unmasked_lo;
#pragma unroll
      for (int p = 0; p < kSP; ++p) {
        // the absent second page of a run's last step reads the first one again
        const uint8_t* blk = st + (p == 0 || two ? p * F::BYTES : 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) x[p][nt][0] = x[p][nt][1] = x[p][nt][2] = x[p][nt][3] = 0.f;
#pragma unroll
        for (int ci = 0; ci < CI; ++ci) {
          const uint4 k1 = *reinterpret_cast<const uint4*>(blk + int8_k_unit(tk, t + 4 * ci));
          const uint4 k2 = *reinterpret_cast<const uint4*>(blk + int8_k_unit(tk + 2, t + 4 * ci));
          const uint32_t w1[4] = {k1.x, k1.y, k1.z, k1.w}, w2[4] = {k2.x, k2.y, k2.z, k2.w};
#pragma unroll
          for (int wi = 0; wi < 4; ++wi) {
            uint32_t a0, a1, a2, a3;
            int8_to_h2(w1[wi], a0, a2);
            int8_to_h2(w2[wi], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(x[p][nt], a0, a1, a2, a3, bq[nt][4 * ci + wi][0], bq[nt][4 * ci + wi][1]);
          }
        }
        const float2 s1 = *reinterpret_cast<const float2*>(blk + F::SCALE_OFF + 8 * tk);
        const float2 s2 = *reinterpret_cast<const float2*>(blk + F::SCALE_OFF + 8 * tk + 16);
        sv[p][0] = s1.y;
        sv[p][1] = s2.y;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          x[p][nt][0] *= s1.x * ra[nt][0];
          x[p][nt][1] *= s1.x * ra[nt][1];
          x[p][nt][2] *= s2.x * ra[nt][0];
          x[p][nt][3] *= s2.x * ra[nt][1];
        }
      }
      if (masked) {
#pragma unroll
        for (int p = 0; p < kSP; ++p)
#pragma unroll
          for (int r2 = 0; r2 < 2; ++r2) {
            const int pos = (pg + p) * kPage + tk + 2 * r2;
            if (pos >= len || pos < first || (p == 1 && !two)) sv[p][r2] = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const bool seen = pos <= plim[nt][e] && (p == 0 || two) &&
                                  (a.window == 0 || pos > plim[nt][e] - a.window);
                if (!seen) x[p][nt][2 * r2 + e] = -INFINITY;
              }
          }
      }
      // ---- references: move only when a score or a scale has outgrown them ----
      float mx[NT][2];
      bool need = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[nt][e] = fmaxf(fmaxf(x[0][nt][e], x[0][nt][2 + e]), fmaxf(x[1][nt][e], x[1][nt][2 + e]));
          need |= mx[nt][e] > m[nt][e] + kInt8Lazy;
        }
      float svm = fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[1][0], sv[1][1]));
      need |= svm * vinv > 1.f;
      // this lane's largest product of a row, from its tokens tk and tk + 2 of each page
      auto largest = [&](int nt, int e) {
        float y = -INFINITY;
#pragma unroll
        for (int p = 0; p < kSP; ++p)
#pragma unroll
          for (int r2 = 0; r2 < 2; ++r2) y = fmaxf(y, x[p][nt][2 * r2 + e] + int8_log2(sv[p][r2]));
        return y;
      };
      if (__builtin_expect(shifted, 0)) {  // rows with an e of their own: no weight may outgrow it
        const float E = int8_scale_exponent(vinv);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            need |= largest(nt, e) - m[nt][e] > E - s_row[warp][8 * nt + 2 * t + e].y + kInt8Lazy;
      }
      if (__builtin_expect(__any_sync(0xffffffffu, need), 0)) {
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) svm = fmaxf(svm, __shfl_xor_sync(0xffffffffu, svm, d));
        const float E0 = int8_scale_exponent(vinv);
        if (svm * vinv > 1.f) vinv = int8_scale_inverse(svm);
        const float E = int8_scale_exponent(vinv);
        bool some = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float y = mx[nt][e], z = largest(nt, e);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
              z = fmaxf(z, __shfl_xor_sync(0xffffffffu, z, d));
            }
            float2& row = s_row[warp][8 * nt + 2 * t + e];
            const float top = fmaxf(row.x, z), m0 = m[nt][e], e0 = E0 - row.y;
            if (y > m0 + kInt8Lazy) m[nt][e] = y;
            const float er = int8_row_exponent(top, m[nt][e], E);
            some |= er != E;
            __syncwarp();
            if (g == 0) row = make_float2(top, E - er);
            f[e] = 0.f;  // of O; a row without a reference has neither O nor l
            if (m0 != -INFINITY) {
              f[e] = fast_exp2((m0 - m[nt][e]) + (e0 - er));
              l[nt][e] *= fast_exp2(m0 - m[nt][e]);
            }
          }
#pragma unroll
          for (int i = 0; i < 2 * NU; ++i) {
            o[i][nt][0] *= f[0];
            o[i][nt][1] *= f[1];
            o[i][nt][2] *= f[0];
            o[i][nt][3] *= f[1];
          }
        }
        shifted = __any_sync(0xffffffffu, some);
        __syncwarp();
      }
      // ---- weights (where the scores were) and O ----
      if (!__builtin_expect(shifted, 0)) {
#pragma unroll
        for (int p = 0; p < kSP; ++p) {
          const float v1 = sv[p][0] * vinv * kInt8WeightUp, v2 = sv[p][1] * vinv * kInt8WeightUp;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float ref = m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1];
              const float pe = fast_exp2(x[p][nt][e] - ref);
              l[nt][e & 1] += pe;
              const bool none = masked && x[p][nt][e] == -INFINITY;
              x[p][nt][e] = none ? 0.f : pe * (e < 2 ? v1 : v2);  // whatever the scale holds
            }
        }
      } else {
        const float ve = kInt8WeightExp - int8_scale_exponent(vinv);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float ref = m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1];
            const float up = ve + s_row[warp][8 * nt + 2 * t + (e & 1)].y;
#pragma unroll
            for (int p = 0; p < kSP; ++p) {
              const float y = x[p][nt][e] - ref;
              l[nt][e & 1] += fast_exp2(y);
              const bool none = masked && x[p][nt][e] == -INFINITY;
              x[p][nt][e] = none ? 0.f : fast_exp2(y + (int8_log2(sv[p][e >> 1]) + up));
            }
          }
      }
#pragma unroll
      for (int p = 0; p < kSP; ++p) {
        const uint8_t* blk = st + (p == 0 || two ? p * F::BYTES : 0) + F::V_OFF;
        uint32_t b0[NT], b1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          b0[nt] = movmatrix_trans(pack_h2(x[p][nt][0], x[p][nt][1]));
          b1[nt] = movmatrix_trans(pack_h2(x[p][nt][2], x[p][nt][3]));
        }
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const uint4 vw = *reinterpret_cast<const uint4*>(blk + (u * 32 + lane) * 16);
          uint32_t a0, a1, a2, a3;
          int8_to_h2(vw.x, a0, a2);
          int8_to_h2(vw.y, a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[2 * u][nt], a0, a1, a2, a3, b0[nt], b1[nt]);
          int8_to_h2(vw.z, a0, a2);
          int8_to_h2(vw.w, a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[2 * u + 1][nt], a0, a1, a2, a3, b0[nt], b1[nt]);
        }
      }
      __syncwarp();
      if (issued < steps) issue(issued++);
    }
    if (!alive)  // let the copies in flight land (each wait bounded) before the ring is reused
      for (int k = max(0, issued - kStages); k < issued; ++k)
        mbar_wait(&bars[(turns + k) % kStages], ((turns + k) / kStages) & 1, nullptr);
    turns += issued;

    // ---- join the warps: rows normalised by their own sums, weighted by l 2^m ----
    float* const so = reinterpret_cast<float*>(smem);  // [warp][row][D]
    __syncthreads();                                   // every ring is idle
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nt][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int r = 8 * nt + 2 * t + e;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        // 2^(e - 5), subnormal at the least
        const float vs = int8_pow2(int8_scale_exponent(vinv) - s_row[warp][r].y) / kInt8WeightUp;
        if (g == 0) {
          s_ml[warp][r][0] = m[nt][e];
          s_ml[warp][r][1] = int8_sqrt(sum);
        }
        float* dst = so + (warp * RB + r) * D + 4 * g;
#pragma unroll
        for (int u = 0; u < NU; ++u)
          *reinterpret_cast<float4*>(dst + 32 * u) =
              make_float4(o[2 * u][nt][e] * inv * vs, o[2 * u][nt][2 + e] * inv * vs,
                          o[2 * u + 1][nt][e] * inv * vs, o[2 * u + 1][nt][2 + e] * inv * vs);
      }
    __syncthreads();
    // the CTAs that share the pair: its first step is in c0's range, its last in c1's
    int c0 = me, c1 = me;
    if (k0 > 0) c0 = static_cast<int>((at - k0) / share);
    if (k1 < d.steps) c1 = static_cast<int>((at - k0 + d.steps - 1) / share);
    const int ns = c1 - c0 + 1, slot = 2 * me + (me == c0 ? 1 : 0);
    for (int i = threadIdx.x; i < rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), c = i % (D / 4) * 4;
      float M = -INFINITY, W = 0.f, u[kWPC];
#pragma unroll
      for (int w = 0; w < kWPC; ++w) M = fmaxf(M, s_ml[w][r][0]);
#pragma unroll
      for (int w = 0; w < kWPC; ++w) {
        u[w] = int8_part_root(s_ml[w][r][1], s_ml[w][r][0], M);
        W = fmaf(u[w], u[w], W);
      }
      const float inv = W == 0.f ? 0.f : 1.f / W;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWPC; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(so + (w * RB + r) * D + c);
        const float f = u[w] * inv;
        acc.x = fmaf(f, v.x * u[w], acc.x);
        acc.y = fmaf(f, v.y * u[w], acc.y);
        acc.z = fmaf(f, v.z * u[w], acc.z);
        acc.w = fmaf(f, v.w * u[w], acc.w);
      }
      if (ns == 1) {
        int8_store4(a, (static_cast<int64_t>(q0 + r / a.grp) * a.num_q_heads + h * a.grp + r % a.grp) * D + c, acc);
      } else {
        *reinterpret_cast<float4*>(sp.part_o + static_cast<int64_t>(slot * RB + r) * D + c) = acc;
        if (c == 0) *reinterpret_cast<float2*>(sp.part_ml + (slot * RB + r) * 2) = make_float2(M, int8_sqrt(W));
      }
    }
    // ---- join the parts: the CTA that counts the last one ----
    bool last = false;
    if (ns > 1) {
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const unsigned int old = atomicAdd(sp.count + c0, 1u);
        s_last = old == static_cast<unsigned int>(ns - 1);
        if (s_last) sp.count[c0] = 0u;
      }
      __syncthreads();
      last = s_last;
    }
    if (last) {
      __threadfence();
      float* const su = reinterpret_cast<float*>(smem);  // [part][row] roots of weights
      auto part = [&](int i) { return i == 0 ? 2 * c0 + 1 : 2 * (c0 + i); };
      for (int r = warp; r < rows; r += kWPC) {
        auto load = [&](int i) {
          return __ldcg(reinterpret_cast<const float2*>(sp.part_ml + (part(i) * RB + r) * 2));
        };
        const float2 own = lane < ns ? load(lane) : make_float2(-INFINITY, 0.f);
        float M = own.x;
        for (int i = lane + 32; i < ns; i += 32) M = fmaxf(M, load(i).x);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
        float W = 0.f;
        for (int i = lane; i < ns; i += 32) {
          const float2 ml = i == lane ? own : load(i);
          const float u = int8_part_root(ml.y, ml.x, M);
          su[i * RB + r] = u;
          W = fmaf(u, u, W);
        }
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) W += __shfl_xor_sync(0xffffffffu, W, d);
        if (lane == 0) s_ml[0][r][0] = W == 0.f ? 0.f : 1.f / W;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < rows * (D / 4); i += kThreads) {
        const int r = i / (D / 4), c = i % (D / 4) * 4;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 16
        for (int k = 0; k < ns; ++k) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(
              sp.part_o + static_cast<int64_t>(part(k) * RB + r) * D + c));
          const float u = su[k * RB + r];
          acc.x = fmaf(u, v.x * u, acc.x);
          acc.y = fmaf(u, v.y * u, acc.y);
          acc.z = fmaf(u, v.z * u, acc.z);
          acc.w = fmaf(u, v.w * u, acc.w);
        }
        const float inv = s_ml[0][r][0];
        acc.x *= inv;
        acc.y *= inv;
        acc.z *= inv;
        acc.w *= inv;
        int8_store4(a, (static_cast<int64_t>(q0 + r / a.grp) * a.num_q_heads + h * a.grp + r % a.grp) * D + c, acc);
      }
    }

    // ---- the next pair ----
    at += k1 - k0;
    if (at >= end) return;
    k0 = 0;
    if (++h == a.n_kv_heads) {
      h = 0;
      for (int base = s + 1;; base += 32) {  // the next sequence of this kernel's
        DecodeSeq e;
        e.steps = 0;
        if (base + lane < a.num_seqs) decode_seq<RB>(a, base + lane, e);
        const unsigned int some = __ballot_sync(0xffffffffu, e.steps > 0);
        if (some) {
          s = base + __ffs(some) - 1;
          break;
        }
        if (base >= a.num_seqs) return;  // not reached: the range has steps left
      }
    }
    umma::fence_smem_to_async();  // what was written and read here, before copies come again
    __syncthreads();
  }
}

template <int D, int NT>
int launch_t(const Int8AttendArgs& a, const Int8Splits& sp, unsigned int grid, cudaStream_t stream) {
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return TKV_BACKEND_ERROR;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(int8_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             smem_bytes<D>()) != cudaSuccess)
      return TKV_BACKEND_ERROR;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  int8_decode_kernel<D, NT><<<grid, kThreads, smem_bytes<D>(), stream>>>(a, sp);
  return cudaGetLastError() == cudaSuccess ? TKV_OK : TKV_BACKEND_ERROR;
}

}  // namespace

int launch_int8_decode(const Int8AttendArgs& a, const Int8Splits& sp, int head_dim,
                       cudaStream_t stream) {
  const unsigned int grid = static_cast<unsigned int>(sp.ctas);
  if (head_dim == 128)
    return sp.rows <= 8 ? launch_t<128, 1>(a, sp, grid, stream) : launch_t<128, 2>(a, sp, grid, stream);
  return sp.rows <= 8 ? launch_t<64, 1>(a, sp, grid, stream) : launch_t<64, 2>(a, sp, grid, stream);
}

}  // namespace tkv
