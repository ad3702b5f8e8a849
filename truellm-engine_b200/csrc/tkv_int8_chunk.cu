// tkv_int8_chunk.cu -- attention over the paged int8 cache for chunks of query
// rows, on the 5th-generation tensor cores (tcgen05).
//
// A CTA takes 256 query rows (query token x q head of the kv head's group) of a
// (sequence, kv head) and a run of 64-token tiles of its pages.  Roles:
//   producers (4 warps)  tiles of codes, loaded one tile ahead into registers,
//                        become exact f16 integers in the K-major operands K
//                        [64 tokens][D] and V^T [D][64 tokens] (four buffers)
//   scales (1 warp)      the tile's scales to shared memory, and the pages of the
//                        tile three ahead to L2
//   MMA (2 warps)        one per softmax warpgroup: S = Q K^T into tensor memory
//                        (two buffers), O += P V with P read from there
//   softmax (2 x 4 warps) one thread per query row: score x key scale, online
//                        softmax, weight x value scale rounded once to f16 and
//                        written to tensor memory over the scores
// S of tile i + 1 is in tensor memory while the weights of tile i are computed;
// S of tile i + 2 takes the buffer of tile i once O += P V of tile i is done.
// Tiles of 64 tokens cost half again as much for S as tiles of 128 (N = 64 reads
// more shared memory per product: 49 cycles where 32 would do), but with 128
// there is room for one buffer only, and every warpgroup then waits for its
// products' latency at each tile (measured: 4800 cycles per 128 tokens).
// Measured, 32 q heads on 8 kv heads of 128 channels: 8 chunks of 512 tokens behind
// 4096 in 340 us, 858 TFLOP/s.  A tile of 256 rows takes 1900 cycles, of which the
// products are 1280; the two softmax warps of a scheduler take 1550 for the weights
// (exponentials alone 1024) and 300 to wait and signal.  A CTA's start (query rows,
// the first tile, whose reference needs a pass for the maximum) and end take
// 18000 cycles that nothing overlaps, as shared memory holds one CTA.
// Scales multiply finished 32-bit numbers only, so the codes enter both products
// exactly; a masked token's weight is exactly 0.
//
// Tensor memory of warpgroup w (256 columns): S of even and odd tiles at 0 and 64
// (their weights P, f16 pairs, over the first 32 columns), O at 128.  Column 8 (4
// u + j) + g of O is channel 32 u + 4 g + j: the order in which a V unit's words
// are stored without conflicts.
#include <limits.h>

#include <algorithm>
#include <atomic>

#include "tkv_int8_attend.cuh"
#include "tkv_umma.cuh"

namespace tkv {
namespace {

constexpr int kRows = 128;       // rows of a softmax warpgroup (the MMA's M)
constexpr int kTN = 64;          // tokens per tile
constexpr int kStages = 4;       // K and V buffers
constexpr int kPrefetch = 3;     // tiles that L2 is ahead (60000 tokens: 140 us without, 135 with)
constexpr int kTP = kTN / kPage; // pages per tile
constexpr int kSoftmax = 256, kProducers = 128;
constexpr int kCtaThreads = kSoftmax + kProducers + 128;  // + MMA (2 warps), scales, Q prefetch
// Registers a thread: launched with 128, then shared out by warpgroup (two tiles ahead
// in the producers' registers, 160 and 128: 346 us where this takes 340)
constexpr int kRegsSoftmax = 176, kRegsProducer = 96, kRegsMma = 64;
static_assert(kSoftmax * kRegsSoftmax + kProducers * kRegsProducer + 128 * kRegsMma <= kCtaThreads * 128,
              "the shares are no more than the launch has");

// True in one lane of the converged warp, the same one at every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(one));
  return one != 0;
}

// 32 words to this thread's lane, 32 consecutive columns
__device__ __forceinline__ void st32u(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
      "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32 "
      "};\n" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
      "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

// 16 consecutive columns of this thread's lane, in flight until wait_ld_of.
// (No memory clobber on either: only tensor memory is read, and the compiler may
// move shared-memory loads across them.)
__device__ __forceinline__ void ld16_issue(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];\n"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
        "=f"(v[14]), "=f"(v[15])
      : "r"(taddr));
}
// Waits for the loads in flight; v's values come out of this statement, so no
// use of them can move before it.
__device__ __forceinline__ void wait_ld_of(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]),
                 "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]),
                 "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :);
}

// n consecutive 32-bit columns of this thread's lane; load and wait are one
// statement, so nothing can use a value before it has arrived
__device__ __forceinline__ void ld16_wait(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "{\n\ttcgen05.ld.sync.aligned.32x32b.x16.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15 "
      "}, [%16];\n\ttcgen05.wait::ld.sync.aligned;\n\t}\n"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
        "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}

// 32 columns in the layout of an MMA accumulator fragment: 16 lanes (rows), lane l of
// the warp holding row l / 4 and columns 2 (l % 4), + 1 of every 8-column group (v[4
// g], v[4 g + 1]), and the same of row l / 4 + 8 (v[4 g + 2], v[4 g + 3])
__device__ __forceinline__ void ld_frag32(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "{\n\ttcgen05.ld.sync.aligned.16x256b.x4.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15 "
      "}, [%16];\n\ttcgen05.wait::ld.sync.aligned;\n\t}\n"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
        "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ float2 fmul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;\n"
      : "=l"(d)
      : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)));
  return *reinterpret_cast<const float2*>(&d);
}

__device__ __forceinline__ float absmax2(uint32_t bf16_pair) {
  const float2 f = unpack2<true>(bf16_pair);
  return fmaxf(fabsf(f.x), fabsf(f.y));
}
__device__ __forceinline__ uint32_t bf16_to_h2(uint32_t bf16_pair, float factor) {
  const float2 f = unpack2<true>(bf16_pair);
  return pack_h2(f.x * factor, f.y * factor);
}

// 16 scores of a row (tokens t ..) times their key scales (kInt8KeyDown included); MASKED: tokens that
// the row does not see (outside [pmin, plim]) become -inf.
template <bool MASKED>
__device__ __forceinline__ void scale_scores(float (&x)[16], const float4* ks4, int t, int pmin,
                                             int plim) {
#pragma unroll
  for (int c = 0; c < 16; c += 4) {
    const float4 k4 = ks4[c / 4];
    const float2 p0 = fmul2(make_float2(x[c], x[c + 1]), make_float2(k4.x, k4.y));
    const float2 p1 = fmul2(make_float2(x[c + 2], x[c + 3]), make_float2(k4.z, k4.w));
    x[c] = p0.x, x[c + 1] = p0.y, x[c + 2] = p1.x, x[c + 3] = p1.y;
  }
  if constexpr (MASKED) {
#pragma unroll
    for (int c = 0; c < 16; ++c) x[c] = t + c <= plim && t + c >= pmin ? x[c] : -INFINITY;
  }
}

// The weights of a tile's 64 tokens (scores at tensor-memory column ts, positions
// t ..): 2^(x ra + nm), added to sum, and times the value scales (2^-E 2^5 included)
// as f16 pairs; MASKED: 0 for tokens outside [pmin, plim].  Sixteen tokens at a
// time, one group's exponentials while the next one's scores are scaled.
template <bool MASKED>
__device__ __forceinline__ void tile_weights(uint32_t ts, const float4* ks4, const float4* vs4,
                                             float2 ra2, float nm, int t, int pmin, int plim,
                                             float2& sum, uint32_t (&pk)[32]) {
  const float2 nm2 = make_float2(nm, nm);
  float x[2][16];
  float2 s1 = make_float2(0.f, 0.f);
  ld16_issue(ts, x[0]);
  wait_ld_of(x[0]);
  ld16_issue(ts + 16, x[1]);
  scale_scores<MASKED>(x[0], ks4, t, pmin, plim);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float(&y)[16] = x[q & 1];
    float2 w[8];
#pragma unroll
    for (int c = 0; c < 16; c += 2) {
      const float2 e = ffma2(make_float2(y[c], y[c + 1]), ra2, nm2);
      w[c / 2] = make_float2(fast_exp2(e.x), fast_exp2(e.y));
    }
    if (q < 3) {
      wait_ld_of(x[(q + 1) & 1]);
      scale_scores<MASKED>(x[(q + 1) & 1], ks4 + 4 * (q + 1), t + 16 * (q + 1), pmin, plim);
    }
#pragma unroll
    for (int c = 0; c < 16; c += 4) {
      const float4 v4 = vs4[4 * q + c / 4];
      sum = fadd2(sum, w[c / 2]);
      s1 = fadd2(s1, w[c / 2 + 1]);
      float2 w0 = fmul2(w[c / 2], make_float2(v4.x, v4.y));
      float2 w1 = fmul2(w[c / 2 + 1], make_float2(v4.z, v4.w));
      if constexpr (MASKED) {  // whatever the scale holds
        if (y[c] == -INFINITY) w0.x = 0.f;
        if (y[c + 1] == -INFINITY) w0.y = 0.f;
        if (y[c + 2] == -INFINITY) w1.x = 0.f;
        if (y[c + 3] == -INFINITY) w1.y = 0.f;
      }
      pk[8 * q + c / 2] = pack_h2(w0.x, w0.y);
      pk[8 * q + c / 2 + 1] = pack_h2(w1.x, w1.y);
    }
    if (q < 2) ld16_issue(ts + 16 * (q + 2), y);
  }
  sum = fadd2(sum, s1);
}

template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N));
}

template <int D>
struct Sm {
  static constexpr int Q_BYTES = kRows * D * 2, K_BYTES = kTN * D * 2, V_BYTES = D * kTN * 2;
  static constexpr int Q_OFF = 0;                      // one operand per warpgroup
  static constexpr int K_OFF = Q_OFF + 2 * Q_BYTES;
  static constexpr int V_OFF = K_OFF + kStages * K_BYTES;
  static constexpr int KS_OFF = V_OFF + kStages * V_BYTES;   // [stage][64] f32 key scales 2^-9
  static constexpr int VS_OFF = KS_OFF + kStages * kTN * 4;  // [stage][64] value scales 2^-E 2^5
  static constexpr int VL_OFF = VS_OFF + kStages * kTN * 4;  // [stage][64] log2 of value scales
  // [stage] 2^-E of the tile, [stage] log2 of its smallest value scale
  static constexpr int VI_OFF = VL_OFF + kStages * kTN * 4;
  static constexpr int ROW_OFF = VI_OFF + 32;                // [256] f32 of the rows
  static constexpr int BAR_OFF = ROW_OFF + kSoftmax * 4;
  static constexpr int BYTES = BAR_OFF + 256;
  static_assert(2 * kStages * 4 <= ROW_OFF - VI_OFF, "");
  static_assert(BYTES <= 227 * 1024, "one CTA's shared memory");
  static_assert(BYTES <= (1 << 18), "descriptor address fields never carry");
  static constexpr uint32_t TWG = 256, TO = 128, TCOLS = 512;
};

// Brings the query rows of a later CTA into L2: they come from DRAM otherwise, and
// a CTA can do nothing before it has them (about 4 us at 128 channels).
template <int D>
__device__ __forceinline__ void prefetch_q(const Int8AttendArgs& a, const Int8ChunkSplits& sp, int cta,
                                           int lane) {
  if (cta >= static_cast<int>(gridDim.x)) return;
  const Int8ChunkItem it(sp, cta);
  const int bh = it.pair(sp), s = bh / a.n_kv_heads, h = bh - s * a.n_kv_heads;
  const int L = __ldg(a.seq_lens + s), q0 = __ldg(a.cu_q + s), n = __ldg(a.cu_q + s + 1) - q0;
  if (!int8_attend_ok(a, L, q0, n)) return;
  const uint32_t grp = a.grp, all_rows = static_cast<uint32_t>(n) * grp, r0 = it.row_tile(sp) * kSoftmax;
  for (uint32_t r = lane; r < kSoftmax && r0 + r < all_rows; r += 32) {
    const uint32_t rho = r0 + r, tok = rho / grp;
    const uint16_t* src = a.q + static_cast<int64_t>(q0 + tok) * a.q_t + (h * grp + rho - tok * grp) * a.q_h;
#pragma unroll
    for (int c = 0; c < D; c += 64) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(src + c));
  }
}

template <int D>
__global__ void __launch_bounds__(kCtaThreads, 1)
    int8_chunk_kernel(const Int8AttendArgs a, const Int8ChunkSplits sp) {
  using F = Int8Fmt<D>;
  using SM = Sm<D>;
  constexpr int UNITS = kPage * D / 16;           // 16-byte units of a page's K (or V) codes
  constexpr int UPT = kTP * UNITS / kProducers;   // units per producer thread and tile
  constexpr int PSTEP = kProducers / UNITS;       // pages covered by one unit of every thread
  static_assert(8 * kTP == 32, "a window of page ids is a lane each");
  extern __shared__ __align__(1024) uint8_t smem[];
  // Barriers (tile i counted from the CTA's first), of stage i % 4:
  //   kready          K stored (128 producer arrivals)
  //   vready          V and the scales stored (128 and 32 arrivals)
  //   kfree, vfree    S, O += P V of the tile done (a commit per warpgroup)
  // and of warpgroup w, [2 w + i % 2]:
  //   sdone           S done (commit)
  //   pready          P written (128 arrivals)
  //   odone           O += P V done (commit)
  // and qready: the Q operands staged (256 arrivals).
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + SM::BAR_OFF);
  uint64_t* const kready = bars;
  uint64_t* const vready = bars + kStages;
  uint64_t* const kfree = bars + 2 * kStages;
  uint64_t* const vfree = bars + 3 * kStages;
  uint64_t* const sdone = bars + 4 * kStages;
  uint64_t* const pready = sdone + 4;
  uint64_t* const odone = pready + 4;
  uint64_t* const qready = odone + 4;
  uint32_t* const tslot = reinterpret_cast<uint32_t*>(qready + 1);
  static_assert((4 * kStages + 13) * 8 + 4 <= 256, "the barriers fit their area");
  float* const ks_s = reinterpret_cast<float*>(smem + SM::KS_OFF);
  float* const vs_s = reinterpret_cast<float*>(smem + SM::VS_OFF);
  float* const vl_s = reinterpret_cast<float*>(smem + SM::VL_OFF);
  float* const vi_s = reinterpret_cast<float*>(smem + SM::VI_OFF);
  float* const row_s = reinterpret_cast<float*>(smem + SM::ROW_OFF);

  const int ctid = threadIdx.x, warp = ctid >> 5, lane = ctid & 31;
  const Int8ChunkItem it(sp, blockIdx.x);
  const int split = it.split, runs = it.runs;
  const int rt = it.row_tile(sp), bh = it.pair(sp), s = bh / a.n_kv_heads, h = bh - s * a.n_kv_heads;
  const int L = __ldg(a.seq_lens + s), q0 = __ldg(a.cu_q + s), n = __ldg(a.cu_q + s + 1) - q0;
  if (!int8_attend_ok(a, L, q0, n)) return;  // flagged by the decode kernel
  // rows of a (sequence, kv head) are below 2^30 (checked on the host)
  const uint32_t grp = a.grp, all_rows = static_cast<uint32_t>(n) * grp, r0 = rt * kSoftmax;
  if (all_rows <= kInt8DecodeRows || r0 >= all_rows) return;
  const int rows = min(all_rows - r0, static_cast<uint32_t>(kSoftmax));
  const int wgs = rows > kRows ? 2 : 1;
  // tiles that some row of this CTA sees, cut into runs
  const int p_first = L - n + static_cast<int>(r0 / grp);
  const int kv_end = L - n + static_cast<int>((r0 + rows - 1) / grp) + 1;
  const int kv_lo = a.window > 0 ? max(0, p_first - a.window + 1) : 0;
  const int tile0 = kv_lo / kTN, tiles = (kv_end + kTN - 1) / kTN - tile0;
  const int per = tiles / runs, more = tiles - per * runs;  // the first `more` runs have one more
  const int j_lo = tile0 + split * per + min(split, more), nj = per + (split < more ? 1 : 0);

  // ---- the Q operands: each softmax warp copies its 32 rows, 8 rows x 4 vectors at a
  // time (64 contiguous bytes a row; 8 lanes' 16-byte stores fill a core matrix), to
  // their places as they are ----
  const int wg = ctid >> 7;
  uint8_t* const qs = smem + SM::Q_OFF + wg * SM::Q_BYTES;
  if (ctid < kSoftmax) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int r = 32 * warp + 8 * g + (lane & 7);
      const uint32_t rho = r0 + min(r, rows - 1), tok = rho / grp;
      const uint16_t* src = a.q + static_cast<int64_t>(q0 + tok) * a.q_t + (h * grp + rho - tok * grp) * a.q_h;
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
        cp_async16_or_zero(smem_u32(qs + umma::umma_off(r & 127, 8 * (4 * c + (lane >> 3)), D)),
                           src + 8 * (4 * c + (lane >> 3)), r < rows ? 16 : 0);
    }
  }
  if (warp == 8) umma::alloc(tslot, SM::TCOLS);
  if (ctid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kready[i], kProducers);
      mbar_init(&vready[i], kProducers + 32);
      mbar_init(&kfree[i], wgs);
      mbar_init(&vfree[i], wgs);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sdone[i], 1);
      mbar_init(&pready[i], kRows);
      mbar_init(&odone[i], 1);
    }
    mbar_init(qready, kSoftmax);
    fence_mbar_init();
  }

  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = *tslot;
  constexpr uint32_t idS = umma::idesc_f16(kRows, kTN, false);
  constexpr uint32_t idO = umma::idesc_f16(kRows, D, false);

  // Of the warps that read pages, lane l holds the id of page 32 w + l of the run
  // (window w: 8 tiles), checked against the pool, and of the next window as loaded:
  // no load of codes waits for a load of the table
  const int32_t* const bt = a.block_tables + static_cast<int64_t>(s) * a.max_blocks;
  const uint8_t* const pool_h = a.pool + static_cast<int64_t>(h) * F::BYTES;
  const int64_t page_stride = static_cast<int64_t>(a.n_kv_heads) * F::BYTES;
  auto load_ids = [&](int w) {
    // the table may have dropped what the window passed
    const int p = j_lo * kTP + 32 * w + lane, n_pages = (kv_end + kPage - 1) / kPage;
    return p >= kv_lo / kPage && p < n_pages ? __ldg(bt + p) : 0;
  };
  auto checked = [&](int id) {
    if (id >= 0 && id < a.num_pages) return id;
    set_err(a.err, TKV_ERR_BAD_PAGE);
    return 0;  // read in bounds; the sequence's output is not meaningful
  };

  if (ctid >= kSoftmax && ctid < kSoftmax + kProducers) {
    // ============================ producers ============================
    regs_down<kRegsProducer>();
    const int tid = ctid - kSoftmax;
    int ids = checked(load_ids(0)), ids_next = load_ids(1);
    // K unit of this thread in page PSTEP i + tid / UNITS: slot x % 16 of chunk
    // x / 16 (x = tid % UNITS): 8 lanes read 128 bytes and fill one core matrix.
    const int x = tid % UNITS, pg0 = tid / UNITS;
    const int kc = x >> 4, ktok = (x & 15) ^ (2 * (kc & 3));
    const uint32_t k_dst = umma::umma_off(ktok, 16 * kc, D);
    // V unit: of its unit u the lane takes (g, t) so that 16 lanes' 8-byte stores
    // fill 128 bytes
    const int vu = x >> 5, vg = (lane >> 1) & 7, vt = (lane & 1) + 2 * (lane >> 4);
    const uint32_t v_src = F::V_OFF + int8_v_unit(vu, vg, vt);
    const uint32_t v_dst = 4 * vu * (16 * kTN) + (vt >> 1) * 128 + vg * 16 + (vt & 1) * 8;
    int pid[UPT];
    uint4 kr[UPT], vr[UPT];
    auto fetch_ids = [&](int i) {  // the pages of tile i of the run, in order of i
      if (i > 0 && (i & 7) == 0) {
        ids = checked(ids_next);
        ids_next = load_ids((i >> 3) + 1);
      }
#pragma unroll
      for (int k = 0; k < UPT; ++k)
        pid[k] = __shfl_sync(0xffffffffu, ids, (i & 7) * kTP + PSTEP * k + pg0);
    };
    auto load_k = [&]() {
#pragma unroll
      for (int i = 0; i < UPT; ++i)
        kr[i] = __ldg(reinterpret_cast<const uint4*>(pool_h + pid[i] * page_stride) + x);
    };
    auto load_v = [&]() {
#pragma unroll
      for (int i = 0; i < UPT; ++i)
        vr[i] = __ldg(reinterpret_cast<const uint4*>(pool_h + pid[i] * page_stride + v_src));
    };
    if (nj > 0) {
      fetch_ids(0);
      load_k();
      load_v();
    }
    for (int i = 0; i < nj; ++i) {
      const int st = i % kStages;
      const uint32_t before = ((i / kStages) & 1) ^ 1;  // parity of the stage's last use
      const bool more = i + 1 < nj;
      if (more) fetch_ids(i + 1);
      if (i >= kStages && !mbar_wait_near(&kfree[st], before, a.err)) break;
      uint8_t* const kd = smem + SM::K_OFF + st * SM::K_BYTES + k_dst;
#pragma unroll
      for (int k = 0; k < UPT; ++k) {
        const uint32_t w[4] = {kr[k].x, kr[k].y, kr[k].z, kr[k].w};
        uint32_t hv[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) int8_to_h2(w[e], hv[2 * e], hv[2 * e + 1]);
        uint8_t* d = kd + (PSTEP * k + pg0) * (32 * D);
        *reinterpret_cast<uint4*>(d) = make_uint4(hv[0], hv[1], hv[2], hv[3]);
        *reinterpret_cast<uint4*>(d + 128) = make_uint4(hv[4], hv[5], hv[6], hv[7]);
      }
      umma::fence_smem_to_async();
      mbar_arrive(&kready[st]);
      if (more) load_k();
      if (i >= kStages && !mbar_wait_near(&vfree[st], before, a.err)) break;
      uint8_t* const vd = smem + SM::V_OFF + st * SM::V_BYTES + v_dst;
#pragma unroll
      for (int k = 0; k < UPT; ++k) {
        const uint32_t w[4] = {vr[k].x, vr[k].y, vr[k].z, vr[k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t lo, hi;
          int8_to_h2(w[e], lo, hi);
          *reinterpret_cast<uint2*>(vd + e * (16 * kTN) + (PSTEP * k + pg0) * 256) = make_uint2(lo, hi);
        }
      }
      umma::fence_smem_to_async();
      mbar_arrive(&vready[st]);
      if (more) load_v();
    }
  } else if (ctid >= kSoftmax + kProducers) {
    // ============================ an MMA warp ============================
    regs_down<kRegsMma>();
    // its softmax warpgroup, known to be one number for the warp
    const int w = __shfl_sync(0xffffffffu, warp, 0) - (kSoftmax + kProducers) / 32;
    if (w == 2 && nj > 0) {
      // ---- the scales: lane l those of tokens 2 l, 2 l + 1 of a tile ----
      int ids = checked(load_ids(0)), ids_next = load_ids(1);
      auto load = [&](int i) {  // in order of i
        if (i > 0 && (i & 7) == 0) {
          ids = checked(ids_next);
          ids_next = load_ids((i >> 3) + 1);
        }
        const int id = __shfl_sync(0xffffffffu, ids, (i & 7) * kTP + (lane >> 3));
        return __ldg(reinterpret_cast<const float4*>(pool_h + id * page_stride + F::SCALE_OFF) + (lane & 7));
      };
      // tile j (later than i, not by a window or more) into L2, a page a lane
      auto prefetch_tile = [&](int i, int j) {
        const int id = __shfl_sync(0xffffffffu, (j >> 3) == (i >> 3) ? ids : ids_next,
                                   (j & 7) * kTP + (lane & 3));
        if (lane < kTP && j < nj && id >= 0 && id < a.num_pages)
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(pool_h + id * page_stride),
                       "r"(F::BYTES));
      };
      for (int j = 1; j < kPrefetch; ++j) prefetch_tile(0, j);
      float vinv = 0x1p126f;  // 2^-E
      float4 next = load(0);
      for (int i = 0; i < nj; ++i) {
        const int st = i % kStages;
        const float4 sr = next;  // key, value scale of two tokens
        if (i + 1 < nj) next = load(i + 1);
        prefetch_tile(i + 1, i + kPrefetch);
        // tokens that no row of the CTA sees count for nothing
        const int t0 = (j_lo + i) * kTN + 2 * lane;
        const bool in0 = t0 < kv_end && t0 >= kv_lo, in1 = t0 + 1 < kv_end && t0 + 1 >= kv_lo;
        const float v0 = in0 ? sr.y : 0.f, v1 = in1 ? sr.w : 0.f;
        float top = fmaxf(fmaxf(v0, v1), 0.f);
        float low = fminf(in0 ? v0 : INFINITY, in1 ? v1 : INFINITY);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          low = fminf(low, __shfl_xor_sync(0xffffffffu, low, d));
        }
        if (top * vinv > 1.f) vinv = int8_scale_inverse(top);
        if (i >= kStages && !mbar_wait_near(&vfree[st], ((i / kStages) & 1) ^ 1, a.err)) break;
        *reinterpret_cast<float2*>(ks_s + st * kTN + 2 * lane) = make_float2(sr.x * kInt8KeyDown, sr.z * kInt8KeyDown);
        *reinterpret_cast<float2*>(vs_s + st * kTN + 2 * lane) =
            make_float2(v0 * vinv * kInt8WeightUp, v1 * vinv * kInt8WeightUp);
        *reinterpret_cast<float2*>(vl_s + st * kTN + 2 * lane) = make_float2(int8_log2(v0), int8_log2(v1));
        if (lane == 0) {
          vi_s[st] = vinv;
          vi_s[kStages + st] = int8_log2(low);
        }
        mbar_arrive(&vready[st]);
      }
    }
    if (w == 3) prefetch_q<D>(a, sp, blockIdx.x + kInt8ChunkSMs, lane);
    if (w < wgs && nj > 0) {
      // The whole warp runs the loop and one lane issues: what the instructions take
      // is then known to be the same for the warp and stays in uniform registers
      // (issued from a loop of one lane, a tile's products took this warp 1300 cycles).
      bool ok = true;
      int last_s = -1, last_o = -1;
      const uint64_t dq = umma::smem_desc(smem_u32(smem + SM::Q_OFF + w * SM::Q_BYTES), 128, 16 * D);
      const uint64_t dk = umma::smem_desc(smem_u32(smem + SM::K_OFF), 128, 16 * D);
      const uint64_t dv = umma::smem_desc(smem_u32(smem + SM::V_OFF), 128, 16 * kTN);
      const uint32_t tS = __shfl_sync(0xffffffffu, tmem, 0) + w * SM::TWG, tO = tS + SM::TO;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait_near(bar, parity, a.err));
      };
      auto issue_s = [&](int i) {
        ok = wait(&kready[i % kStages], (i / kStages) & 1);
        if (!ok) return;
        umma::fence_after_sync();
        const uint64_t d = dk + (i % kStages) * (SM::K_BYTES >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma::mma_f16(tS + (i & 1) * kTN, dq + 16 * kk, d + 16 * kk, idS, kk > 0);
          umma::commit(&sdone[2 * w + (i & 1)]);
          umma::commit(&kfree[i % kStages]);
        }
        __syncwarp();
        last_s = i;
      };
      ok = wait(qready, 0);
      if (ok) issue_s(0);
      if (ok && nj > 1) issue_s(1);
      for (int i = 0; ok && i < nj; ++i) {
        ok = wait(&vready[i % kStages], (i / kStages) & 1) &&
             wait(&pready[2 * w + (i & 1)], (i >> 1) & 1);
        if (!ok) break;
        umma::fence_after_sync();
        const uint64_t d = dv + (i % kStages) * (SM::V_BYTES >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kTN / 16; ++kk)
            umma::mma_f16_ta(tO, tS + (i & 1) * kTN + 8 * kk, d + 16 * kk, idO, i > 0 || kk > 0);
          umma::commit(&odone[2 * w + (i & 1)]);
          umma::commit(&vfree[i % kStages]);
        }
        __syncwarp();
        last_o = i;
        if (i + 2 < nj) {
          // S of tile i + 2 overwrites the scores and weights of this one
          ok = wait(&odone[2 * w + (i & 1)], (i >> 1) & 1);
          if (ok) issue_s(i + 2);
        }
      }
      // no MMA may still run when tensor memory is released
      for (int i = max(0, last_s - 1); i <= last_s; ++i)
        mbar_wait_near(&sdone[2 * w + (i & 1)], (i >> 1) & 1, nullptr);
      for (int i = max(0, last_o - 1); i <= last_o; ++i)
        mbar_wait_near(&odone[2 * w + (i & 1)], (i >> 1) & 1, nullptr);
    }
  } else {
    // ============================ softmax ============================
    regs_up<kRegsSoftmax>();
    // ---- the Q operands: bf16 becomes f16 where it is ----
    {
      cp_async_wait_all();
      __syncwarp();
#pragma unroll 1
      for (int g = 0; g < 4; ++g) {
        const int r = 32 * warp + 8 * g + (lane & 7);
        uint4* const at = reinterpret_cast<uint4*>(qs + umma::umma_off(r & 127, 8 * (lane >> 3), D));
        float up = 1.f, down = 1.f, m = 0.f;
        if (a.q_bf16) {
          uint4 x[D / 32];
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            x[c] = at[32 * c];  // 4 core matrices of 8 channels on
            m = fmaxf(fmaxf(m, absmax2(x[c].x)), fmaxf(absmax2(x[c].y), fmaxf(absmax2(x[c].z), absmax2(x[c].w))));
          }
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          int8_row_power(m, up, down);
#pragma unroll
          for (int c = 0; c < D / 32; ++c)
            at[32 * c] = make_uint4(bf16_to_h2(x[c].x, down), bf16_to_h2(x[c].y, down),
                                    bf16_to_h2(x[c].z, down), bf16_to_h2(x[c].w, down));
        }
        if (lane < 8) row_s[r] = up;
      }
      umma::fence_smem_to_async();
      mbar_arrive(qready);
      __syncwarp();
    }
    // thread ctid owns row ctid
    const bool valid = ctid < rows;
    const int qi = valid ? static_cast<int>((r0 + ctid) / grp) : 0;
    // 2^e * scale * log2(e) * 2^9, not 0: a masked token's -inf times it stays -inf (and a score
    // is below 2^-21 with the smallest float)
    const float ra = fmaxf(row_s[ctid] * kInt8KeyUp * a.alpha, 0x1p-149f);
    if (wg < wgs && kRows * wg + 32 * (warp & 3) >= rows) {
      // no row of this warp exists: it only keeps the hand-overs going
      for (int i = 0; i < nj; ++i) {
        if (!mbar_wait_near(&sdone[2 * wg + (i & 1)], (i >> 1) & 1, a.err)) break;
        mbar_arrive(&pready[2 * wg + (i & 1)]);
      }
    } else if (wg < wgs) {
    const uint32_t lane_base = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t tS = tmem + wg * SM::TWG + lane_base, tO = tS + SM::TO;
    const int plim = valid ? L - n + qi : -1;  // last position that the row sees
    const int pmin = a.window > 0 ? max(0, plim - a.window + 1) : 0;
    // a row that does not exist sees nothing and has no reference to move
    float m = valid ? -INFINITY : 0.f, l = 0.f, vinv = 0x1p126f;
    // c = E - e of the row; shift: 0 when c is 0 in all rows of the warp, 2 when it is more
    // than kInt8Far in one.  row_s keeps log2 of the row's largest product of weight and
    // scale, m included (a lower bound).
    row_s[ctid] = -INFINITY;
    float c = 0.f;
    int shift = 0;
    bool ok = true;
    const float2 ra2 = make_float2(ra, ra);
    bool fresh = true;  // a row of the warp has no reference yet
    for (int i = 0; i < nj; ++i) {
      const int st = i % kStages, t0 = (j_lo + i) * kTN;
      ok = mbar_wait_near(&vready[st], (i / kStages) & 1, a.err) &&
           mbar_wait_near(&sdone[2 * wg + (i & 1)], (i >> 1) & 1, a.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      umma::fence_after_sync();
      const bool masked = __any_sync(0xffffffffu, valid && (t0 + kTN - 1 > plim || t0 < pmin));
      const float vnew = vi_s[st];
      const uint32_t tSi = tS + (i & 1) * kTN;
      const float4* ks4 = reinterpret_cast<const float4*>(ks_s + st * kTN);
      const float4* vs4 = reinterpret_cast<const float4*>(vs_s + st * kTN);
      bool plain = !fresh && vnew == vinv && shift < 2;
      if (plain) {
        // A pass with the reference and the power of two as they are: no maximum is
        // taken.  A sum of 2^kInt8Lazy or less shows that no p has outgrown the one; where
        // the other is a row's own, the weights themselves show that none has outgrown it.
        float2 sum = make_float2(0.f, 0.f);
        uint32_t pk[32];
        if (masked)
          tile_weights<true>(tSi, ks4, vs4, ra2, c - m, t0, pmin, plim, sum, pk);
        else
          tile_weights<false>(tSi, ks4, vs4, ra2, c - m, 0, 0, 0, sum, pk);
        float all = sum.x + sum.y;
        bool grown = all > kInt8LazyWeight;
        if (__builtin_expect(shift, 0)) {
          all *= fast_exp2(-c);
          uint32_t w = pk[0];  // f16s that are not negative, as whole numbers: infinity is 0x7c00
#pragma unroll
          for (int k = 1; k < 32; ++k) w = __vmaxu2(w, pk[k]);
          grown = all > kInt8LazyWeight || (w & 0xffffu) >= 0x7c00u || w >= 0x7c000000u;
        }
        plain = !__any_sync(0xffffffffu, grown);
        if (plain) {
          l += all;
          st32u(tSi, pk);
        }
      }
      if (!plain) {
        // A first reference, one that has to move, or a power of two of the value scales
        // that has: the tile's largest score (and product), O and l brought to the new
        // reference, then the weights.  (Compact code: it is rare, and instruction
        // fetches cost the CTA's start and end more than its loops.)
        const float4* vl4 = reinterpret_cast<const float4*>(vl_s + st * kTN);
        float mx = -INFINITY;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          float x[16];
          ld16_wait(tSi + 16 * q, x);
          scale_scores<true>(x, ks4 + 4 * q, t0 + 16 * q, pmin, plim);
#pragma unroll
          for (int k = 0; k < 16; k += 2) mx = fmaxf(mx, fmaxf(x[k], x[k + 1]));
        }
        mx *= ra;  // ra > 0 keeps the order
        const float m0 = m;
        const bool up = mx > m;
        m = up ? mx : m;
        l *= up ? (m0 == -INFINITY ? 0.f : fast_exp2(m0 - mx)) : 1.f;
        fresh = __any_sync(0xffffffffu, m == -INFINITY);
        const float E = int8_scale_exponent(vnew), e0 = int8_scale_exponent(vinv) - c;
        // The largest product is that of the largest score with the tile's smallest scale
        // or more.  Where that does not show a row to be loud enough, it is taken exactly.
        float top = fmaxf(row_s[ctid], mx + vi_s[kStages + st]);
        float er = valid ? int8_row_exponent(top, m, E) : E;
        if (__builtin_expect(__any_sync(0xffffffffu, er != E), 0)) {
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            float x[16];
            ld16_wait(tSi + 16 * q, x);
            scale_scores<true>(x, ks4 + 4 * q, t0 + 16 * q, pmin, plim);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const float4 v4 = vl4[4 * q + e / 4];
              top = fmaxf(top, fmaxf(fmaxf(fmaf(x[e], ra, v4.x), fmaf(x[e + 1], ra, v4.y)),
                                     fmaxf(fmaf(x[e + 2], ra, v4.z), fmaf(x[e + 3], ra, v4.w))));
            }
          }
          er = valid ? int8_row_exponent(top, m, E) : E;
        }
        row_s[ctid] = top;
        c = E - er;
        vinv = vnew;
        shift = __any_sync(0xffffffffu, c > kInt8Far) ? 2 : __any_sync(0xffffffffu, c != 0.f) ? 1 : 0;
        // O's factor (O is 0 in a row without a reference)
        const float f = m0 == -INFINITY ? (m == -INFINITY ? 1.f : 0.f) : fast_exp2((m0 - m) + (e0 - er));
        if (i > 0 && __any_sync(0xffffffffu, f != 1.f)) {
          // O holds the tiles before, once the last one's products are in
          ok = __all_sync(0xffffffffu,
                          mbar_wait_near(&odone[2 * wg + ((i - 1) & 1)], ((i - 1) >> 1) & 1, a.err));
          if (!ok) break;
          umma::fence_after_sync();
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 16) {
            float o[16];
            ld16_wait(tO + c0, o);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] *= f;
            umma::st16(tO + c0, o);
          }
        }
        const float nm = m == -INFINITY ? 0.f : -m;
        // P of tokens 16 q .. goes over columns 8 q .., whose scores have been read
        if (!__builtin_expect(shift, 0)) {
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            float x[16];
            uint32_t pw[8];
            ld16_wait(tSi + 16 * q, x);
            scale_scores<true>(x, ks4 + 4 * q, t0 + 16 * q, pmin, plim);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const float4 v4 = vs4[4 * q + e / 4];
              const float v[4] = {v4.x, v4.y, v4.z, v4.w};
              float w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float p = fast_exp2(fmaf(x[e + k], ra, nm));
                l += p;
                w[k] = x[e + k] == -INFINITY ? 0.f : p * v[k];  // masked: whatever the scale holds
              }
              pw[e / 2] = pack_h2(w[0], w[1]);
              pw[e / 2 + 1] = pack_h2(w[2], w[3]);
            }
            umma::st8(tSi + 8 * q, pw);
          }
        } else {
          const float ve = kInt8WeightExp - er;
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            float x[16];
            uint32_t pw[8];
            ld16_wait(tSi + 16 * q, x);
            scale_scores<true>(x, ks4 + 4 * q, t0 + 16 * q, pmin, plim);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const float4 v4 = vl4[4 * q + e / 4];
              const float v[4] = {v4.x, v4.y, v4.z, v4.w};
              float w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float y = fmaf(x[e + k], ra, nm);
                l += fast_exp2(y);
                w[k] = x[e + k] == -INFINITY ? 0.f : fast_exp2(y + (v[k] + ve));
              }
              pw[e / 2] = pack_h2(w[0], w[1]);
              pw[e / 2 + 1] = pack_h2(w[2], w[3]);
            }
            umma::st8(tSi + 8 * q, pw);
          }
        }
      }
      umma::wait_st();
      umma::fence_before_sync();
      mbar_arrive(&pready[2 * wg + (i & 1)]);
    }
    if (ok && nj > 0)
      ok = mbar_wait_near(&odone[2 * wg + ((nj - 1) & 1)], ((nj - 1) >> 1) & 1, a.err);
    ok = __all_sync(0xffffffffu, ok);
    umma::fence_after_sync();
    // ---- normalise and write the rows (a run's partial when the context is split),
    // eight channels a thread, 64 contiguous bytes a quad ----
    // 2^(e - 5) / l, where the power may be subnormal
    row_s[ctid] = (l == 0.f ? 0.f : 1.f / l) *
                  (int8_pow2(int8_scale_exponent(vinv) - c) / kInt8WeightUp);
    __syncwarp();
    const int64_t slot0 = static_cast<int64_t>(blockIdx.x - sp.whole) * kSoftmax;  // of a split item
    if (ok) {
#pragma unroll 1
      for (int hh = 0; hh < 2; ++hh) {
        const int row0 = (ctid & ~31) + 16 * hh + (lane >> 2);  // and + 8
        float inv[2];
        int64_t at[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t rho = r0 + row0 + 8 * k, tok = rho / grp;
          inv[k] = row_s[row0 + 8 * k];
          at[k] = (static_cast<int64_t>(q0 + tok) * a.num_q_heads + h * grp + rho - tok * grp) * D;
        }
#pragma unroll 1
        for (int u = 0; u < D / 32; ++u) {
          float o[16];
          __syncwarp();
          if (nj > 0) {
            ld_frag32(tO + 32 * u + (static_cast<uint32_t>(16 * hh) << 16), o);
          } else {
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = 0.f;
          }
          // column 8 j + g of the 32 is channel 4 g + j: this thread's g are 2 (lane %
          // 4) and + 1, eight channels in a row
          const int c = 32 * u + 8 * (lane & 3);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (row0 + 8 * k >= rows) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = o[4 * (e & 3) + 2 * k + (e >> 2)] * inv[k];
            if (runs > 1) {
              float4* dst = reinterpret_cast<float4*>(sp.part_o + (slot0 + row0 + 8 * k) * D + c);
              dst[0] = make_float4(v[0], v[1], v[2], v[3]);
              dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
              uint4 w;
              if (a.out_bf16)
                w = make_uint4(pack2<true>(v[0], v[1]), pack2<true>(v[2], v[3]),
                               pack2<true>(v[4], v[5]), pack2<true>(v[6], v[7]));
              else
                w = make_uint4(pack2<false>(v[0], v[1]), pack2<false>(v[2], v[3]),
                               pack2<false>(v[4], v[5]), pack2<false>(v[6], v[7]));
              *reinterpret_cast<uint4*>(a.out + at[k] + c) = w;
            }
          }
        }
      }
      if (runs > 1 && valid)
        *reinterpret_cast<float2*>(sp.part_ml + (slot0 + ctid) * 2) = make_float2(m, int8_sqrt(l));
    }
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (warp == 8) umma::dealloc(tmem, SM::TCOLS);
}

// Joins the runs of split contexts: a warp per row, the runs in order.
template <int D>
__global__ void __launch_bounds__(256) int8_chunk_join_kernel(const Int8AttendArgs a,
                                                              const Int8ChunkSplits sp) {
  const int lane = threadIdx.x & 31;
  const int item = blockIdx.x / (kSoftmax / 8);  // of the split ones
  const int r = blockIdx.x % (kSoftmax / 8) * 8 + (threadIdx.x >> 5);
  const Int8ChunkItem it(sp, sp.whole + item * sp.n);
  const int rt = it.row_tile(sp), bh = it.pair(sp), s = bh / a.n_kv_heads, h = bh - s * a.n_kv_heads;
  const int L = __ldg(a.seq_lens + s), q0 = __ldg(a.cu_q + s), n = __ldg(a.cu_q + s + 1) - q0;
  if (!int8_attend_ok(a, L, q0, n)) return;
  const uint32_t grp = a.grp, rows = static_cast<uint32_t>(n) * grp, rho = rt * kSoftmax + r;
  if (rows <= kInt8DecodeRows || rho >= rows) return;
  const long long slot0 = static_cast<long long>(item) * sp.n * kSoftmax + r;
  float M = -INFINITY;
  for (int i = 0; i < sp.n; ++i) M = fmaxf(M, __ldcg(sp.part_ml + (slot0 + static_cast<long long>(i) * kSoftmax) * 2));
  float W = 0.f, acc[D / 32] = {};
  for (int i = 0; i < sp.n; ++i) {
    const long long slot = slot0 + static_cast<long long>(i) * kSoftmax;
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(sp.part_ml + slot * 2));
    const float u = int8_part_root(ml.y, ml.x, M);
    W = fmaf(u, u, W);
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
      acc[c] = fmaf(u, __ldcg(sp.part_o + slot * D + (D / 32) * lane + c) * u, acc[c]);
  }
  const float inv = W == 0.f ? 0.f : 1.f / W;
  const uint32_t tok = rho / grp;
  const int64_t at = (static_cast<int64_t>(q0 + tok) * a.num_q_heads + h * grp + rho - tok * grp) * D +
                     (D / 32) * lane;
#pragma unroll
  for (int c = 0; c < D / 32; c += 2) {
    const uint32_t w = a.out_bf16 ? pack2<true>(acc[c] * inv, acc[c + 1] * inv)
                                  : pack2<false>(acc[c] * inv, acc[c + 1] * inv);
    *reinterpret_cast<uint32_t*>(a.out + at + c) = w;
  }
}

template <int D>
int launch_t(const Int8AttendArgs& a, const Int8ChunkSplits& sp, cudaStream_t stream) {
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return TKV_BACKEND_ERROR;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(int8_chunk_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Sm<D>::BYTES) != cudaSuccess)
      return TKV_BACKEND_ERROR;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const long long items = static_cast<long long>(a.num_seqs) * a.n_kv_heads * sp.row_tiles;
  const long long ctas = sp.whole + (items - sp.whole) * sp.n, joins = (items - sp.whole) * (kSoftmax / 8);
  int8_chunk_kernel<D><<<static_cast<unsigned int>(ctas), kCtaThreads, Sm<D>::BYTES, stream>>>(a, sp);
  if (cudaGetLastError() != cudaSuccess) return TKV_BACKEND_ERROR;
  if (sp.n > 1) {
    int8_chunk_join_kernel<D><<<static_cast<unsigned int>(joins), 256, 0, stream>>>(a, sp);
    if (cudaGetLastError() != cudaSuccess) return TKV_BACKEND_ERROR;
  }
  return TKV_OK;
}

}  // namespace

int launch_int8_chunk(const Int8AttendArgs& a, const Int8ChunkSplits& sp, int head_dim,
                      cudaStream_t stream) {
  return head_dim == 128 ? launch_t<128>(a, sp, stream) : launch_t<64>(a, sp, stream);
}

}  // namespace tkv
