// tkv_int8_attend.cu -- attention over the paged int8 cache: which kernel takes
// a sequence, and how contexts are split.
//
// A sequence with at most 16 query rows per kv head (query tokens x q heads of
// the group) is the decode kernel's, any other the chunk kernel's; both read the
// lengths on the device, so one call serves a batch that mixes them.  A call
// whose largest sequence has 16 rows or less launches the decode kernel alone.  (2 x
// 60000 tokens, 4 q heads a kv head: 16 rows 78 us by the decode kernel, 20 rows 106
// us by the other, whose time does not fall with the rows.)
#include <limits.h>

#include <algorithm>

#include "tkv_int8_attend.cuh"

namespace tkv {
namespace {

constexpr int kSlots = 148 * 3;  // resident CTAs of the decode kernel
// The workspace starts with the decode kernel's counters, in a place that does not
// depend on the call's sizes, so calls of different sizes that take turns with one
// workspace never write partials over each other's counters.
constexpr size_t kCounterBytes = 2048;
static_assert(kCounterBytes >= kSlots * sizeof(unsigned int), "");

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

// one CTA for every place on the GPU, or for every step where there are fewer
void decode_splits(Int8Splits& sp, int num_seqs, int num_kv_heads, int grp, int max_q, int max_len) {
  constexpr int kStep = kInt8StepPages * kPage;  // tokens
  const long long steps = (static_cast<long long>(max_len) + kStep - 1) / kStep;
  const long long pairs = static_cast<long long>(num_seqs) * num_kv_heads;
  sp.ctas = pairs >= kSlots
                ? kSlots
                : static_cast<int>(std::max<long long>(1, std::min<long long>(kSlots, pairs * steps)));
  // Contexts of 4 steps (512 tokens) or less are not cut.  8 kv heads, whole and in parts
  // of one step, us: 1 sequence, heads of 64, 256 tokens 5.6 and 7.3, 512 7.1 and 8.4, 640
  // 7.8 and 8.7, 1024 10.0 and 9.2; heads of 128 6.4 and 8.3, 8.2 and 8.7, 9.2 and 9.1,
  // 11.7 and 9.7; 16 sequences, heads of 128, 4 q heads each: 7.0 and 9.6, 10.1 and 11.6,
  // 11.3 and 16.2, 14.7 and 17.3, 2048 tokens 24.2 and 21.8.
  sp.least = steps <= 4 ? static_cast<int>(std::max<long long>(1, steps)) : 1;
  sp.rows = static_cast<int>(std::min<long long>(kInt8DecodeRows, static_cast<long long>(max_q) * grp));
}

int row_block(const Int8Splits& sp) { return sp.rows <= 8 ? 8 : 16; }

size_t decode_ml_bytes(const Int8Splits& sp) {
  return round256(static_cast<size_t>(2 * sp.ctas) * row_block(sp) * 8);
}

// bytes of the decode kernel's partials
size_t decode_bytes(const Int8Splits& sp, int head_dim) {
  return decode_ml_bytes(sp) + round256(static_cast<size_t>(2 * sp.ctas) * row_block(sp) * head_dim * 4);
}

// 64-token tiles of a run at least: 8 tokens behind 1200 (8 heads) 17.5 us, with 8
// tiles 21.0 us; behind 2400 19.1 us, with 2 tiles 20.6 us
constexpr int kMinTiles = 4;

// How chunk items are cut: those that fill whole rounds of the SMs not at all; the
// rest (or all, when there are few) into as many runs as leave no SM idle.
void chunk_splits(Int8ChunkSplits& sp, int num_seqs, int num_kv_heads, int grp, int max_q, int max_len) {
  const long long rows = static_cast<long long>(max_q) * grp;
  sp.row_tiles = static_cast<int>(std::max<long long>(1, (rows + kInt8ChunkRows - 1) / kInt8ChunkRows));
  const long long items = std::min<long long>(INT_MAX, static_cast<long long>(num_seqs) * num_kv_heads * sp.row_tiles);
  const long long rest = items % kInt8ChunkSMs;
  const long long tiles = (static_cast<long long>(max_len) + 63) / 64;
  sp.n = rest == 0 ? 1 : static_cast<int>(std::max<long long>(1, std::min(kInt8ChunkSMs / rest, tiles / kMinTiles)));
  sp.whole = static_cast<int>(sp.n > 1 ? items - rest : items);
}

// Bytes of the chunk kernel's share of the workspace, for every call of at most these
// sizes.  A call's own need rises and falls with them (`rest` does), but it never has
// more parts than the SMs, nor than its items' contexts have runs: rest * n <=
// min(148, items * tiles / kMinTiles).  That bound only grows.
size_t chunk_bytes(int num_seqs, int num_kv_heads, int grp, int max_q, int max_len, int head_dim) {
  const long long runs = (static_cast<long long>(max_len) + 63) / 64 / kMinTiles;
  if (runs <= 1) return 0;  // no context is cut
  const long long row_tiles =
      (static_cast<long long>(max_q) * grp + kInt8ChunkRows - 1) / kInt8ChunkRows;
  const long long items =
      std::min<long long>(kInt8ChunkSMs, static_cast<long long>(num_seqs) * num_kv_heads) * row_tiles;
  const size_t slots = static_cast<size_t>(std::min<long long>(kInt8ChunkSMs, items * runs)) * kInt8ChunkRows;
  return round256(slots * 8) + slots * head_dim * 4;
}

bool has_chunks(int grp, int max_q) {
  return static_cast<long long>(max_q) * grp > kInt8DecodeRows;
}

}  // namespace

// Never falls when num_seqs, num_q_heads, max_q or max_len grow.
size_t int8_attend_workspace(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                             int max_q, int max_len) {
  Int8Splits sp;
  decode_splits(sp, num_seqs, num_kv_heads, num_q_heads / num_kv_heads, max_q, max_len);
  size_t n = kCounterBytes + decode_bytes(sp, head_dim);
  const int grp = num_q_heads / num_kv_heads;
  if (has_chunks(grp, max_q)) n += chunk_bytes(num_seqs, num_kv_heads, grp, max_q, max_len, head_dim);
  return n;
}

int launch_int8_attend(const Int8AttendArgs& a, int head_dim, void* workspace, size_t,
                       cudaStream_t stream) {
  Int8Splits sp;
  decode_splits(sp, a.num_seqs, a.n_kv_heads, a.grp, a.max_q, a.max_len);
  const size_t pairs = static_cast<size_t>(a.num_seqs) * a.n_kv_heads;
  sp.count = static_cast<unsigned int*>(workspace);
  uint8_t* ws = static_cast<uint8_t*>(workspace) + kCounterBytes;
  uint8_t* chunk_ws = ws + decode_bytes(sp, head_dim);
  sp.part_ml = reinterpret_cast<float*>(ws);
  sp.part_o = reinterpret_cast<float*>(ws + decode_ml_bytes(sp));
  Int8ChunkSplits cs;
  chunk_splits(cs, a.num_seqs, a.n_kv_heads, a.grp, a.max_q, a.max_len);
  const bool chunks = has_chunks(a.grp, a.max_q);
  // more CTAs than a grid has (the items beyond `whole` add fewer than 148)
  if (chunks && static_cast<long long>(pairs) > (INT_MAX - kInt8ChunkSMs) / cs.row_tiles)
    return TKV_INVALID_ARGUMENT;
  const int st = launch_int8_decode(a, sp, head_dim, stream);
  if (st != TKV_OK || !chunks) return st;
  cs.part_ml = reinterpret_cast<float*>(chunk_ws);
  cs.part_o = reinterpret_cast<float*>(
      chunk_ws + round256((pairs * cs.row_tiles - cs.whole) * cs.n * kInt8ChunkRows * 8));
  return launch_int8_chunk(a, cs, head_dim, stream);
}

}  // namespace tkv
