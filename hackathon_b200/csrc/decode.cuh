// What the attention kernels over a decoding cache share (decode.cu, decode_mma.cu,
// decode_tc.cu, decode_f32.cu, decode_simt.cu):
// arguments, the split of the work over blocks, and the walk of a block over its pieces.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace c3b {
namespace dec {

enum { STATUS_ATTN = 41, STATUS_COMMIT = 42 };

struct Args {
  const void *q, *k, *v;
  void* out;
  const int* lengths;
  const uint8_t* mask;   // null: a chain, each draft sees those before it
  int64_t mask_stride;   // from one sequence's mask to the next (0: shared)
  int64_t capacity;
  float* part;           // [2 * blocks][tile rows][d]: sums of weighted values of unfinished segments
  float2* part_ml;       // [2 * blocks][tile rows]: their running maximum (base 2) and sum
  int2* segments;        // [segments]: the first slot and the last block of each, x = -1 where finished
  int batch, tokens, heads, kv_heads, group, d, dtype;
  int rows;              // query rows of a kv head: tokens * group
  int rtiles;            // row tiles of a kv head
  int split;             // 1: blocks share units evenly; 0: blocks take whole segments
  int min_units;         // units a block takes at least
  int ahead;             // units that a segment counts for besides its own: what starting and ending a piece costs
  float scale_log2, inv_group;
};

// A row's weights are 2^(score - reference).  The reference is a running maximum
// less lift(); it is raised when a score passes that maximum by more than LAG,
// which skips most rescales of the sums.  fp16 weights are lifted as far as the
// type reaches (2^(LAG + lift) = 2^15): they lose bits only below 2^-21 of the
// largest weight, and none above 2^-32 of it is lost.  bf16 and fp32 have
// exponents to spare, but so do their values: their weights are at most 1, so
// that a weighted value stays within the type.  The factor is the same in sums
// of weights and of weighted values, and drops out of their quotient.
constexpr float LAG = 8.f;
__host__ __device__ constexpr float lift(bool h16) { return h16 ? 7.f : -LAG; }

// How a call runs (host).
struct Plan {
  int kernel;       // which of them
  int dp, rows, rtiles, grid, split, min_units, ahead;
  int64_t segments;
  size_t part, part_ml, seg, bytes;  // workspace: offsets and size
};

// A block's way through its pieces.  A segment is one (sequence, kv head, row
// tile); a piece is the part of a segment that the block has, units tile ..
// tile + count - 1 (count = 0: none, the block only has some of the units
// `ahead` that the segment counts for).  All counts fit 32 bits (checked at
// launch).
struct Walk {
  int b, head, rtile;
  int n, end;       // committed rows; rows with the drafts (0, 0 where the sequence does not fit)
  int tiles;        // units of the segment
  int tile, count;
  int left;         // units (split) or segments (not split) after this piece; -1: no more
  int u, span;      // the segment's first unit among all of them, ahead included; the piece's end in the segment
  int share, extra; // units a block has: share + 1 for the first `extra` blocks, share for the others
  bool first;       // the block's first piece
};

template <int UNIT>
__device__ __forceinline__ void set_length(const Args& a, Walk& w, int n) {
  const bool fits = n >= 0 && n <= (int)a.capacity - a.tokens;
  if (!fits) atomicExch(&g_status, STATUS_ATTN);
  w.n = fits ? n : 0;
  w.end = fits ? n + a.tokens : 0;
  w.tiles = max(1, (w.end + UNIT - 1) / UNIT);  // one unit at least: somebody writes the zeros
}

// Units of a sequence of n committed rows.
template <int UNIT>
__device__ __forceinline__ int units_of(const Args& a, int n) {
  const bool fits = n >= 0 && n <= (int)a.capacity - a.tokens;
  return (a.ahead + max(1, fits ? (n + a.tokens + UNIT - 1) / UNIT : 0)) * (a.kv_heads * a.rtiles);
}

// The piece that begins `from` units into the segment, those ahead included.
__device__ __forceinline__ void take(const Args& a, Walk& w, int from) {
  w.span = min(a.ahead + w.tiles, from + w.left);
  w.tile = max(from - a.ahead, 0);
  w.count = max(w.span - a.ahead, 0) - w.tile;
}

// The block's first piece, with units of UNIT cached rows; every warp finds it
// for itself.
template <int UNIT>
__device__ __forceinline__ Walk start(const Args& a, int lane) {
  Walk w = {};
  w.first = true;
  const int per = a.kv_heads * a.rtiles;
  int in_b;  // the first segment, within its sequence
  if (!a.split) {
    const int segments = a.batch * per;
    const int share = segments / (int)gridDim.x, extra = segments - share * (int)gridDim.x;
    const int s0 = (int)blockIdx.x * share + min((int)blockIdx.x, extra);
    w.left = share + ((int)blockIdx.x < extra) - 1;
    if (w.left < 0) return w;
    w.b = s0 / per;
    in_b = s0 - w.b * per;
    set_length<UNIT>(a, w, a.lengths[w.b]);
    w.count = w.tiles;
  } else {
    const int mine = lane < a.batch ? a.lengths[lane] : 0;  // the first 32 sequences stay in registers
    int sum = lane < a.batch ? units_of<UNIT>(a, mine) : 0;
    for (int i = 32 + lane; i < a.batch; i += 32) sum += units_of<UNIT>(a, a.lengths[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int blocks = min((int)gridDim.x, (sum + a.min_units - 1) / a.min_units);  // that have work
    w.left = -1;
    if ((int)blockIdx.x >= blocks) return w;
    w.share = sum / blocks;
    w.extra = sum - w.share * blocks;
    const int u = (int)blockIdx.x * w.share + min((int)blockIdx.x, w.extra);
    w.left = w.share + ((int)blockIdx.x < w.extra);
    int before = 0;
    for (int i0 = 0;; i0 += 32) {
      // running sums of 32 sequences; the first that reaches past u holds it
      const int n = i0 == 0 ? mine : i0 + lane < a.batch ? a.lengths[i0 + lane] : 0;
      int x = i0 + lane < a.batch ? units_of<UNIT>(a, n) : 0;
      const int own = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + x > u);
      if (past) {
        const int k = __ffs(past) - 1;
        w.b = i0 + k;
        before += __shfl_sync(0xffffffffu, x - own, k);
        set_length<UNIT>(a, w, __shfl_sync(0xffffffffu, n, k));
        break;
      }
      before += __shfl_sync(0xffffffffu, x, 31);
    }
    in_b = (u - before) / (a.ahead + w.tiles);
    w.u = before + in_b * (a.ahead + w.tiles);
    take(a, w, u - w.u);
    w.left -= w.span - (u - w.u);
  }
  w.head = a.rtiles == 1 ? in_b : in_b / a.rtiles;
  w.rtile = in_b - w.head * a.rtiles;
  return w;
}

template <int UNIT>
__device__ __forceinline__ void next(const Args& a, Walk& w) {
  if (w.left <= 0) {
    w.left = -1;
    return;
  }
  w.u += a.ahead + w.tiles;
  w.first = false;
  if (++w.rtile == a.rtiles) {
    w.rtile = 0;
    if (++w.head == a.kv_heads) {
      w.head = 0;
      ++w.b;
      set_length<UNIT>(a, w, a.lengths[w.b]);
    }
  }
  if (a.split) {
    take(a, w, 0);
    w.left -= w.span;
  } else {
    w.tile = 0;
    w.count = w.tiles;
    --w.left;
  }
}

// The workspace slot of an unfinished piece: a block has one for the segment it
// begins within, one for the segment it ends within.
__device__ __forceinline__ int slot(const Walk& w) { return 2 * blockIdx.x + (w.first ? 0 : 1); }

// The block with a segment's first unit writes down where its parts stand: in
// its own slot, and in the first slots of the blocks up to that of the last unit.
__device__ __forceinline__ void note_segment(const Args& a, const Walk& w) {
  if (!a.split || w.tile != 0) return;
  const int64_t s = ((int64_t)w.b * a.kv_heads + w.head) * a.rtiles + w.rtile;
  const int end = w.u + a.ahead + w.tiles - 1;  // the segment's last unit
  const int large = w.extra * (w.share + 1);
  const int last = end < large ? end / (w.share + 1) : w.extra + (end - large) / w.share;
  a.segments[s] = w.count == w.tiles ? make_int2(-1, -1) : make_int2(slot(w), last);
}

// Whether draft `tok` of the sequence sees cache row `key`.
__device__ __forceinline__ bool visible(const Args& a, const Walk& w, int tok, int key) {
  if (key < w.n) return true;
  if (key >= w.end) return false;
  const int j = key - w.n;
  return a.mask ? a.mask[w.b * a.mask_stride + (int64_t)tok * a.tokens + j] != 0 : j <= tok;
}

// Which of cache rows key .. key + N - 1 (N = 8, 16 or 32) the lane's draft `tok`
// sees, as bits; the warp's drafts are tok of its lanes with `live` set.  Lanes
// side by side read neighbouring bytes of the mask, 32 / N drafts at a time.
template <int N>
__device__ __forceinline__ uint32_t see(const Args& a, const Walk& w, int tok, bool live, int key, int lane) {
  constexpr uint32_t ALL = N == 32 ? ~0u : (1u << (N & 31)) - 1u;
  const int first = key - w.n;  // the first row among the drafts; below 0: committed
  const int drafts = w.end - w.n;
  const uint32_t committed = first >= 0 ? 0u : first <= -N ? ALL : (1u << -first) - 1u;
  if (first >= drafts) return committed;
  if (!a.mask) {
    const int last = min(tok, drafts - 1) - first;  // of the N rows
    return last < 0 ? committed : committed | (last >= N - 1 ? ALL : (2u << last) - 1u);
  }
  const uint8_t* mask = a.mask + w.b * a.mask_stride;
  const int t0 = __reduce_min_sync(0xffffffffu, live ? tok : a.tokens);
  const int t1 = __reduce_max_sync(0xffffffffu, live ? tok : -1);
  const int j = first + lane % N;
  const bool draft = j >= 0 && j < drafts;
  uint32_t bits = 0;
  constexpr int PER = 32 / N;
#pragma unroll 4
  for (int t = t0; t <= t1; t += PER) {
    const int mine = t + lane / N;
    const uint32_t seen = __ballot_sync(0xffffffffu, draft && mine <= t1 && mask[(int64_t)mine * a.tokens + j] != 0);
    if (tok >= t && tok < t + PER) bits = seen >> ((tok - t) * N & 31);
  }
  return committed | (bits & ALL);
}

// The draft of query row r: r / group.  Rows are below 2^20, so (r + 1/2) / group is off by less than the 1/2.
__device__ __forceinline__ int token_of(const Args& a, int r) { return (int)(((float)r + 0.5f) * a.inv_group); }

// Element offset, in q and the output, of query row r of a kv head.
__device__ __forceinline__ int64_t row_offset(const Args& a, int b, int head, int r) {
  const int tok = token_of(a, r);
  return (((int64_t)b * a.tokens + tok) * a.heads + head * a.group + (r - tok * a.group)) * a.d;
}

// Tensor maps of the caches: rows of all heads one below the other, boxes of 128 bytes and `box_rows` rows.
int cache_maps(const Args& a, int box_rows, CUtensorMap* k, CUtensorMap* v);
int mma_blocks_per_sm(int dp, int rows);
int run_mma(bool h16, const Plan& pl, const Args& a, cudaStream_t s);
int run_tc(bool h16, const Plan& pl, const Args& a, cudaStream_t s);
int f32_unit(int dp, int rows);
int run_f32(const Plan& pl, const Args& a, cudaStream_t s);
int simt_unit(int dp);
int run_simt(const Plan& pl, const Args& a, cudaStream_t s);

}  // namespace dec
}  // namespace c3b
