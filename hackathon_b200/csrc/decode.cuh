// What the attention kernels over a decoding cache share (decode.cu, decode_mma.cu,
// decode_tc.cu, decode_f32.cu):
// arguments, the split of the work over blocks, and the walk of a block over its pieces.
#pragma once

#include <cuda.h>

#include <atomic>

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
  float scale_log2;
};

// How a call runs (host).
struct Plan {
  int kernel;       // which of them
  int dp, rows, rtiles, grid, split, min_units;
  int64_t segments;
  size_t part, part_ml, seg, bytes;  // workspace: offsets and size
};

// A block's way through its pieces.  A segment is one (sequence, kv head, row
// tile); a piece is the part of a segment that the block has, units tile ..
// tile + count - 1.
struct Walk {
  int b, head, rtile;
  int n, end;       // committed rows; rows with the drafts (0, 0 where the sequence does not fit)
  int tiles;        // units of the segment
  int tile, count;
  int64_t left;     // units (split) or segments (not split) still to do, this piece included
  int64_t u, total; // the piece's first unit among all of them
  int blocks;       // blocks that have work
  bool first;       // the block's first piece
};

template <int UNIT>
__device__ __forceinline__ void load_sequence(const Args& a, Walk& w) {
  const int n = a.lengths[w.b];
  const bool fits = n >= 0 && (int64_t)n + a.tokens <= a.capacity;
  if (!fits) atomicExch(&g_status, STATUS_ATTN);
  w.n = fits ? n : 0;
  w.end = fits ? n + a.tokens : 0;
  w.tiles = max(1, (w.end + UNIT - 1) / UNIT);  // one unit at least: somebody writes the zeros
}

template <int UNIT>
__device__ __forceinline__ int64_t units_of(const Args& a, int b) {
  const int n = a.lengths[b];
  const bool fits = n >= 0 && (int64_t)n + a.tokens <= a.capacity;
  return (int64_t)max(1, fits ? (n + a.tokens + UNIT - 1) / UNIT : 0) * a.kv_heads * a.rtiles;
}

// The block's first piece, with units of UNIT cached rows; every warp finds it
// for itself.
template <int UNIT>
__device__ __forceinline__ Walk start(const Args& a, int lane) {
  Walk w = {};
  w.first = true;
  const int per = a.kv_heads * a.rtiles;
  int64_t in_b;  // the first segment, within its sequence
  if (!a.split) {
    const int64_t segments = (int64_t)a.batch * per;
    const int64_t s0 = segments * blockIdx.x / gridDim.x;
    w.left = segments * (blockIdx.x + 1) / gridDim.x - s0;
    if (w.left <= 0) return w;
    w.b = (int)(s0 / per);
    in_b = s0 - (int64_t)w.b * per;
    load_sequence<UNIT>(a, w);
    w.count = w.tiles;
  } else {
    int64_t sum = 0;
    for (int i = lane; i < a.batch; i += 32) sum += units_of<UNIT>(a, i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    w.total = sum;
    const int64_t most = (sum + a.min_units - 1) / a.min_units;
    w.blocks = most < gridDim.x ? (int)most : (int)gridDim.x;
    if ((int)blockIdx.x >= w.blocks) return w;
    w.u = sum * blockIdx.x / w.blocks;
    w.left = sum * (blockIdx.x + 1) / w.blocks - w.u;
    int64_t before = 0;
    for (int i0 = 0;; i0 += 32) {
      // running sums of 32 sequences; the first that reaches past u holds it
      int64_t x = i0 + lane < a.batch ? units_of<UNIT>(a, i0 + lane) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + x > w.u);
      if (past) {
        const int k = __ffs(past) - 1;
        const int64_t prior = __shfl_sync(0xffffffffu, x, k ? k - 1 : 0);
        w.b = i0 + k;
        before += k ? prior : 0;
        break;
      }
      before += __shfl_sync(0xffffffffu, x, 31);
    }
    load_sequence<UNIT>(a, w);
    in_b = (w.u - before) / w.tiles;
    w.tile = (int)(w.u - before - in_b * w.tiles);
    w.count = (int)min((int64_t)(w.tiles - w.tile), w.left);
  }
  w.head = (int)(in_b / a.rtiles);
  w.rtile = (int)(in_b - (int64_t)w.head * a.rtiles);
  return w;
}

template <int UNIT>
__device__ __forceinline__ void next(const Args& a, Walk& w) {
  w.left -= a.split ? w.count : 1;
  if (w.left <= 0) return;
  w.u += w.count;
  w.first = false;
  if (++w.rtile == a.rtiles) {
    w.rtile = 0;
    if (++w.head == a.kv_heads) {
      w.head = 0;
      ++w.b;
      load_sequence<UNIT>(a, w);
    }
  }
  w.tile = 0;
  w.count = a.split ? (int)min((int64_t)w.tiles, w.left) : w.tiles;
}

// The workspace slot of an unfinished piece: a block has one for the segment it
// begins within, one for the segment it ends within.
__device__ __forceinline__ int slot(const Walk& w) { return 2 * blockIdx.x + (w.first ? 0 : 1); }

// The block with a segment's first unit writes down where its parts stand: in
// its own slot, and in the first slots of the blocks up to that of the last unit.
__device__ __forceinline__ void note_segment(const Args& a, const Walk& w) {
  if (!a.split || w.tile != 0) return;
  const int64_t s = ((int64_t)w.b * a.kv_heads + w.head) * a.rtiles + w.rtile;
  const int last = (int)(((w.u + w.tiles) * w.blocks - 1) / w.total);
  a.segments[s] = w.count == w.tiles ? make_int2(-1, -1) : make_int2(slot(w), last);
}

// Whether draft `tok` of the sequence sees cache row `key`.
__device__ __forceinline__ bool visible(const Args& a, const Walk& w, int tok, int key) {
  if (key < w.n) return true;
  if (key >= w.end) return false;
  const int j = key - w.n;
  return a.mask ? a.mask[w.b * a.mask_stride + (int64_t)tok * a.tokens + j] != 0 : j <= tok;
}

// Element offset, in q and the output, of query row r of a kv head.
__device__ __forceinline__ int64_t row_offset(const Args& a, int b, int head, int r) {
  const int tok = r / a.group;
  return (((int64_t)b * a.tokens + tok) * a.heads + head * a.group + (r - tok * a.group)) * a.d;
}

// Dynamic shared memory above 48 KB, allowed once for each kernel and device.
template <typename K>
inline int allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  C3B_CHECK_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    C3B_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  return C3B_OK;
}

// Tensor maps of the caches: rows of all heads one below the other, boxes of 128 bytes and `box_rows` rows.
int cache_maps(const Args& a, int box_rows, CUtensorMap* k, CUtensorMap* v);
int mma_blocks_per_sm(int dp, int rows);
int run_mma(bool h16, const Plan& pl, const Args& a, cudaStream_t s);
int run_tc(bool h16, const Plan& pl, const Args& a, cudaStream_t s);
int f32_blocks_per_sm(int dp, int rows);
int run_f32(const Plan& pl, const Args& a, cudaStream_t s);

}  // namespace dec
}  // namespace c3b
