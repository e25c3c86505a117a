// Attention of drafted tokens over a decoding cache, and the commit of the
// drafts that were accepted.
#include <cmath>

#include "decode.cuh"
#include "tc_prims.cuh"

namespace c3b {

namespace dec {

// Any type, head size up to 256 and alignment: one block for each query row,
// four warps stride over the cache rows, each with its own running maximum and
// sum, joined at the end.  It is there for what the others cannot take, not for
// speed: each query row reads its cache for itself in 2- or 4-byte pieces.  8 x 1
// tokens, 32 / 8 heads of 128 one element off alignment, 2000 rows: 1.76 ms in
// bf16, where the aligned call takes 28 us; heads of 100: 1.50 ms.
__global__ void __launch_bounds__(128) tree_rows_kernel(const Args a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int PL = 8;  // elements a lane: head_dim <= 256
  __shared__ float part[4][PL * 32], pm[4], pl[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x % a.heads;
  const int64_t token = blockIdx.x / a.heads;
  const int b = (int)(token / a.tokens), t = (int)(token % a.tokens);
  const int n = a.lengths[b];
  const bool fits = n >= 0 && (int64_t)n + a.tokens <= a.capacity;
  if (!fits && threadIdx.x == 0) atomicExch(&g_status, STATUS_ATTN);
  const int64_t q0 = (token * a.heads + h) * a.d;
  const int64_t kv0 = ((int64_t)b * a.kv_heads + h / (a.heads / a.kv_heads)) * a.capacity * a.d;
  const uint8_t* mask = a.mask ? a.mask + b * a.mask_stride + (int64_t)t * a.tokens : nullptr;
  float q[PL], o[PL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < PL; ++i) {
    q[i] = lane + 32 * i < a.d ? load_as_f32(a.q, a.dtype, q0 + lane + 32 * i) * a.scale_log2 : 0.f;
    o[i] = 0.f;
  }
  const int end = fits ? n + (mask ? a.tokens : t + 1) : 0;
  for (int j = warp; j < end; j += 4) {
    if (j >= n && mask && !mask[j - n]) continue;
    const int64_t at = kv0 + (int64_t)j * a.d;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < PL; ++i)
      if (lane + 32 * i < a.d) x = fmaf(q[i], load_as_f32(a.k, a.dtype, at + lane + 32 * i), x);
    x = warp_sum(x);
    const float mn = fmaxf(m, x), base = mn == -INFINITY ? 0.f : mn;
    const float f = exp2f(m - base), p = exp2f(x - base);
    m = mn;
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < PL; ++i)
      if (lane + 32 * i < a.d) o[i] = fmaf(p, load_as_f32(a.v, a.dtype, at + lane + 32 * i), o[i] * f);
  }
#pragma unroll
  for (int i = 0; i < PL; ++i) part[warp][lane + 32 * i] = o[i];
  if (lane == 0) pm[warp] = m, pl[warp] = l;
  __syncthreads();
  float top = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]));
  if (top == -INFINITY) top = 0.f;
  float f[4], sum = 0.f;
  for (int i = 0; i < 4; ++i) {
    f[i] = exp2f(pm[i] - top);
    sum += f[i] * pl[i];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing is zero
  for (int i = threadIdx.x; i < a.d; i += 128) {
    const float x = f[0] * part[0][i] + f[1] * part[1][i] + f[2] * part[2][i] + f[3] * part[3][i];
    store_from_f32(a.out, a.dtype, q0 + i, x * inv);
  }
}

// Joins the parts of the segments that were split, in block order: a warp for RW
// query rows of a segment.  At most 64 registers, so that its blocks fit beside
// the attention kernel's and are there when that ends; what it costs is a chain
// of three loads (segment, statistics, sums), so eight are on their way together.
// K: 128-dim halves of a head.
template <int K, int RW>
__global__ void __launch_bounds__(256, 4) tree_join_kernel(const Args a, int tile_rows, int items) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int item = (int)(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5));  // threads may pass 32 bits, warps do not
  if (item >= items) return;
  const int per = tile_rows / RW, seg = item / per, r0 = (item - seg * per) * RW;
  const int bh = seg / a.rtiles, row0 = (seg - bh * a.rtiles) * tile_rows + r0;
  if (row0 >= a.rows) return;
  const int2 where = a.segments[seg];
  if (where.x < 0) return;
  const int first = where.x / 2, parts = where.y - first + 1;
  // row r0 of part i's slot; rows past the last of the tile's are there, whatever they hold
  auto slot = [&](int i) { return (int64_t)(i ? 2 * (first + i) : where.x) * tile_rows + r0; };
  float mx[RW], sum[RW];
  float4 o[RW][K];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    mx[r] = -INFINITY, sum[r] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) o[r][k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int i0 = 0; i0 < parts; i0 += 32) {  // 32 parts at a time, their statistics a lane each
    float f[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      const bool on = i0 + lane < parts && row0 + r < a.rows;
      const float2 ml = on ? a.part_ml[slot(i0 + lane) + r] : make_float2(-INFINITY, 0.f);
      const float top = fmaxf(mx[r], warp_max(ml.x)), base = top == -INFINITY ? 0.f : top;
      const float before = exp2f(mx[r] - base);
      f[r] = exp2f(ml.x - base);
      mx[r] = top;
      sum[r] = sum[r] * before + f[r] * ml.y;
#pragma unroll
      for (int k = 0; k < K; ++k) o[r][k].x *= before, o[r][k].y *= before, o[r][k].z *= before, o[r][k].w *= before;
    }
    const int here = min(32, parts - i0);
    constexpr int NB = 8 / (K * RW);
#pragma unroll 1
    for (int i = 0; i < here; i += NB) {
      float4 x[NB][RW][K];
#pragma unroll
      for (int q = 0; q < NB; ++q)
#pragma unroll
        for (int r = 0; r < RW; ++r)
#pragma unroll
          for (int k = 0; k < K; ++k) {
            const int c = 4 * lane + 128 * k;
            x[q][r][k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c < a.d && i + q < here && row0 + r < a.rows)
              x[q][r][k] = *reinterpret_cast<const float4*>(a.part + (slot(i0 + i + q) + r) * a.d + c);
          }
#pragma unroll
      for (int q = 0; q < NB; ++q)
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          const float fi = __shfl_sync(0xffffffffu, f[r], i + q);
#pragma unroll
          for (int k = 0; k < K; ++k) {
            o[r][k].x = fmaf(fi, x[q][r][k].x, o[r][k].x);
            o[r][k].y = fmaf(fi, x[q][r][k].y, o[r][k].y);
            o[r][k].z = fmaf(fi, x[q][r][k].z, o[r][k].z);
            o[r][k].w = fmaf(fi, x[q][r][k].w, o[r][k].w);
          }
        }
    }
  }
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const float total = warp_sum(sum[r]);
    if (row0 + r >= a.rows) continue;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int64_t at = row_offset(a, bh / a.kv_heads, bh % a.kv_heads, row0 + r);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = 4 * lane + 128 * k;
      if (c >= a.d) break;
      const float4 x = make_float4(o[r][k].x * inv, o[r][k].y * inv, o[r][k].z * inv, o[r][k].w * inv);
      if (a.dtype == C3B_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at + c) = x;
      } else {
        const bool h16 = a.dtype == C3B_F16;
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at + c) =
            make_uint2(pack2h(make_float2(x.x, x.y), h16), pack2h(make_float2(x.z, x.w), h16));
      }
    }
  }
}

// The kernel that takes a call of these sizes: whole 16-byte pieces of a head,
// and cache rows that TMA's 32-bit coordinates reach; else tree_rows_kernel.
enum { ROWS_ANY = 0, MMA16, TC16, MMA32, SIMT32 };

static Plan make_plan(const c3b_tree_attn_params& p, int dtype) {
  Plan pl = {};
  const bool f32 = dtype == C3B_F32;
  if (p.head_dim % (f32 ? 4 : 8) || p.head_dim > 256 || p.capacity <= 0 ||
      (int64_t)p.batch * p.kv_heads * p.capacity >= (1ll << 31))
    return pl;
  const int64_t rows = (int64_t)p.tokens * (p.heads / p.kv_heads);
  if (rows >= 1 << 20) return pl;  // token_of()
  pl.dp = p.head_dim <= 64 ? 64 : p.head_dim <= 128 ? 128 : 256;
  int unit = 64, per_sm;
  if (f32 && rows <= 8) {
    pl.kernel = SIMT32;
    pl.rows = rows <= 4 ? 4 : 8;
    unit = simt_unit(pl.dp);
    per_sm = 1;
  } else if (f32) {
    pl.kernel = MMA32;
    pl.rows = rows <= 16 || pl.dp == 256 ? 16 : 32;
    unit = f32_unit(pl.dp, pl.rows);
    per_sm = 1;
  } else if (pl.dp <= 128 && rows > 32) {
    // 33 to 128 rows: one tile for both softmax groups; more: a tile each.  At head size 128 mma.sync takes 52 us for 17
    // rows and this kernel 67, but 81 against 71 for 33 rows and 169 against 79 for 128 (16 sequences of 500 to 4000
    // rows, 8 heads).  At head size 64 mma.sync would stay ahead up to 64 rows (48 us against 54).
    pl.kernel = TC16;
    unit = 128;
    pl.rows = rows <= 128 ? 128 : 256;
    per_sm = 1;
  } else {
    pl.kernel = MMA16;
    pl.rows = rows <= 16 || pl.dp == 256 ? 16 : 32;
    per_sm = mma_blocks_per_sm(pl.dp, pl.rows);
  }
  pl.rtiles = (int)((rows + pl.rows - 1) / pl.rows);
  pl.segments = (int64_t)p.batch * p.kv_heads * pl.rtiles;
  const int64_t blocks = (int64_t)sm_count() * per_sm;
  const int64_t units = (p.capacity + unit - 1) / unit;
  pl.split = p.capacity > 256;
  pl.min_units = 256 / unit;
  // Starting and ending a piece costs about as much as 3 units (queries, masks of the last unit, the join of the
  // groups), 8 of the tcgen05 kernel's.  0, 1, 3 and 8 of them measured 34, 28, 24 and 26 us for 128 fp32 segments of 0 to
  // 1000 rows, 50, 44, 38 and 40 us for 512 bf16 segments of 100 to 1500, 67, 65, 65 and 65 us for 256 of 500 to 7000;
  // tcgen05: 0, 4, 8 and 16 of them 202, 118, 106 and 110 us for 512 segments of 100 to 1500 rows (64 query rows
  // each), 179, 169, 167 and 173 us for 128 of 2000 to 4100 (512 query rows).
  pl.ahead = pl.kernel == TC16 ? 8 : 3;
  const int64_t grid = pl.split ? pl.segments * units : pl.segments;
  if (pl.segments * (units + pl.ahead) >= (1ll << 31) || pl.segments * pl.rows >= (1ll << 31)) return Plan{};  // 32-bit counts
  pl.grid = (int)(grid < blocks ? grid : blocks);
  if (pl.split) {
    pl.part_ml = (size_t)2 * pl.grid * pl.rows * p.head_dim * 4;
    pl.seg = pl.part_ml + (size_t)2 * pl.grid * pl.rows * 8;
    pl.bytes = pl.seg + (size_t)pl.segments * 8;
  }
  return pl;
}

struct CommitArgs {
  void* cache[2];
  const int *lengths, *path, *accepted;
  int* new_lengths;
  int64_t capacity;
  int batch, kv_heads, path_len, units;  // units of sizeof(W) bytes a row
};

// A warp for each sequence, head and cache.  The path rises, so row i never
// reads what a row before it wrote: a piece is loaded whole, then stored.
template <typename W>
__global__ void __launch_bounds__(128) commit_kernel(const CommitArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (item >= (int64_t)a.batch * a.kv_heads * 2) return;
  const int which = (int)(item & 1);
  const int64_t bh = item >> 1;
  const int b = (int)(bh / a.kv_heads);
  const int n = a.lengths[b], m = a.accepted[b];
  const int* path = a.path + (int64_t)b * a.path_len;
  bool ok = n >= 0 && m >= 0 && m <= a.path_len && (int64_t)n + m <= a.capacity;
  bool moves = false;
  if (ok) {
    for (int i = lane; i < m; i += 32) {
      const int r = path[i], before = i > 0 ? path[i - 1] : -1;
      ok = ok && r > before && r >= 0 && (int64_t)n + r < a.capacity;
      moves = moves || r != i;
    }
  }
  ok = __all_sync(0xffffffffu, ok);
  moves = __any_sync(0xffffffffu, moves);
  if (lane == 0 && which == 0 && bh % a.kv_heads == 0) {
    a.new_lengths[b] = ok ? n + m : n;
    if (!ok) atomicExch(&g_status, STATUS_COMMIT);
  }
  if (!ok || !moves) return;
  W* base = static_cast<W*>(a.cache[which]) + (bh * a.capacity + n) * a.units;
  constexpr int NB = 4;
  const int64_t total = (int64_t)m * a.units;
  for (int64_t e0 = 0; e0 < total; e0 += 32 * NB) {
    W v[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int64_t e = e0 + 32 * i + lane;
      if (e < total) v[i] = base[(int64_t)path[e / a.units] * a.units + e % a.units];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int64_t e = e0 + 32 * i + lane;
      if (e < total) base[e] = v[i];
    }
    __syncwarp();
  }
}

}  // namespace dec

int64_t tree_attn_workspace(const c3b_tree_attn_params& p, int dtype) {
  if (p.batch <= 0 || p.tokens <= 0 || p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads) return 0;
  return (int64_t)dec::make_plan(p, dtype).bytes;
}

// in: q, k cache, v cache, lengths, [mask] ; out: o, [workspace]
int launch_tree_attn(const c3b_tensor* in, int n_in, const c3b_tensor* out, int n_out, const c3b_tree_attn_params& p,
                     cudaStream_t s) {
  using namespace dec;
  C3B_REQUIRE(n_in == (p.mask_mode ? 5 : 4) && (n_out == 1 || n_out == 2),
              "tree attention: q, k, v, lengths [, mask] -> out [, workspace]");
  const c3b_tensor &q = in[0], &k = in[1], &v = in[2], &len = in[3];
  C3B_REQUIRE(is_float(q.dtype) && k.dtype == q.dtype && v.dtype == q.dtype && out[0].dtype == q.dtype,
              "tree attention: f32, bf16 or fp16, the same for q, caches and output");
  C3B_REQUIRE(p.batch >= 0 && p.tokens >= 0 && p.heads > 0 && p.kv_heads > 0 && p.heads % p.kv_heads == 0,
              "tree attention: heads is a multiple of kv_heads");
  C3B_REQUIRE(p.head_dim >= 1 && p.head_dim <= 256, "tree attention: head_dim is 1 to 256");
  // rows are rounded up to whole units in 32 bits
  C3B_REQUIRE(p.capacity >= 0 && p.capacity <= (1ll << 31) - 256, "tree attention: the capacity is 0 to 2^31 - 256");
  // the kernels multiply by scale / ln 2
  C3B_REQUIRE(std::isfinite(p.scale * 1.4426950408889634f) && p.scale > 0.f, "tree attention: the scale is positive and below 2e38");
  const int64_t rows = (int64_t)p.batch * p.tokens * p.heads;
  C3B_REQUIRE(numel(q) == rows * p.head_dim && numel(out[0]) == numel(q),
              "tree attention: q and the output are [batch, tokens, heads, head_dim]");
  const int64_t kv = (int64_t)p.batch * p.kv_heads * p.capacity * p.head_dim;
  C3B_REQUIRE(numel(k) == kv && numel(v) == kv, "tree attention: caches are [batch, kv_heads, capacity, head_dim]");
  C3B_REQUIRE(len.dtype == C3B_I32 && numel(len) == p.batch, "tree attention: lengths are int32 [batch]");
  C3B_REQUIRE(p.mask_mode >= 0 && p.mask_mode <= 2, "tree attention: bad mask mode");
  const int64_t tt = (int64_t)p.tokens * p.tokens;
  if (p.mask_mode)
    C3B_REQUIRE(in[4].dtype == C3B_U8 && numel(in[4]) == (p.mask_mode == 2 ? p.batch * tt : tt),
                "tree attention: the mask is one byte an entry, [tokens, tokens] or [batch, tokens, tokens]");
  for (int i = 0; i < n_in; ++i) C3B_REQUIRE(!overlaps(out[0], in[i]), "tree attention: the output overlaps an input");
  if (rows == 0) return C3B_OK;
  C3B_REQUIRE(rows < (1ll << 31), "tree attention: too many query rows");
  Args a = {};
  a.q = q.ptr, a.k = k.ptr, a.v = v.ptr, a.out = out[0].ptr;
  a.lengths = (const int*)len.ptr;
  a.mask = p.mask_mode ? (const uint8_t*)in[4].ptr : nullptr;
  a.mask_stride = p.mask_mode == 2 ? tt : 0;
  a.capacity = p.capacity;
  a.batch = p.batch, a.tokens = p.tokens, a.heads = p.heads, a.kv_heads = p.kv_heads, a.d = p.head_dim;
  a.group = p.heads / p.kv_heads;
  a.rows = p.tokens * a.group;
  a.inv_group = 1.f / (float)a.group;
  a.dtype = q.dtype;
  a.scale_log2 = p.scale * 1.4426950408889634f;
  const uintptr_t at = (uintptr_t)q.ptr | (uintptr_t)k.ptr | (uintptr_t)v.ptr | (uintptr_t)out[0].ptr;
  const Plan pl = make_plan(p, q.dtype);
  if (pl.kernel != ROWS_ANY && at % 16 == 0) {
    if (pl.bytes) {
      C3B_REQUIRE(n_out == 2 && numel(out[1]) * dtype_size(out[1].dtype) >= pl.bytes && ((uintptr_t)out[1].ptr & 15) == 0,
                  "tree attention: needs a workspace of " + std::to_string(pl.bytes) + " bytes, 16-byte aligned");
      for (int i = 0; i < n_in; ++i) C3B_REQUIRE(!overlaps(out[1], in[i]), "tree attention: the workspace overlaps an input");
      C3B_REQUIRE(!overlaps(out[1], out[0]), "tree attention: the workspace overlaps the output");
      a.part = (float*)out[1].ptr;
      a.part_ml = (float2*)((char*)out[1].ptr + pl.part_ml);
      a.segments = (int2*)((char*)out[1].ptr + pl.seg);
    }
    a.rtiles = pl.rtiles;
    a.split = pl.split;
    a.min_units = pl.min_units;
    a.ahead = pl.split ? pl.ahead : 0;
    const bool h16 = q.dtype == C3B_F16;
    if (int rc = pl.kernel == SIMT32  ? run_simt(pl, a, s)
                 : pl.kernel == MMA32 ? run_f32(pl, a, s)
                 : pl.kernel == TC16  ? run_tc(h16, pl, a, s)
                                      : run_mma(h16, pl, a, s))
      return rc;
    if (!pl.split) return C3B_OK;
    // four rows a warp once one a warp would take several rounds of the GPU
    const int rw = p.head_dim <= 128 && pl.segments * pl.rows > 64ll * sm_count() ? 4 : 1;
    const int items = (int)(pl.segments * pl.rows / rw);
    auto join = p.head_dim > 128 ? tree_join_kernel<2, 1> : rw == 4 ? tree_join_kernel<1, 4> : tree_join_kernel<1, 1>;
    return launch_pdl(join, (int)((items + 7ll) / 8), 256, 0, s, a, pl.rows, items);
  }
  return launch_pdl(tree_rows_kernel, (int)rows, 128, 0, s, a);
}

// in: lengths, path, accepted ; out: k cache, v cache, new lengths
int launch_kv_commit(const c3b_tensor* in, const c3b_tensor* out, const c3b_kv_commit_params& p, cudaStream_t s) {
  using namespace dec;
  const c3b_tensor &len = in[0], &path = in[1], &acc = in[2];
  C3B_REQUIRE(p.batch >= 0 && p.kv_heads >= 0 && p.head_dim >= 0 && p.path >= 0, "kv commit: bad extents");
  C3B_REQUIRE(p.capacity >= 0 && p.capacity < (1ll << 31), "kv commit: bad capacity");
  C3B_REQUIRE(len.dtype == C3B_I32 && numel(len) == p.batch && acc.dtype == C3B_I32 && numel(acc) == p.batch,
              "kv commit: lengths and accepted are int32 [batch]");
  C3B_REQUIRE(path.dtype == C3B_I32 && numel(path) == (int64_t)p.batch * p.path, "kv commit: path is int32 [batch, longest path]");
  const int64_t kv = (int64_t)p.batch * p.kv_heads * p.capacity * p.head_dim;
  C3B_REQUIRE(is_float(out[0].dtype) && out[1].dtype == out[0].dtype && numel(out[0]) == kv && numel(out[1]) == kv,
              "kv commit: caches are [batch, kv_heads, capacity, head_dim], of one type");
  C3B_REQUIRE(out[2].dtype == C3B_I32 && numel(out[2]) == p.batch, "kv commit: the new lengths are int32 [batch]");
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 3; ++j) {
      C3B_REQUIRE(!overlaps(out[i], in[j]), "kv commit: an output overlaps an input");
      C3B_REQUIRE(i == j || !overlaps(out[i], out[j]), "kv commit: the outputs overlap");
    }
  if (p.batch == 0) return C3B_OK;
  C3B_REQUIRE(p.kv_heads > 0, "kv commit: no heads");
  CommitArgs a = {};
  a.cache[0] = out[0].ptr, a.cache[1] = out[1].ptr;
  a.lengths = (const int*)len.ptr, a.path = (const int*)path.ptr, a.accepted = (const int*)acc.ptr;
  a.new_lengths = (int*)out[2].ptr;
  a.capacity = p.capacity;
  a.batch = p.batch, a.kv_heads = p.kv_heads, a.path_len = p.path;
  const int64_t bytes = (int64_t)p.head_dim * dtype_size(out[0].dtype);
  const uintptr_t at = (uintptr_t)out[0].ptr | (uintptr_t)out[1].ptr | (uintptr_t)bytes;
  const int64_t blocks = ((int64_t)p.batch * p.kv_heads * 2 + 3) / 4;
  C3B_REQUIRE(blocks < (1ll << 31), "kv commit: too many heads");
  if (at % 16 == 0) {
    a.units = (int)(bytes / 16);
    return launch_pdl(commit_kernel<uint4>, (int)blocks, 128, 0, s, a);
  }
  a.units = (int)(bytes / 2);
  return launch_pdl(commit_kernel<uint16_t>, (int)blocks, 128, 0, s, a);
}

}  // namespace c3b
