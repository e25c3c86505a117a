// fp32 attention of few query rows over a decoding cache.
//
// The operator, split and block layout of decode_f32.cu for up to 8 rows of a
// kv head, in packed fp32 pairs: with so few rows a product costs less in plain
// multiply-adds (rows / 2 a cached value) than splitting the value for tf32
// does: 44 us against 56 at 1 row of 64 dims (16 sequences of 500 to 4000 rows, 8
// heads), 36 against 38 at 8 rows of 64, 52 against 60 at 8 rows of 128, 63 against
// 71 at 8 rows of 256 (8 sequences).  More rows do not fit a lane's registers.
//
// A consumer warp takes KPW keys of a unit, as many at a time as fit:
//   scores   LK lanes share a key, each with 16-byte pieces LK apart and the
//            rows' queries for them in registers.  The lanes' partial sums are
//            added by a butterfly that halves the rows a lane carries at each
//            step, so a lane ends up with the score of one row and key.
//   softmax  on those single values; the weights go through shared memory, each
//            twice, side by side.
//   sums     a lane has four dims (two at head_dim 64 per half warp, which take
//            alternate keys) of every row.
// Weights of zero are skipped in the units that reach past the committed rows,
// so nothing that a row does not see reaches it.
#include "common.cuh"
#include "decode.cuh"
#include "tc_prims.cuh"

namespace c3b {

namespace dsimt {
using namespace tc;
using dec::Args;

constexpr int NW = 8;

// Byte offset of 16-byte chunk `ch` (4 dims) of row `row`: 128-byte rows (32
// dims) under the 128-byte swizzle, further dims in tiles of ROWS rows.
template <int ROWS>
__device__ __forceinline__ uint32_t at(int row, int ch) {
  return (uint32_t)((ch >> 3) * (ROWS * 128) + row * 128 + (((ch ^ row) & 7) << 4));
}

// DP: head_dim rounded up to 64, 128 or 256.  RW: rows, 4 or 8.
template <int DP, int RW>
struct Shape {
  static constexpr int KPW = DP == 256 ? 4 : 8;    // keys of a warp in a unit
  static constexpr int KEYS = KPW * NW;
  static constexpr int PIECES = RW == 4 ? 4 : 2;   // 16-byte pieces of a key a lane takes
  static constexpr int LK = DP / (4 * PIECES);     // lanes a key
  static constexpr int KPP = 32 / LK;              // keys at a time
  static constexpr int PASSES = KPW / KPP;
  static constexpr int THREADS = 32 * (NW + 1);
  static constexpr uint32_t TILE = KEYS * DP * 4;
  static constexpr uint32_t O_BYTES = NW * RW * DP * 4;
  static constexpr uint32_t P_BYTES = NW * KPW * RW * 8;
  static constexpr uint32_t REST = O_BYTES + P_BYTES + (NW + 1) * RW * 8 + 256;
  static constexpr int FIT = (int)((226 * 1024 - REST - 1024) / (2 * TILE));
  static constexpr int STAGES = FIT > 6 ? 6 : FIT;
  static_assert(STAGES >= 2, "a ring needs two stages");
  static_assert(KPW % KPP == 0, "whole passes");
  static constexpr uint32_t SMEM = STAGES * 2 * TILE + REST + 1024;
};

template <int DP, int RW>
__global__ void __launch_bounds__((Shape<DP, RW>::THREADS), 1)
    tree_simt_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Args a) {
  typedef Shape<DP, RW> S;
  constexpr int KEYS = S::KEYS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* o_sm = reinterpret_cast<float*>(sm + S::STAGES * 2 * S::TILE);  // [NW][RW][DP]
  float2* p_sm = reinterpret_cast<float2*>(o_sm + S::O_BYTES / 4);      // [NW][KPW][RW]: a weight, twice
  float2* ml_sm = p_sm + S::P_BYTES / 8;                                // [NW][RW]: maximum and sum
  float2* row_sm = ml_sm + NW * RW;                                     // [RW]
  uint64_t* full = reinterpret_cast<uint64_t*>(row_sm + RW);
  uint64_t* empty = full + S::STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + S::STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], NW);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  dec::Walk w = dec::start<KEYS>(a, lane);

  if (warp == NW) {
    if (lane == 0) {
      uint32_t it = 0;
      for (; w.left >= 0; dec::next<KEYS>(a, w)) {
        if (w.count == 0) continue;
        const int64_t row0 = ((int64_t)w.b * a.kv_heads + w.head) * a.capacity;
        for (int u = w.tile; u < w.tile + w.count; ++u, ++it) {
          const uint32_t st = it % S::STAGES;
          if (!mbar_wait(&empty[st], ((it / S::STAGES) & 1) ^ 1, abort_flag, 43)) goto produced;
          uint8_t* k_sm = sm + st * 2 * S::TILE;
          mbar_arrive_tx(&full[st], 2 * S::TILE);
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            tma_load_2d(k_sm + c * (KEYS * 128), &k_map, &full[st], c * 32, (int)(row0 + (int64_t)u * KEYS));
            tma_load_2d(k_sm + S::TILE + c * (KEYS * 128), &v_map, &full[st], c * 32, (int)(row0 + (int64_t)u * KEYS));
          }
        }
      }
    produced:;
    }
  } else {
    auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * NW) : "memory"); };
    const int lk = lane % S::LK;
    // the lane's key in a pass; at four lanes a key, neighbours four keys apart, whose pieces fall on other banks
    const int kk = S::LK == 4 ? ((lane >> 2) & 1) * 4 + (lane >> 3) : lane / S::LK;
    // the row whose scores the lane ends up with: the butterfly's choices, highest bit first
    const int row = S::LK == 4 || RW == 8 ? (RW == 8 ? lk / (S::LK / 8) : lk) : lk / (S::LK / 4);
    constexpr bool HALVES = DP == 64;  // half warps take alternate keys in P V
    const int dim = HALVES ? (lane & 15) * 4 : lane * 4;  // and + 128 at head_dim 256
    constexpr int DG = DP == 256 ? 2 : 1;
    float2* p_mine = p_sm + warp * (S::KPW * RW);
    uint32_t it = 0;
    for (; w.left >= 0; dec::next<KEYS>(a, w)) {
      if (w.count == 0) continue;
      // ---- the rows' queries at the lane's pieces
      const float* q = static_cast<const float*>(a.q);
      float4 qv[RW][S::PIECES];
#pragma unroll
      for (int r = 0; r < RW; ++r)
#pragma unroll
        for (int i = 0; i < S::PIECES; ++i) {
          const int c = (i * S::LK + lk) * 4;
          qv[r][i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < a.rows && c < a.d) qv[r][i] = *reinterpret_cast<const float4*>(q + dec::row_offset(a, w.b, w.head, r) + c);
        }
      const int tok = row < a.rows ? dec::token_of(a, row) : 0;
      float2 o[RW][DG][2];
#pragma unroll
      for (int r = 0; r < RW; ++r)
#pragma unroll
        for (int g = 0; g < DG; ++g) o[r][g][0] = o[r][g][1] = make_float2(0.f, 0.f);
      float m = -INFINITY, l = 0.f;  // of the lane's row; l over the lane's keys

      for (int u = w.tile; u < w.tile + w.count; ++u, ++it) {
        const uint32_t st = it % S::STAGES;
        mbar_wait(&full[st], (it / S::STAGES) & 1, abort_flag, 44);  // on expiry every wait returns: all warps finish
        const uint8_t* k_sm = sm + st * 2 * S::TILE;
        const uint8_t* v_sm = k_sm + S::TILE;
        // ---- scores
        float s[S::PASSES];
#pragma unroll
        for (int pass = 0; pass < S::PASSES; ++pass) {
          float2 acc[RW];
#pragma unroll
          for (int r = 0; r < RW; ++r) acc[r] = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < S::PIECES; ++i) {
            const float4 k = *reinterpret_cast<const float4*>(
                k_sm + at<KEYS>(warp * S::KPW + pass * S::KPP + kk, i * S::LK + lk));
#pragma unroll
            for (int r = 0; r < RW; ++r) {
              acc[r] = __ffma2_rn(make_float2(k.x, k.y), make_float2(qv[r][i].x, qv[r][i].y), acc[r]);
              acc[r] = __ffma2_rn(make_float2(k.z, k.w), make_float2(qv[r][i].z, qv[r][i].w), acc[r]);
            }
          }
          float x[RW];
#pragma unroll
          for (int r = 0; r < RW; ++r) x[r] = acc[r].x + acc[r].y;
          // halve the rows while lanes and rows last, then add what lanes are left
          int rows = RW;
#pragma unroll
          for (int half = S::LK / 2; half > 0; half >>= 1) {
            if (rows > 1) {
              rows >>= 1;
              const bool high = (lk & half) != 0;
#pragma unroll
              for (int r = 0; r < RW / 2; ++r)
                if (r < rows) {
                  const float keep = high ? x[r + rows] : x[r], give = high ? x[r] : x[r + rows];
                  x[r] = keep + __shfl_xor_sync(0xffffffffu, give, half);
                }
            } else {
              x[0] += __shfl_xor_sync(0xffffffffu, x[0], half);
            }
          }
          s[pass] = __fmul_rn(x[0], a.scale_log2);
        }
        const int key0 = u * KEYS + warp * S::KPW;
        const bool open = key0 + S::KPW > w.n;  // the warp's keys reach past the committed rows
        if (open) {
#pragma unroll
          for (int pass = 0; pass < S::PASSES; ++pass)
            if (!dec::visible(a, w, tok, key0 + pass * S::KPP + kk)) s[pass] = -INFINITY;
        }
        // ---- the row's running maximum, raised lazily; all lanes of a row agree; m is the reference of dec::LAG, dec::lift
        float top = s[0];
#pragma unroll
        for (int pass = 1; pass < S::PASSES; ++pass) top = fmaxf(top, s[pass]);
#pragma unroll
        for (int x = S::LK; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        if (__any_sync(0xffffffffu, top > m + (dec::LAG + dec::lift(false)))) {
          const float mn = fmaxf(m, top - dec::lift(false)), f = mn == -INFINITY ? 1.f : exp2f(m - mn);
          m = mn;
          l *= f;
#pragma unroll
          for (int r = 0; r < RW; ++r) {
            // a lane that has row r
            const int from = S::LK == 4 ? r : r * (S::LK / RW);
            const float fr = __shfl_sync(0xffffffffu, f, from);
#pragma unroll
            for (int g = 0; g < DG; ++g)
#pragma unroll
              for (int j = 0; j < 2; ++j) o[r][g][j] = __fmul2_rn(o[r][g][j], make_float2(fr, fr));
          }
        }
        // ---- weights
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int pass = 0; pass < S::PASSES; ++pass) {
          const float p = exp2f(s[pass] - base);
          // lanes that share a row and key have the same score; one of them counts it
          if (S::LK <= RW || lk % (S::LK / RW) == 0) {
            l += p;
            p_mine[(pass * S::KPP + kk) * RW + row] = make_float2(p, p);
          }
        }
        __syncwarp();
        // ---- sums
#pragma unroll
        for (int k = 0; k < S::KPW; k += HALVES ? 2 : 1) {
          const int key = HALVES ? k + (lane >> 4) : k;
          float2 p[RW];
#pragma unroll
          for (int r = 0; r < RW; r += 2) {
            const float4 x = *reinterpret_cast<const float4*>(p_mine + key * RW + r);
            p[r] = make_float2(x.x, x.y);
            p[r + 1] = make_float2(x.z, x.w);
          }
#pragma unroll
          for (int g = 0; g < DG; ++g) {
            const float4 v = *reinterpret_cast<const float4*>(v_sm + at<KEYS>(warp * S::KPW + key, dim / 4 + 32 * g));
#pragma unroll
            for (int r = 0; r < RW; ++r)
              if (!open || p[r].x != 0.f) {
                o[r][g][0] = __ffma2_rn(p[r], make_float2(v.x, v.y), o[r][g][0]);
                o[r][g][1] = __ffma2_rn(p[r], make_float2(v.z, v.w), o[r][g][1]);
              }
          }
        }
        __syncwarp();  // the weights have been read, the unit too
        if (lane == 0) mbar_arrive(&empty[st]);
      }

      // ---- join the warps
#pragma unroll
      for (int x = S::LK; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
      if (lane < S::LK && (S::LK <= RW || lk % (S::LK / RW) == 0)) ml_sm[warp * RW + row] = make_float2(m, l);
      if constexpr (HALVES) {
#pragma unroll
        for (int r = 0; r < RW; ++r)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            o[r][0][j].x += __shfl_xor_sync(0xffffffffu, o[r][0][j].x, 16);
            o[r][0][j].y += __shfl_xor_sync(0xffffffffu, o[r][0][j].y, 16);
          }
      }
      if (!HALVES || lane < 16) {
#pragma unroll
        for (int r = 0; r < RW; ++r)
#pragma unroll
          for (int g = 0; g < DG; ++g)
            *reinterpret_cast<float4*>(o_sm + (warp * RW + r) * DP + dim + 128 * g) =
                make_float4(o[r][g][0].x, o[r][g][0].y, o[r][g][1].x, o[r][g][1].y);
      }
      sync();
      // ---- out, or to the block's workspace slot
      const bool whole = w.count == w.tiles;
      const int slot = dec::slot(w);
      for (int e = threadIdx.x; e < RW * (DP / 4); e += 32 * NW) {
        const int r = e / (DP / 4), c = e % (DP / 4) * 4;
        if (r >= a.rows || c >= a.d) continue;
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < NW; ++k) mx = fmaxf(mx, ml_sm[k * RW + r].x);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < NW; ++k) {
          const float2 ml = ml_sm[k * RW + r];
          const float f = mx == -INFINITY ? 1.f : exp2f(ml.x - mx);
          const float4 y = *reinterpret_cast<const float4*>(o_sm + (k * RW + r) * DP + c);
          sum += f * ml.y;
          x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
        }
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing is zero
          *reinterpret_cast<float4*>(static_cast<float*>(a.out) + dec::row_offset(a, w.b, w.head, r) + c) =
              make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        } else {
          *reinterpret_cast<float4*>(a.part + ((int64_t)slot * RW + r) * a.d + c) = x;
          if (c == 0) a.part_ml[(int64_t)slot * RW + r] = make_float2(mx, sum);
        }
      }
      if (threadIdx.x == 0) dec::note_segment(a, w);
      sync();
    }
  }
  __syncthreads();
  if (*abort_flag) {  // loads still in flight land before the block's shared memory is given back
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
}

template <int DP, int RW>
static int run(const CUtensorMap& km, const CUtensorMap& vm, const Args& a, int grid, cudaStream_t s) {
  typedef Shape<DP, RW> S;
  auto kernel = tree_simt_kernel<DP, RW>;
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_smem(kernel, (int)S::SMEM, done)) return rc;
  return launch_pdl(kernel, grid, S::THREADS, (size_t)S::SMEM, s, km, vm, a);
}

}  // namespace dsimt

namespace dec {

int simt_unit(int dp) { return dp == 256 ? dsimt::Shape<256, 4>::KEYS : dsimt::Shape<128, 4>::KEYS; }

int run_simt(const Plan& pl, const Args& a, cudaStream_t s) {
  CUtensorMap km, vm;
  if (int rc = cache_maps(a, simt_unit(pl.dp), &km, &vm)) return rc;
  if (pl.dp == 64) return pl.rows == 4 ? dsimt::run<64, 4>(km, vm, a, pl.grid, s) : dsimt::run<64, 8>(km, vm, a, pl.grid, s);
  if (pl.dp == 128) return pl.rows == 4 ? dsimt::run<128, 4>(km, vm, a, pl.grid, s) : dsimt::run<128, 8>(km, vm, a, pl.grid, s);
  return pl.rows == 4 ? dsimt::run<256, 4>(km, vm, a, pl.grid, s) : dsimt::run<256, 8>(km, vm, a, pl.grid, s);
}

}  // namespace dec
}  // namespace c3b
