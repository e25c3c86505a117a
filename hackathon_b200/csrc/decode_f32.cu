// fp32 attention of drafted tokens over a decoding cache, on tensor cores.
//
// The same operator, split, masks and block layout as decode_mma.cu, with 8 keys
// a warp.  Products are tf32 (mma.sync m16n8k8) on operands split in two:
// x = hi + lo, each rounded to tf32's 11 bits, and
//   x y = hi hi' + hi lo' + lo hi'   (lo lo' is below 2^-22 of the product),
// each of the three with its own accumulators for the scores, which shortens
// the chains and adds the small terms to each other first.  Rounding to tf32 is
// an integer addition, a mask and a minimum.  Queries are split once a piece.  In plain FMA
// 16 rows would fill the FMA pipe for longer than HBM needs.
//
// In P V the k index runs over the keys in the order 0 2 4 6 1 3 5 7: a thread's
// score accumulators are then its weight operands as they stand, and the eight
// rows a warp reads of V fall on different banks.
#include <type_traits>

#include "common.cuh"
#include "decode.cuh"
#include "exp2.cuh"
#include "tc_prims.cuh"

namespace c3b {

namespace df32 {
using namespace tc;
using dec::Args;

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c += a, rounded to nearest.  A product's own addition to its accumulator cuts off, so sums over many
// units would drift towards 0: by 1.2e-5 over 20000 keys, where this leaves 5e-7, for 3 to 9 % of the time.
__device__ __forceinline__ void add4(float* c, const float* a) {
  const float2 x = __fadd2_rn(make_float2(c[0], c[1]), make_float2(a[0], a[1]));
  const float2 y = __fadd2_rn(make_float2(c[2], c[3]), make_float2(a[2], a[3]));
  c[0] = x.x, c[1] = x.y, c[2] = y.x, c[3] = y.y;
}

// ldmatrix and the products are not volatile, so that the compiler may overlap
// them; pinned registers keep them in their place: a stage's address is pinned
// after the wait for its data, the sums before its release.
__device__ __forceinline__ void pin(uint32_t& x) { asm volatile("" : "+r"(x) : : "memory"); }
__device__ __forceinline__ void pin(float& x) { asm volatile("" : "+f"(x) : : "memory"); }

// x = hi + lo for tf32 products, which ignore the low 13 bits: hi is x rounded to
// the 11 that count and held at the largest finite one, lo the rest, of which they
// see 11 more.  What is infinite or no number stands in lo alone.
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  const float r = __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
  float h;
  asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(h) : "f"(r), "f"(0x1.ffcp127f));
  hi = __float_as_uint(h);
  lo = __float_as_uint(x - h);
}
// `part`: hi for the products with another value's lo, 0 where x is infinite: beside
// an infinity of one sign they could overflow to the other.
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo, uint32_t& part) {
  split(x, hi, lo);
  part = fabsf(x) == INFINITY ? 0u : hi;
}

// Byte offset of 16-byte chunk `ch` (4 dims) of row `row` in a tile of 128-byte
// rows (32 dims) under the 128-byte swizzle; further dims follow in tiles of ROWS rows.
template <int ROWS>
__device__ __forceinline__ uint32_t at(int row, int ch) {
  return (uint32_t)((ch >> 3) * (ROWS * 128) + row * 128 + (((ch ^ row) & 7) << 4));
}

// DP: head_dim rounded up to 64, 128 or 256.  MT: 16-row tiles.  NW: consumer warps.
template <int DP, int MT, int NW>
struct Shape {
  static constexpr int ROWS = 16 * MT;
  static constexpr int CONSUMERS = NW;
  static constexpr int KEYS = 8 * NW;
  static constexpr int THREADS = 32 * (CONSUMERS + 1);
  static constexpr uint32_t TILE = KEYS * DP * 4;
  static constexpr int OSTRIDE = DP + 8;  // floats: fragment rows fall on different banks
  static constexpr uint32_t O_BYTES = (uint32_t)ROWS * OSTRIDE * 4;
  static constexpr uint32_t Q_BYTES = 2u * ROWS * DP * 4;  // hi, lo
  static constexpr uint32_t ML_BYTES = 2u * (NW + 1) * ROWS * 4;
  static constexpr uint32_t QO_BYTES = O_BYTES > Q_BYTES ? O_BYTES : Q_BYTES;  // the sums are joined where Q stood
  static constexpr uint32_t REST = QO_BYTES + ML_BYTES + 256;
  static constexpr uint32_t BUDGET = 226u * 1024;
  static constexpr int FIT = (int)((BUDGET - REST - 1024) / (2 * TILE));
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static_assert(STAGES >= 2, "a ring needs two stages");
  static constexpr uint32_t SMEM = STAGES * 2 * TILE + REST + 1024;
};

template <int DP, int MT, int NW>
__global__ void __launch_bounds__((Shape<DP, MT, NW>::THREADS), 1)
    tree_f32_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Args a) {
  typedef Shape<DP, MT, NW> S;
  constexpr int KEYS = S::KEYS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* q_sm = sm + S::STAGES * 2 * S::TILE;
  float* o_sm = reinterpret_cast<float*>(q_sm);
  float* m_sm = reinterpret_cast<float*>(q_sm + S::QO_BYTES);  // [NW][ROWS]
  float* l_sm = m_sm + NW * S::ROWS;     // [NW][ROWS]
  float2* row_sm = reinterpret_cast<float2*>(l_sm + NW * S::ROWS);  // [ROWS]
  uint64_t* full = reinterpret_cast<uint64_t*>(row_sm + S::ROWS);
  uint64_t* empty = full + S::STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + S::STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], S::CONSUMERS);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  dec::Walk w = dec::start<KEYS>(a, lane);

  if (warp == S::CONSUMERS) {
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
    const int kg = warp;
    const int g = lane >> 2, t = lane & 3;
    auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * S::CONSUMERS) : "memory"); };
    uint32_t it = 0;
    for (; w.left >= 0; dec::next<KEYS>(a, w)) {
      if (w.count == 0) continue;
      // ---- the piece's query rows: row r is token r / G, head r % G of the group
      const int r0 = w.rtile * S::ROWS;
      const float* q = static_cast<const float*>(a.q);
      constexpr int LOADS = S::ROWS * (DP / 4) / (32 * S::CONSUMERS);
      float4 qv[LOADS];  // all on their way before the first is stored
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = threadIdx.x + i * 32 * S::CONSUMERS, r = e / (DP / 4), ch = e % (DP / 4);
        qv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r0 + r < a.rows && ch * 4 < a.d)
          qv[i] = *reinterpret_cast<const float4*>(q + dec::row_offset(a, w.b, w.head, r0 + r) + ch * 4);
      }
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = threadIdx.x + i * 32 * S::CONSUMERS;
        const uint32_t to = at<S::ROWS>(e / (DP / 4), e % (DP / 4));
        uint4 hi, lo;
        split(qv[i].x, hi.x, lo.x), split(qv[i].y, hi.y, lo.y), split(qv[i].z, hi.z, lo.z), split(qv[i].w, hi.w, lo.w);
        *reinterpret_cast<uint4*>(q_sm + to) = hi;
        *reinterpret_cast<uint4*>(q_sm + S::ROWS * DP * 4 + to) = lo;
      }
      sync();
      uint32_t q_base = smem_u32(q_sm);
      pin(q_base);
      const int qrow = (lane & 7) + ((lane >> 3) & 1) * 8;
      float o[MT][DP / 8][4], m[MT][2], l[MT][2];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int nb = 0; nb < DP / 8; ++nb) o[i][nb][0] = o[i][nb][1] = o[i][nb][2] = o[i][nb][3] = 0.f;
        m[i][0] = m[i][1] = -INFINITY;
        l[i][0] = l[i][1] = 0.f;
      }

      for (int u = w.tile; u < w.tile + w.count; ++u, ++it) {
        const uint32_t st = it % S::STAGES;
        mbar_wait(&full[st], (it / S::STAGES) & 1, abort_flag, 44);  // on expiry every wait returns: all warps finish
        uint8_t* v_sm = sm + st * 2 * S::TILE + S::TILE;
        uint32_t k_base = smem_u32(sm + st * 2 * S::TILE);
        pin(k_base);
        // ---- S = Q K^T for the warp's 8 keys: hi hi', hi lo', lo hi'
        float s[MT][4], acc[MT][3][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int c = 0; c < 3; ++c) acc[i][c][0] = acc[i][c][1] = acc[i][c][2] = acc[i][c][3] = 0.f;
#pragma unroll 2
        for (int ks = 0; ks < DP / 8; ks += 2) {
          uint32_t b[4], bh[4], bl[4], bp[4];  // two steps of 8 dims
          ldsm4(k_base + at<KEYS>(kg * 8 + (lane & 7), 2 * ks + (lane >> 3)), b);
#pragma unroll
          for (int c = 0; c < 4; ++c) split(__uint_as_float(b[c]), bh[c], bl[c], bp[c]);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t fh[4], fl[4];
              const uint32_t q_at = q_base + at<S::ROWS>(qrow + 16 * i, 2 * (ks + h) + (lane >> 4));
              ldsm4(q_at, fh);
              ldsm4(q_at + S::ROWS * DP * 4, fl);
              mma(acc[i][0], fh, bh[2 * h], bh[2 * h + 1]);
              mma(acc[i][1], fh, bl[2 * h], bl[2 * h + 1]);
              mma(acc[i][2], fl, bp[2 * h], bp[2 * h + 1]);
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][j] = __fmul_rn(acc[i][0][j] + (acc[i][1][j] + acc[i][2][j]), a.scale_log2);
        // ---- mask
        const int key0 = u * KEYS + kg * 8;
        const bool open = key0 + 8 > w.n;  // the warp's keys reach past the committed rows
        bool poison = false;
        if (open) {
          const int row = r0 + (lane & (S::ROWS - 1));  // whose keys the lane looks up
          const uint32_t mine = dec::see<8>(a, w, row < a.rows ? dec::token_of(a, row) : 0, row < a.rows, key0, lane);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t bits = __shfl_sync(0xffffffffu, mine, 16 * i + 8 * half + g) >> (2 * t);
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (!(bits >> j & 1)) s[i][2 * half + j] = -INFINITY;
            }
          // rows behind the drafts become zero; drafts are looked at for infinities and NaN
          for (int e = lane; e < 8 * (DP / 4); e += 32) {
            const int r = e / (DP / 4), ch = e % (DP / 4);
            float4* p = reinterpret_cast<float4*>(v_sm + at<KEYS>(kg * 8 + r, ch));
            if (key0 + r >= w.end) {
              *p = make_float4(0.f, 0.f, 0.f, 0.f);
            } else if (key0 + r >= w.n) {
              const float4 v = *p;
              const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) poison = poison || !(fabsf(x[k]) < INFINITY);
            }
          }
          fence_proxy_async();  // these writes come before the next load into the stage
          __syncwarp();         // and before the other lanes read the unit
          poison = __any_sync(0xffffffffu, poison);
        }
        // ---- running maxima; m is the reference of dec::LAG and dec::lift
        bool grow = false;
        float top[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float x = fmaxf(s[i][2 * half], s[i][2 * half + 1]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            top[i][half] = x;
            grow = grow || x > m[i][half] + (dec::LAG + dec::lift(false));
          }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float mn = fmaxf(m[i][half], top[i][half] - dec::lift(false));
              const float f = mn == -INFINITY ? 1.f : exp2f(m[i][half] - mn);
              m[i][half] = mn;
              l[i][half] *= f;
#pragma unroll
              for (int nb = 0; nb < DP / 8; ++nb) {
                o[i][nb][2 * half] *= f;
                o[i][nb][2 * half + 1] *= f;
              }
            }
        }
        // ---- weights: key 2 t of rows g, g + 8 and key 2 t + 1, as k = t and k = t + 4
        uint32_t ph[MT][4], pl[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float base = m[i][half] == -INFINITY ? 0.f : m[i][half];
            float& x = s[i][2 * half];
            float& y = s[i][2 * half + 1];
            x = exp2f(x - base);
            y = exp2f(y - base);
            l[i][half] += x + y;
            split(x, ph[i][half], pl[i][half]);
            split(y, ph[i][2 + half], pl[i][2 + half]);
          }
        // ---- O += P V
        if (!poison) {
          const int r = kg * 8 + 2 * t;
#pragma unroll
          for (int nb = 0; nb < DP / 8; ++nb) {
            const int ch = 2 * nb + (g >> 2);
            uint32_t h0, l0, h1, l1;
            split(*reinterpret_cast<const float*>(v_sm + at<KEYS>(r, ch) + 4 * (g & 3)), h0, l0);
            split(*reinterpret_cast<const float*>(v_sm + at<KEYS>(r + 1, ch) + 4 * (g & 3)), h1, l1);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              float part[4] = {0.f, 0.f, 0.f, 0.f};
              mma(part, pl[i], h0, h1);
              mma(part, ph[i], l0, l1);
              mma(part, ph[i], h0, h1);
              add4(o[i][nb], part);
            }
          }
        } else {
#pragma unroll 1
          for (int key = 0; key < 8; ++key) {
            // the key's weights for rows g and g + 8, from the lane that has them
            float x[MT], y[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              x[i] = __shfl_sync(0xffffffffu, key & 1 ? s[i][1] : s[i][0], (g << 2) | (key >> 1));
              y[i] = __shfl_sync(0xffffffffu, key & 1 ? s[i][3] : s[i][2], (g << 2) | (key >> 1));
            }
#pragma unroll
            for (int nb = 0; nb < DP / 8; ++nb) {
              const float2 f = *reinterpret_cast<const float2*>(v_sm + at<KEYS>(kg * 8 + key, 2 * nb + (t >> 1)) + 8 * (t & 1));
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                if (x[i] != 0.f) o[i][nb][0] += x[i] * f.x, o[i][nb][1] += x[i] * f.y;
                if (y[i] != 0.f) o[i][nb][2] += y[i] * f.x, o[i][nb][3] += y[i] * f.y;
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int nb = 0; nb < DP / 8; ++nb)
#pragma unroll
            for (int j = 0; j < 4; ++j) pin(o[i][nb][j]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }

      // ---- join the key groups
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x = l[i][half];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          const int r = 16 * i + 8 * half + g;
          if (t == 0) m_sm[kg * S::ROWS + r] = m[i][half], l_sm[kg * S::ROWS + r] = x;
        }
      sync();
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = 16 * i + 8 * half + g;
          float mx = m_sm[r];
#pragma unroll
          for (int k = 1; k < NW; ++k) mx = fmaxf(mx, m_sm[k * S::ROWS + r]);
          const float f = mx == -INFINITY ? 1.f : exp2f(m[i][half] - mx);
#pragma unroll
          for (int nb = 0; nb < DP / 8; ++nb) o[i][nb][2 * half] *= f, o[i][nb][2 * half + 1] *= f;
        }
      // In round k warp kg adds part (kg + k) mod NW of the dims: always the same order, all warps at work.
      auto add = [&](auto me) {
        constexpr int KG = decltype(me)::value;
#pragma unroll
        for (int round = 0; round < NW; ++round) {
          const int c = (KG + round) % NW;
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int nb = c * (DP / 8 / NW); nb < (c + 1) * (DP / 8 / NW); ++nb) {
                float2* d = reinterpret_cast<float2*>(o_sm + (16 * i + 8 * half + g) * S::OSTRIDE + nb * 8 + 2 * t);
                float2 x = make_float2(o[i][nb][2 * half], o[i][nb][2 * half + 1]);
                if (round) {
                  const float2 y = *d;
                  x.x += y.x, x.y += y.y;
                }
                *d = x;
              }
          if (round == 0 && KG == 0 && lane < S::ROWS) {
            // the rows' maxima and sums over the groups
            float mx = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < NW; ++k) mx = fmaxf(mx, m_sm[k * S::ROWS + lane]);
#pragma unroll
            for (int k = 0; k < NW; ++k) {
              const float x = l_sm[k * S::ROWS + lane];
              sum += mx == -INFINITY ? x : exp2f(m_sm[k * S::ROWS + lane] - mx) * x;
            }
            row_sm[lane] = make_float2(mx, sum);
          }
          sync();
        }
      };
      switch (kg) {
        case 0: add(std::integral_constant<int, 0>()); break;
        case 1: add(std::integral_constant<int, 1>()); break;
        case 2: add(std::integral_constant<int, 2>()); break;
        case 3: add(std::integral_constant<int, 3>()); break;
        default:
          if constexpr (NW == 8) {
            if (kg == 4) add(std::integral_constant<int, 4>());
            else if (kg == 5) add(std::integral_constant<int, 5>());
            else if (kg == 6) add(std::integral_constant<int, 6>());
            else add(std::integral_constant<int, 7>());
          }
      }
      // ---- out, or to the block's workspace slot
      const bool whole = w.count == w.tiles;
      const int slot = dec::slot(w);
      for (int e = threadIdx.x; e < S::ROWS * (DP / 8); e += 32 * S::CONSUMERS) {
        const int r = e / (DP / 8), c = e % (DP / 8) * 8;
        if (r0 + r >= a.rows || c >= a.d) continue;
        const float2 ml = row_sm[r];
        const float* x0 = o_sm + r * S::OSTRIDE + c;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x0[i];
        if (whole) {
          const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;  // a row that sees nothing is zero
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= inv;
          float* dst = static_cast<float*>(a.out) + dec::row_offset(a, w.b, w.head, r0 + r) + c;
          *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
          if (c + 4 < a.d) *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
          float* dst = a.part + ((int64_t)slot * S::ROWS + r) * a.d + c;
          *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
          if (c + 4 < a.d) *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
          if (c == 0) a.part_ml[(int64_t)slot * S::ROWS + r] = ml;
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

template <int DP, int MT, int NW>
static int run(const CUtensorMap& km, const CUtensorMap& vm, const Args& a, int grid, cudaStream_t s) {
  typedef Shape<DP, MT, NW> S;
  auto kernel = tree_f32_kernel<DP, MT, NW>;
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_smem(kernel, (int)S::SMEM, done)) return rc;
  return launch_pdl(kernel, grid, S::THREADS, (size_t)S::SMEM, s, km, vm, a);
}

}  // namespace df32

namespace dec {

int f32_unit(int dp, int rows) { return dp == 64 || (dp == 128 && rows == 16) ? 64 : 32; }

int run_f32(const Plan& pl, const Args& a, cudaStream_t s) {
  CUtensorMap km, vm;
  if (int rc = cache_maps(a, f32_unit(pl.dp, pl.rows), &km, &vm)) return rc;
  if (pl.dp == 64)
    return pl.rows == 16 ? df32::run<64, 1, 8>(km, vm, a, pl.grid, s) : df32::run<64, 2, 8>(km, vm, a, pl.grid, s);
  if (pl.dp == 128)  // 32 rows: twice the accumulators, so half the warps
    return pl.rows == 16 ? df32::run<128, 1, 8>(km, vm, a, pl.grid, s) : df32::run<128, 2, 4>(km, vm, a, pl.grid, s);
  return df32::run<256, 1, 4>(km, vm, a, pl.grid, s);
}

}  // namespace dec
}  // namespace c3b
