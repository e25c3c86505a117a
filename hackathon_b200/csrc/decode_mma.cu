// Tensor-core attention of drafted tokens over a decoding cache, 16-bit types.
//
// o = softmax(q k^T scale + mask) v for T drafts a sequence.  All T * G query
// rows that share a key/value head (G = heads / kv_heads) stand in one tile, so
// each cached row is read once: 4 D bytes a cached row against 4 T G D
// operations, T G operations a byte.  With one 16-row tile HBM bounds it (85 us
// for 32 sequences of up to 7000 rows, floor 75), with two the products begin to
// (54 us for 16 sequences of up to 4000 rows and 8 heads of 128, floor 23); more
// rows would read the cache again for every 32.
//
// Split.  The work is cut into units of 64 cached rows of one (sequence, kv
// head, row tile) and the units, laid out in that order, are shared evenly over
// a grid that fills the GPU once: block c takes units [c W / C, (c + 1) W / C).
// Lengths live on the device, so each warp finds its block's place by a scan of
// `lengths`; ragged batches, one long sequence and many short ones all come out
// even.  A block's pieces that cover a whole segment are finished in place; the
// first and the last may be parts, which go to two workspace slots of the block
// and are joined by a second small kernel in block order (results do not depend
// on timing).  Caches of few units a segment are not cut: block c takes whole
// segments and nothing is joined.
//
// A block: four consumer warps and one producer.  The producer loads K and V
// units by TMA (128-byte swizzle; dims past head_dim arrive as zeros) into a
// ring of stages.  Consumer warp kg takes all 16 MT rows and keys 16 kg ..
// 16 kg + 15 of every unit, with its own running maximum and sum, so
// warps meet only at the end of a piece.  The maximum is raised lazily (by more
// than 2^8), which skips most rescales of the accumulators.
//
// Masks only touch units past the committed rows.  There, values of rows behind
// the drafts are zeroed in shared memory (whatever lies there), and a unit
// whose drafts hold infinities or NaN is multiplied element by element without
// the masked ones, since 0 times those is not 0.
#include <type_traits>

#include "common.cuh"
#include "decode.cuh"
#include "exp2.cuh"
#include "tc_prims.cuh"

namespace c3b {

namespace dmma {
using namespace tc;
using dec::Args;

constexpr int KEYS = 64;

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool H16>
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (H16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two values with infinities (and NaN) replaced by the type's largest.
template <bool H16>
__device__ __forceinline__ uint32_t finite(uint32_t v) {
  uint32_t r;
  if constexpr (H16)
    asm("min.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x7bff7bffu));
  else
    asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x7f7f7f7fu));
  return r;
}

// Byte offset of 16-byte chunk `ch` of row `row` in a tile of 128-byte rows
// (64 dims) under the 128-byte swizzle; further dims follow in tiles of ROWS rows.
template <int ROWS>
__device__ __forceinline__ uint32_t at(int row, int ch) {
  return (uint32_t)((ch >> 3) * (ROWS * 128) + row * 128 + (((ch ^ row) & 7) << 4));
}

// DP: head_dim rounded up to 64, 128 or 256.  MT: 16-row tiles.
template <int DP, int MT>
struct Shape {
  static constexpr int ROWS = 16 * MT;
  static constexpr int CONSUMERS = 4;
  static constexpr int THREADS = 32 * (CONSUMERS + 1);
  static constexpr uint32_t TILE = KEYS * DP * 2;
  static constexpr int OSTRIDE = DP + 8;  // floats: fragment rows fall on different banks
  static constexpr uint32_t O_BYTES = (uint32_t)ROWS * OSTRIDE * 4;
  static constexpr uint32_t Q_BYTES = (uint32_t)ROWS * DP * 2;
  static constexpr uint32_t ML_BYTES = 2u * 5 * ROWS * 4;
  static constexpr uint32_t QO_BYTES = O_BYTES > Q_BYTES ? O_BYTES : Q_BYTES;  // the sums are joined where Q stood
  static constexpr uint32_t REST = QO_BYTES + ML_BYTES + 256;
  // two blocks an SM where both fit with three stages
  static constexpr bool PAIR = 3 * 2 * TILE + REST + 1024 <= 113 * 1024;
  static constexpr uint32_t BUDGET = (PAIR ? 113u : 226u) * 1024;
  static constexpr int FIT = (int)((BUDGET - REST - 1024) / (2 * TILE));
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static_assert(STAGES >= 2, "a ring needs two stages");
  static constexpr uint32_t SMEM = STAGES * 2 * TILE + REST + 1024;
};

template <int DP, int MT, bool H16>
__global__ void __launch_bounds__((Shape<DP, MT>::THREADS), (Shape<DP, MT>::PAIR ? 2 : 1))
    tree_mma_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Args a) {
  typedef Shape<DP, MT> S;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* q_sm = sm + S::STAGES * 2 * S::TILE;
  float* o_sm = reinterpret_cast<float*>(q_sm);
  float* m_sm = reinterpret_cast<float*>(q_sm + S::QO_BYTES);  // [4][ROWS]
  float* l_sm = m_sm + 4 * S::ROWS;     // [4][ROWS]
  float2* row_sm = reinterpret_cast<float2*>(l_sm + 4 * S::ROWS);  // [ROWS]
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
          for (int c = 0; c < DP / 64; ++c) {
            tma_load_2d(k_sm + c * (KEYS * 128), &k_map, &full[st], c * 64, (int)(row0 + (int64_t)u * KEYS));
            tma_load_2d(k_sm + S::TILE + c * (KEYS * 128), &v_map, &full[st], c * 64, (int)(row0 + (int64_t)u * KEYS));
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
      const uint16_t* q = static_cast<const uint16_t*>(a.q);
      constexpr int LOADS = S::ROWS * (DP / 8) / (32 * S::CONSUMERS);
      uint4 qv[LOADS];  // all on their way before the first is stored
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = threadIdx.x + i * 32 * S::CONSUMERS, r = e / (DP / 8), ch = e % (DP / 8);
        qv[i] = make_uint4(0, 0, 0, 0);
        if (r0 + r < a.rows && ch * 8 < a.d)
          qv[i] = *reinterpret_cast<const uint4*>(q + dec::row_offset(a, w.b, w.head, r0 + r) + ch * 8);
      }
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = threadIdx.x + i * 32 * S::CONSUMERS;
        *reinterpret_cast<uint4*>(q_sm + at<S::ROWS>(e / (DP / 8), e % (DP / 8))) = qv[i];
      }
      sync();
      const uint32_t q_base = smem_u32(q_sm);
      const int qrow = (lane & 7) + ((lane >> 3) & 1) * 8;
      uint32_t qa[MT == 1 ? DP / 16 : 1][4];  // one row tile a warp: its fragments stay in registers
      if constexpr (MT == 1) {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) ldsm4(q_base + at<S::ROWS>(qrow, 2 * ks + (lane >> 4)), qa[ks]);
      }
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
        const uint32_t k_base = smem_u32(sm + st * 2 * S::TILE), v_base = k_base + S::TILE;
        // ---- S = Q K^T for the warp's rows and 16 keys
        float s[MT][2][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int nb = 0; nb < 2; ++nb) s[i][nb][0] = s[i][nb][1] = s[i][nb][2] = s[i][nb][3] = 0.f;
        const int krow = kg * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          uint32_t b[4];
          ldsm4(k_base + at<KEYS>(krow, 2 * ks + ((lane >> 3) & 1)), b);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            uint32_t f[4];
            if constexpr (MT == 1) {
              f[0] = qa[ks][0], f[1] = qa[ks][1], f[2] = qa[ks][2], f[3] = qa[ks][3];
            } else {
              ldsm4(q_base + at<S::ROWS>(qrow + 16 * i, 2 * ks + (lane >> 4)), f);
            }
            mma<H16>(s[i][0], f, b[0], b[1]);
            mma<H16>(s[i][1], f, b[2], b[3]);
          }
        }
        // ---- scale, mask
        const int key0 = u * KEYS + kg * 16;
        const bool open = key0 + 16 > w.n;  // the warp's keys reach past the committed rows
        bool poison = false;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][nb][j] = __fmul_rn(s[i][nb][j], a.scale_log2);  // rounded for all its uses
        if (open) {
          const int row = r0 + (lane & (S::ROWS - 1));  // whose keys the lane looks up
          const uint32_t mine = dec::see<16>(a, w, row < a.rows ? dec::token_of(a, row) : 0, row < a.rows, key0, lane);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t bits = __shfl_sync(0xffffffffu, mine, 16 * i + 8 * half + g) >> (2 * t);
#pragma unroll
              for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                  if (!(bits >> (8 * nb + j) & 1)) s[i][nb][2 * half + j] = -INFINITY;
            }
          // rows behind the drafts become zero; drafts are looked at for infinities and NaN
          const uint32_t inf = H16 ? 0x7c00u : 0x7f80u;
          for (int e = lane; e < 16 * (DP / 8); e += 32) {
            const int r = e / (DP / 8), ch = e % (DP / 8);
            uint4* p = reinterpret_cast<uint4*>(sm + st * 2 * S::TILE + S::TILE + at<KEYS>(kg * 16 + r, ch));
            if (key0 + r >= w.end) {
              *p = make_uint4(0, 0, 0, 0);
            } else if (key0 + r >= w.n) {
              const uint4 v = *p;
              const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int k = 0; k < 4; ++k)
                poison = poison || (x[k] & inf) == inf || ((x[k] >> 16) & inf) == inf;
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
            float x = fmaxf(fmaxf(s[i][0][2 * half], s[i][0][2 * half + 1]), fmaxf(s[i][1][2 * half], s[i][1][2 * half + 1]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            top[i][half] = x;
            grow = grow || x - m[i][half] > dec::LAG + dec::lift(H16);  // the sum of the two would be rounded above 2^24
          }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float mn = fmaxf(m[i][half], top[i][half] - dec::lift(H16));
              const float f = mn == -INFINITY ? 1.f : exp2_sfu(m[i][half] - mn);
              m[i][half] = mn;
              l[i][half] *= f;
#pragma unroll
              for (int nb = 0; nb < DP / 8; ++nb) {
                o[i][nb][2 * half] *= f;
                o[i][nb][2 * half + 1] *= f;
              }
            }
        }
        // ---- weights
        // With up to 16 rows HBM leaves time to multiply what the type leaves of a weight as well, so the weights'
        // rounding adds nothing to the output's (82.9 -> 84.1 us for 32 sequences of up to 7000); with 32 rows it
        // does not (107 -> 121 us), and the two roundings add up to 1.4 times the output's (2-norm, fp16: 2.9e-4
        // against 2.1e-4).
        uint32_t p[MT][4], rest[4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float base = m[i][half] == -INFINITY ? 0.f : m[i][half];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
              float& x = s[i][nb][2 * half];
              float& y = s[i][nb][2 * half + 1];
              x = exp2_sfu(x - base);
              y = exp2_sfu(y - base);
              l[i][half] += x + y;
              p[i][2 * nb + half] = pack2h(make_float2(x, y), H16);
              if constexpr (MT == 1) {
                const float2 z = unpack2h(p[i][2 * nb + half], H16);
                rest[2 * nb + half] = pack2h(make_float2(x - z.x, y - z.y), H16);
              }
            }
          }
        // ---- O += P V
        if (!poison) {
          const int vrow = kg * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
          for (int nb = 0; nb < DP / 8; nb += 2) {
            uint32_t b[4];
            ldsm4_t(v_base + at<KEYS>(vrow, nb + (lane >> 4)), b);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              mma<H16>(o[i][nb], p[i], b[0], b[1]);
              mma<H16>(o[i][nb + 1], p[i], b[2], b[3]);
              if constexpr (MT == 1) {
                // a rest may be 0 or negative: what is infinite is left to the weight itself
                mma<H16>(o[i][nb], rest, finite<H16>(b[0]), finite<H16>(b[1]));
                mma<H16>(o[i][nb + 1], rest, finite<H16>(b[2]), finite<H16>(b[3]));
              }
            }
          }
        } else {
#pragma unroll 1
          for (int key = 0; key < 16; ++key) {
            // the key's weights for rows g and g + 8, from the lane that has them
            float x[MT], y[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const float* lo = s[i][0];
              const float* hi = s[i][1];
              const float u = key & 8 ? (key & 1 ? hi[1] : hi[0]) : (key & 1 ? lo[1] : lo[0]);
              const float v = key & 8 ? (key & 1 ? hi[3] : hi[2]) : (key & 1 ? lo[3] : lo[2]);
              x[i] = __shfl_sync(0xffffffffu, u, (g << 2) | ((key >> 1) & 3));
              y[i] = __shfl_sync(0xffffffffu, v, (g << 2) | ((key >> 1) & 3));
            }
            const uint8_t* row = sm + st * 2 * S::TILE + S::TILE;
#pragma unroll
            for (int c = 0; c < DP / 8; ++c) {
              const float2 f = unpack2h(*reinterpret_cast<const uint32_t*>(row + at<KEYS>(kg * 16 + key, c) + 4 * t), H16);
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                if (x[i] != 0.f) o[i][c][0] += x[i] * f.x, o[i][c][1] += x[i] * f.y;
                if (y[i] != 0.f) o[i][c][2] += y[i] * f.x, o[i][c][3] += y[i] * f.y;
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }

      // ---- join the four key groups
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
          const float mx = fmaxf(fmaxf(m_sm[r], m_sm[S::ROWS + r]), fmaxf(m_sm[2 * S::ROWS + r], m_sm[3 * S::ROWS + r]));
          const float f = mx == -INFINITY ? 1.f : exp2_sfu(m[i][half] - mx);
#pragma unroll
          for (int nb = 0; nb < DP / 8; ++nb) o[i][nb][2 * half] *= f, o[i][nb][2 * half + 1] *= f;
        }
      // In round k warp kg adds a quarter of the dims, quarter (kg + k) mod 4: always the same order, all warps at work.
      auto add = [&](auto me) {
        constexpr int KG = decltype(me)::value;
#pragma unroll
        for (int round = 0; round < 4; ++round) {
          const int c = (KG + round) & 3;
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int nb = c * (DP / 32); nb < (c + 1) * (DP / 32); ++nb) {
                float2* d = reinterpret_cast<float2*>(o_sm + (16 * i + 8 * half + g) * S::OSTRIDE + nb * 8 + 2 * t);
                float2 x = make_float2(o[i][nb][2 * half], o[i][nb][2 * half + 1]);
                if (round) {
                  const float2 y = *d;
                  x.x += y.x, x.y += y.y;
                }
                *d = x;
              }
          if (round == 0 && KG == 0 && lane < S::ROWS) {
            // the rows' maxima and sums over the four groups
            float mx = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) mx = fmaxf(mx, m_sm[k * S::ROWS + lane]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float x = l_sm[k * S::ROWS + lane];
              sum += mx == -INFINITY ? x : exp2_sfu(m_sm[k * S::ROWS + lane] - mx) * x;
            }
            row_sm[lane] = make_float2(mx, sum);
          }
          sync();
        }
      };
      if (kg == 0) add(std::integral_constant<int, 0>());
      else if (kg == 1) add(std::integral_constant<int, 1>());
      else if (kg == 2) add(std::integral_constant<int, 2>());
      else add(std::integral_constant<int, 3>());
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
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + dec::row_offset(a, w.b, w.head, r0 + r) + c) = pack8h(x, H16);
        } else {
          float* dst = a.part + ((int64_t)slot * S::ROWS + r) * a.d + c;
          *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
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

template <int DP, int MT, bool H16>
static int run(const CUtensorMap& km, const CUtensorMap& vm, const Args& a, int grid, cudaStream_t s) {
  typedef Shape<DP, MT> S;
  auto kernel = tree_mma_kernel<DP, MT, H16>;
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_smem(kernel, (int)S::SMEM, done)) return rc;
  return launch_pdl(kernel, grid, S::THREADS, (size_t)S::SMEM, s, km, vm, a);
}

template <int DP>
static int run_rows(int rows, bool h16, const CUtensorMap& km, const CUtensorMap& vm, const Args& a, int grid,
                    cudaStream_t s) {
  if constexpr (DP < 256) {
    if (rows == 32) return h16 ? run<DP, 2, true>(km, vm, a, grid, s) : run<DP, 2, false>(km, vm, a, grid, s);
  }
  return h16 ? run<DP, 1, true>(km, vm, a, grid, s) : run<DP, 1, false>(km, vm, a, grid, s);
}

}  // namespace dmma

namespace dec {

int mma_blocks_per_sm(int dp, int rows) {
  if (dp == 256) return 1;
  if (dp == 128) return (rows == 16 ? dmma::Shape<128, 1>::PAIR : dmma::Shape<128, 2>::PAIR) ? 2 : 1;
  return (rows == 16 ? dmma::Shape<64, 1>::PAIR : dmma::Shape<64, 2>::PAIR) ? 2 : 1;
}

int cache_maps(const Args& a, int box_rows, CUtensorMap* k, CUtensorMap* v) {
  const uint64_t dims[2] = {(uint64_t)a.d, (uint64_t)a.batch * a.kv_heads * a.capacity};
  const bool f32 = a.dtype == C3B_F32;
  const uint64_t str[1] = {(uint64_t)a.d * (f32 ? 4 : 2)};
  const uint32_t box[2] = {f32 ? 32u : 64u, (uint32_t)box_rows};
  const CUtensorMapDataType dt = f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (int rc = encode(k, const_cast<void*>(a.k), 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B, dt)) return rc;
  return encode(v, const_cast<void*>(a.v), 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B, dt);
}

int run_mma(bool h16, const Plan& pl, const Args& a, cudaStream_t s) {
  CUtensorMap km, vm;
  if (int rc = cache_maps(a, dmma::KEYS, &km, &vm)) return rc;
  switch (pl.dp) {
    case 64: return dmma::run_rows<64>(pl.rows, h16, km, vm, a, pl.grid, s);
    case 128: return dmma::run_rows<128>(pl.rows, h16, km, vm, a, pl.grid, s);
    default: return dmma::run_rows<256>(pl.rows, h16, km, vm, a, pl.grid, s);
  }
}

}  // namespace dec
}  // namespace c3b
