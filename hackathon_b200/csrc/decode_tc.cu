// tcgen05 attention of drafted tokens over a decoding cache, 16-bit types,
// head_dim up to 128: the calls with many query rows for each key/value head.
//
// Same operator, split and masks as decode_mma.cu; a unit is 128 cached rows.
// One block an SM, two softmax groups of 128 threads (one query row each):
//   rows of a kv head <= 128   one row tile: group i takes units of parity i and
//                              the two halves of the softmax are joined at the
//                              end of a piece;
//   more                       two row tiles (256 rows): group i has tile i, both
//                              read the same units.
// Group i has S (128 columns, overwritten by P as it is read) and O (up to 128
// columns) in TMEM, 512 columns in all.  Warp 8 loads K and V units by TMA into
// one ring of slots; one thread of warp 9 issues every product: S = Q K^T
// (M = 128, N = 128) and O += P V (P from TMEM, V as an MN-major operand).
// Products execute in issue order: S of the next unit follows the P V that
// reads the P standing in the same columns, and a group that sees its S knows
// its O complete, so it may rescale O (lazily: when a maximum grows by more
// than 2^8) without another barrier.  While one group computes its softmax the
// tensor core works for the other.  Half of the exponentials run on the FMA
// pipe (polynomial), half on the SFU.
//
// Weights are rounded to the type, since P is an operand of it: multiplying what
// that leaves as well would double P V, which with S is what the kernel waits
// for.  The roundings of weights and output add up to 1.4 times the output's own
// (2-norm, bf16: 2.3e-3 against 1.7e-3).  The polynomial of degree 3 is off by
// 7.5e-5, a seventh of half a step in fp16, a fiftieth in bf16.  Sums in TMEM are
// cut off, not rounded, at each product: 1.8e-4 of a sum of 100000 equal weights,
// less than half a step of fp16 (4.9e-4); shorter pieces lose in proportion.
//
// Values behind the drafts are zeroed in shared memory before they are
// multiplied; so are drafts' values that hold infinities or NaN, and those are
// then added row by row where the mask lets them through.  Where both groups
// read the same unit, group 0 alone does that: the issuing thread waits for
// group 0's weights of a unit before it goes on to group 1's, so group 1's
// product finds the unit cleared as well.
#include <type_traits>

#include "common.cuh"
#include "decode.cuh"
#include "exp2.cuh"
#include "tc_prims.cuh"

namespace c3b {

namespace dtc {
using namespace tc;
using dec::Args;

constexpr int KEYS = 128;
constexpr int ROWS = 128;      // rows of a softmax group
constexpr int THREADS = 320;   // two softmax groups, loader, MMA
constexpr uint32_t COL_S = 0, COL_O = 256;

template <int DP>
struct Shape {
  static constexpr uint32_t TILE = KEYS * DP * 2;          // K or V unit, and a Q tile
  static constexpr uint32_t ATOM = KEYS * 128;             // 64 dims of it
  static constexpr int SLOTS = DP == 128 ? 5 : 10;
  static constexpr uint32_t OFF_RING = 2 * TILE;
  static constexpr uint32_t OFF_META = OFF_RING + SLOTS * TILE;
  static constexpr uint32_t META = 1024 + 512;             // row statistics of group 1, barriers
  static constexpr uint32_t SMEM = OFF_META + META + 1024;
  static_assert(SMEM <= 227 * 1024, "a block's shared memory");
};

// Byte offset of 16-byte chunk `ch` of row `row`: 128-byte rows, 128-byte swizzle, 64 dims a tile.
__device__ __forceinline__ uint32_t at(int row, int ch) {
  return (uint32_t)((ch >> 3) * (KEYS * 128) + row * 128 + (((ch ^ row) & 7) << 4));
}

__device__ __forceinline__ void ld32(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// Waits for the loads; the values take part, so no use moves before it.
__device__ __forceinline__ void ld_wait32(float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// D (+)= A B, A (128 rows x 16, packed pairs) in TMEM, B in shared memory.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accum));
}

// One lane of a warp that runs together.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// NaN-propagating three-input maximum.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ bool non_finite(const uint4& v, uint32_t inf) {
  bool x = false;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) x = x || (w[k] & inf) == inf || ((w[k] >> 16) & inf) == inf;
  return x;
}

template <int DP, bool H16>
__global__ void __launch_bounds__(THREADS, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Args a) {
  typedef Shape<DP> S;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ring = sm + S::OFF_RING;
  float2* ml_sm = reinterpret_cast<float2*>(sm + S::OFF_META);  // [128]: group 1's maxima and sums
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + S::OFF_META + 1024);
  uint64_t* empty = full + S::SLOTS;
  uint64_t* q_full = empty + S::SLOTS;  // a piece's queries stand in shared memory
  uint64_t* s_full = q_full + 1;        // [2]
  uint64_t* p_full = s_full + 2;        // [2]
  uint64_t* o_full = p_full + 2;        // [2]: a piece's last product of the group
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* poison_flag = abort_flag + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool two = a.rows > ROWS;  // two row tiles
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    *abort_flag = 0;
    *poison_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp >= 8) {
    dec::Walk w = dec::start<KEYS>(a, lane);
    if (warp == 8) {
      // ------------------------------------------------ loads: K, V, K, V, ... of the block's units
      if (lane == 0) {
        uint32_t it = 0;
        for (; w.left >= 0; dec::next<KEYS>(a, w)) {
          if (w.count == 0) continue;
          const int64_t row0 = ((int64_t)w.b * a.kv_heads + w.head) * a.capacity;
          for (int u = w.tile; u < w.tile + w.count; ++u) {
#pragma unroll
            for (int which = 0; which < 2; ++which, ++it) {
              const uint32_t st = it % S::SLOTS;
              if (!mbar_wait(&empty[st], ((it / S::SLOTS) & 1) ^ 1, abort_flag, 45)) goto loaded;
              mbar_arrive_tx(&full[st], S::TILE);
#pragma unroll
              for (int c = 0; c < DP / 64; ++c)
                tma_load_2d(ring + st * S::TILE + c * S::ATOM, which ? &v_map : &k_map, &full[st], c * 64,
                            (int)(row0 + (int64_t)u * KEYS));
            }
          }
        }
      loaded:;
      }
    } else if (warp == 9) {
      // ------------------------------------------------ products: the warp walks together, one thread issues
      {
        const bool one = elect_one();
        const uint32_t id_s = instr_desc_h(ROWS, KEYS, H16);
        const uint32_t id_pv = instr_desc_h(ROWS, DP, H16) | (1u << 16);  // B (V) is MN-major
        const uint64_t q_desc = smem_desc(smem_u32(sm)), r_desc = smem_desc(smem_u32(ring));
        // V's second 64 dims lie one atom further (leading offset), its key groups 1024 bytes apart
        const uint64_t v_desc = (r_desc & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(S::ATOM >> 4) << 16);
        uint32_t base = 0;  // loads of the pieces before
        uint32_t pt[2] = {0, 0};
        bool ok = true;
        int piece = 0;
        for (; w.left >= 0 && ok; dec::next<KEYS>(a, w)) {
          if (w.count == 0) continue;
          const int n = w.count;
          const int steps = two ? n : (n + 1) / 2;
          // unit of group i's step k; >= n: none
          auto unit = [&](int i, int k) { return two ? k : 2 * k + i; };
          if (!mbar_wait(q_full, piece++ & 1, abort_flag, 46)) break;
          auto scores = [&](int i, int k) {
            const int u = unit(i, k);
            if (u >= n) return;
            const uint32_t ld = base + 2 * u, st = ld % S::SLOTS;
            if (!mbar_wait(&full[st], (ld / S::SLOTS) & 1, abort_flag, 47)) { ok = false; return; }
            tc_fence_after();
            const uint64_t qd = q_desc + (two && i ? S::TILE >> 4 : 0), kd = r_desc + ((st * S::TILE) >> 4);
            const uint32_t d = tmem + COL_S + 128 * i;
            if (one) {
#pragma unroll
              for (int ks = 0; ks < DP / 16; ++ks) {
                const uint64_t step = (ks >> 2) * (S::ATOM >> 4) + (ks & 3) * 2;
                mma_bf16(d, qd + step, kd + step, id_s, ks > 0);
              }
              mma_commit(&s_full[i]);
              if (!two || i) mma_commit(&empty[st]);
            }
            __syncwarp();
          };
          scores(0, 0);
          scores(1, 0);
          for (int k = 0; k < steps && ok; ++k) {
#pragma unroll 1
            for (int i = 0; i < 2; ++i) {
              const int u = unit(i, k);
              if (u >= n || !ok) continue;
              const uint32_t ld = base + 2 * u + 1, st = ld % S::SLOTS;
              if (!mbar_wait(&p_full[i], pt[i]++ & 1, abort_flag, 48) ||
                  !mbar_wait(&full[st], (ld / S::SLOTS) & 1, abort_flag, 47)) {
                ok = false;
                continue;
              }
              tc_fence_after();
              const uint64_t vd = v_desc + ((st * S::TILE) >> 4);
              const uint32_t d = tmem + COL_O + 128 * i, p = tmem + COL_S + 128 * i;
              if (one) {
#pragma unroll
                for (int ks = 0; ks < KEYS / 16; ++ks)
                  mma_ts(d, p + 8 * ks, vd + (uint64_t)(ks * (16 * 128 / 16)), id_pv, ks > 0 || k > 0);
                if (!two || i) mma_commit(&empty[st]);
                if (unit(i, k + 1) >= n) mma_commit(&o_full[i]);
              }
              __syncwarp();
              if (unit(i, k + 1) < n) scores(i, k + 1);
            }
          }
          base += 2 * n;
        }
      }
    }
  } else {
    // ------------------------------------------------ softmax groups
    dec::Walk w = dec::start<KEYS>(a, lane);
    const int grp = warp >> 2;
    // Up to 64 rows: they stand in the tile twice, and group 1 takes the second copy, whose warps run on the
    // other two schedulers of the SM.
    const int copy = !two && a.rows <= 64 ? 64 : 0;
    const int lane_row = threadIdx.x & 127, r = lane_row - (grp ? copy : 0);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + COL_S + 128 * grp, t_o = tmem + lanes + COL_O + 128 * grp;
    constexpr uint32_t inf = H16 ? 0x7c00u : 0x7f80u;
    uint32_t ts = 0, to = 0, base = 0;
    for (; w.left >= 0; dec::next<KEYS>(a, w)) {
      if (w.count == 0) continue;
      const int r0 = w.rtile * (two ? 2 * ROWS : ROWS) + (two ? grp * ROWS : 0);
      const bool live = r >= 0 && r0 + r < a.rows;
      const bool warp_live = __any_sync(0xffffffffu, live);
      const int tok = live ? dec::token_of(a, r0 + r) : 0;
      // ---- the row's queries (both groups share tile 0 when there is one: group i brings half of the rows)
      {
        uint8_t* q_sm = sm + (two && grp ? S::TILE : 0);
        // a warp's 32 rows of the tile, DP / 8 lanes side by side in a row
        constexpr int PER = DP / 8, STEP = 32 / PER;
        const int c = lane % PER;
        const int i0 = two ? 0 : grp * 16, i1 = two ? 32 : i0 + 16;
        // sixteen loads on their way before the first is stored
        uint4 v[32 / STEP];
#pragma unroll
        for (int i = 0; i < 32 / STEP; ++i) {
          const int row = (warp & 3) * 32 + i * STEP + lane / PER;
          const int qr = r0 + (copy ? row & 63 : row);  // the query row at this row of the tile
          v[i] = make_uint4(0, 0, 0, 0);
          if (i * STEP >= i0 && i * STEP < i1 && qr < a.rows && c * 8 < a.d)
            v[i] = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + dec::row_offset(a, w.b, w.head, qr))[c];
        }
#pragma unroll
        for (int i = 0; i < 32 / STEP; ++i)
          if (i * STEP >= i0 && i * STEP < i1)
            *reinterpret_cast<uint4*>(q_sm + at((warp & 3) * 32 + i * STEP + lane / PER, c)) = v[i];
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      float m = -INFINITY, l = 0.f;
      const int n = w.count;
      int mine = 0;
      bool poison = false;
      for (int k = two ? 0 : grp; k < n; k += two ? 1 : 2, ++mine) {
        mbar_wait(&s_full[grp], ts++ & 1, abort_flag, 49);  // on expiry every wait returns: all warps finish
        tc_fence_after();
        const int key0 = (w.tile + k) * KEYS;
        const bool open = key0 + KEYS > w.n;  // the unit reaches past the committed rows
        if (open && !(two && grp)) {
          // values behind the drafts, and drafts' that are not finite, become zero: one key a thread
          const uint32_t ld = base + 2 * k + 1, st = ld % S::SLOTS;
          mbar_wait(&full[st], (ld / S::SLOTS) & 1, abort_flag, 47);
          if (key0 + lane_row >= w.n) {
            uint8_t* v_sm = ring + st * S::TILE;
            bool clear = key0 + lane_row >= w.end;
            if (!clear) {
              for (int c = 0; c < DP / 8; ++c) clear = clear || non_finite(*reinterpret_cast<uint4*>(v_sm + at(lane_row, c)), inf);
              if (clear) *poison_flag = 1;
            }
            if (clear)
              for (int c = 0; c < DP / 8; ++c) *reinterpret_cast<uint4*>(v_sm + at(lane_row, c)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
        }
        if (warp_live) {
          uint32_t sees[4] = {~0u, ~0u, ~0u, ~0u};
          if (open) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sees[i] = dec::see<32>(a, w, tok, live, key0 + 32 * i, lane);
          }
          // the row's largest score; scores are read from TMEM twice, so that 64 at a time are in registers
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float s[32];
            ld32(t_s + 32 * c, s);
            ld_wait32(s);
            if (open) {
              const uint32_t bits = c < 2 ? (c ? sees[1] : sees[0]) : (c == 2 ? sees[2] : sees[3]);
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(bits >> i & 1)) s[i] = -INFINITY;
            }
            float mx[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              mx[i] = max3_nan(s[8 * i], s[8 * i + 1], s[8 * i + 2]);
              mx[i] = max3_nan(mx[i], s[8 * i + 3], s[8 * i + 4]);
              mx[i] = max3_nan(mx[i], s[8 * i + 5], s[8 * i + 6]);
            }
            top = max3_nan(top, max3_nan(mx[0], s[7], s[15]), max3_nan(mx[1], s[23], s[31]));
            top = max3_nan(top, mx[2], mx[3]);
          }
          top *= a.scale_log2;
          if (!(top < INFINITY)) l = NAN;  // a NaN or an infinite score: so is the row, as its definition has it
          // m: the reference of dec::LAG and dec::lift; a difference of two scores is exact where their sum with LAG is not
          const bool grow = top - m > dec::LAG + dec::lift(H16);
          if (__any_sync(0xffffffffu, grow)) {
            const float mn = grow ? top - dec::lift(H16) : m;
            const float f = mn == -INFINITY ? 1.f : exp2_sfu(m - mn);
            l *= f;
            m = mn;
            if (mine > 0) {
#pragma unroll 1
              for (int c = 0; c < DP; c += 32) {
                float o[32];
                ld32(t_o + c, o);
                ld_wait32(o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] *= f;
                st16(t_o + c, reinterpret_cast<const uint32_t*>(o));
                st16(t_o + c + 16, reinterpret_cast<const uint32_t*>(o) + 16);
              }
            }
          }
          const float neg = m == -INFINITY ? 0.f : -m;
          const float2 sc2 = make_float2(a.scale_log2, a.scale_log2), neg2 = make_float2(neg, neg);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          // One fused multiply-add from score to exponent, as long as the rounding of m is a fraction of a power of two.
          // Scores beyond that are rounded like the maximum that m came from, then subtracted, which keeps exponents
          // below LAG + lift.
          auto weights = [&](auto masked) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              float x[32];
              ld32(t_s + 32 * c, x);
              ld_wait32(x);
              const uint32_t bits = c < 2 ? (c ? sees[1] : sees[0]) : (c == 2 ? sees[2] : sees[3]);
              uint32_t pk[16];
#pragma unroll
              for (int q = 0; q < 16; ++q) {
                float2 z = make_float2(x[2 * q], x[2 * q + 1]), e;
                if constexpr (decltype(masked)::value)  // not packed, whose product and sum the compiler would fuse
                  z = make_float2(__fadd_rn(__fmul_rn(z.x, sc2.x), neg), __fadd_rn(__fmul_rn(z.y, sc2.y), neg));
                else
                  z = __ffma2_rn(z, sc2, neg2);
                if constexpr (decltype(masked)::value) {  // the SFU, whose 2^-inf is 0
                  e.x = bits >> (2 * q) & 1 ? exp2_sfu(z.x) : 0.f;
                  e.y = bits >> (2 * q + 1) & 1 ? exp2_sfu(z.y) : 0.f;
                } else {
                  e = q & 1 ? exp2_fma2_p3(z) : make_float2(exp2_sfu(z.x), exp2_sfu(z.y));
                }
                sum[q & 1] = __fadd2_rn(sum[q & 1], e);
                pk[q] = pack2h(e, H16);
              }
              st16(t_s + 16 * c, pk);  // columns whose scores have been read
            }
          };
          if (open || __any_sync(0xffffffffu, fabsf(top) > 4194304.f)) {  // 2^22
            weights(std::true_type());
          } else {
            weights(std::false_type());
          }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[grp]);
      }
      base += 2 * n;

      // ---- end of the piece
      if (mine > 0) {
        mbar_wait(&o_full[grp], to++ & 1, abort_flag, 50);
        tc_fence_after();
      }
      auto both = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
      both();
      poison = *poison_flag != 0;
      // o[0..31] += the weights of drafts with non-finite values times those values
      auto add_poisoned = [&](float* o, int c0) {
        if (!live || mine == 0) return;
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + dec::row_offset(a, w.b, w.head, r0 + r);
        const int64_t kv0 = ((int64_t)w.b * a.kv_heads + w.head) * a.capacity;
        const int from = max(w.n, w.tile * KEYS), to_key = min(w.end, (w.tile + n) * KEYS);
        for (int key = from; key < to_key; ++key) {
          if (!two && ((key / KEYS - w.tile) & 1) != grp) continue;  // the other group's unit
          if (!dec::visible(a, w, tok, key)) continue;
          const uint16_t* kr = static_cast<const uint16_t*>(a.k) + (kv0 + key) * a.d;
          const uint16_t* vr = static_cast<const uint16_t*>(a.v) + (kv0 + key) * a.d;
          bool bad = false;
          for (int c = 0; c < a.d; ++c) bad = bad || (vr[c] & inf) == inf;
          if (!bad) continue;
          float x = 0.f;
          for (int c = 0; c < a.d; ++c)
            x = fmaf(load_as_f32(q, a.dtype, c), load_as_f32(kr, a.dtype, c), x);
          const float p = exp2_sfu(__fadd_rn(__fmul_rn(x, a.scale_log2), m == -INFINITY ? 0.f : -m));
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c0 + c < a.d) o[c] += p * load_as_f32(vr, a.dtype, c0 + c);
        }
      };
      const bool whole = w.count == w.tiles;
      const int64_t slot_row = (int64_t)dec::slot(w) * (two ? 2 * ROWS : ROWS) + (two ? grp * ROWS : 0);
      // The warp's 32 rows pass through its part of the Q tile, 32 dims at a time, so that lanes side by side write
      // neighbours: [32 rows][8 pieces of 4 dims], pieces turned by the row.
      float4* stage = reinterpret_cast<float4*>(sm + (two && grp ? S::TILE : 0) + (warp & 3) * 4096);
      const int row_base = (warp & 3) * 32;  // copies (up to 64 rows) are group 1's, which writes nothing
      int64_t out_at[4];  // elements of the output at the rows this lane writes
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = r0 + row_base + i * 8 + lane / 4;
        out_at[i] = row < a.rows ? dec::row_offset(a, w.b, w.head, row) : -1;
      }
      // f: what the group's sums are multiplied by; `other`: group 1's rows in shared memory to add
      auto finish = [&](float f, float f_other, float mm, float ll, int c, float* o, const float4* other) {
        const float inv = !whole ? 1.f : ll == 0.f ? 0.f : 1.f / ll;  // a row that sees nothing is zero
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 x = other && live ? other[i * ROWS] : make_float4(0.f, 0.f, 0.f, 0.f);
          stage[lane * 8 + (i ^ (lane & 7))] =
              make_float4(fmaf(o[4 * i], f, x.x * f_other) * inv, fmaf(o[4 * i + 1], f, x.y * f_other) * inv,
                          fmaf(o[4 * i + 2], f, x.z * f_other) * inv, fmaf(o[4 * i + 3], f, x.w * f_other) * inv);
        }
        if (!whole && c == 0 && live) a.part_ml[slot_row + r] = make_float2(mm, ll);
        __syncwarp();
        if (whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + lane / 4, p = lane & 3;
            const float4 u = stage[row * 8 + ((2 * p) ^ (row & 7))], v = stage[row * 8 + ((2 * p + 1) ^ (row & 7))];
            const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
            if (out_at[i] >= 0 && c + 8 * p < a.d)
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + out_at[i] + c + 8 * p) = pack8h(x, H16);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = i * 4 + lane / 8, p = lane & 7;
            if (r0 + row_base + row < a.rows && c + 4 * p < a.d)
              *reinterpret_cast<float4*>(a.part + (slot_row + row_base + row) * a.d + c + 4 * p) =
                  stage[row * 8 + (p ^ (row & 7))];
          }
        }
        __syncwarp();
      };
      auto load_o = [&](int c, float* o) {
        __syncwarp();  // the load is the warp's
        if (mine > 0) {
          ld32(t_o + c, o);
          ld_wait32(o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        if (poison) add_poisoned(o, c);
      };
      if (two) {
        if (warp_live)
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          float o[32];
          load_o(c, o);
          finish(1.f, 0.f, m, l, c, o, nullptr);
        }
      } else {
        // group 1 hands its sums to group 0 through the second Q tile, half of the dims at a time
        float4* buf = reinterpret_cast<float4*>(sm + S::TILE);  // [DP / 8][128]
        if (grp == 1 && live) ml_sm[r] = make_float2(m, l);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (grp == 1 && n > 1 && warp_live) {
#pragma unroll 1
            for (int c = 0; c < DP / 2; c += 32) {
              float o[32];
              load_o(half * (DP / 2) + c, o);
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (live) buf[(c / 4 + i) * ROWS + r] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
          }
          both();
          if (grp == 0 && warp_live) {
            const float2 other = live ? ml_sm[r] : make_float2(-INFINITY, 0.f);
            const float mm = fmaxf(m, other.x);
            const float f = mm == -INFINITY ? 1.f : exp2_sfu(m - mm), fo = mm == -INFINITY ? 1.f : exp2_sfu(other.x - mm);
            const float ll = l * f + other.y * fo;
#pragma unroll 1
            for (int c = 0; c < DP / 2; c += 32) {
              float o[32];
              load_o(half * (DP / 2) + c, o);
              finish(f, fo, mm, ll, half * (DP / 2) + c, o, n > 1 ? buf + (c / 4) * ROWS + r : nullptr);
            }
          }
          both();
        }
      }
      if (threadIdx.x == 0) dec::note_segment(a, w);
      tc_fence_before();
      both();
      if (threadIdx.x == 0) *poison_flag = 0;  // before this thread's warp brings the next piece's queries
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // loads and products still in flight end before shared memory and TMEM are given back
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

template <int DP, bool H16>
static int run(const CUtensorMap& km, const CUtensorMap& vm, const Args& a, int grid, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_smem(tree_tc_kernel<DP, H16>, (int)Shape<DP>::SMEM, done)) return rc;
  return launch_pdl(tree_tc_kernel<DP, H16>, grid, THREADS, (size_t)Shape<DP>::SMEM, s, km, vm, a);
}

}  // namespace dtc

namespace dec {

int run_tc(bool h16, const Plan& pl, const Args& a, cudaStream_t s) {
  CUtensorMap km, vm;
  if (int rc = cache_maps(a, dtc::KEYS, &km, &vm)) return rc;
  if (pl.dp == 64) return h16 ? dtc::run<64, true>(km, vm, a, pl.grid, s) : dtc::run<64, false>(km, vm, a, pl.grid, s);
  return h16 ? dtc::run<128, true>(km, vm, a, pl.grid, s) : dtc::run<128, false>(km, vm, a, pl.grid, s);
}

}  // namespace dec
}  // namespace c3b
