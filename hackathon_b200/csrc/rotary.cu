// Rotary positions, per-head query/key RMS norms fused with the rotation, and
// the append of the rotated keys (and the values) to a decoding cache.
//
// One pass over the heads of each token.  With t = position * step_i / 2^64
// turns, pair i of a head becomes
//   (a', b') = scale * (a cos 2 pi t - b sin 2 pi t, b cos 2 pi t + a sin 2 pi t),
// pair i being elements (i, i + R/2) of the head (half layout) or (2i, 2i + 1)
// (interleaved) of its first R elements; the rest passes through.  Queries and
// keys are first scaled by w / sqrt(mean(x^2) + eps) where the call normalises.
//
// Frequencies come as 64-bit fixed-point fractions of a turn, so the product
// with an integer position wraps modulo one turn exactly: the range reduction
// of far positions costs one 64-bit multiplication, loses nothing, and there is
// no cosine table to read.  The upper 32 bits of the phase go to sincospif.
//
// Everything is computed in fp32 and rounded once, to the output's type.
#include <atomic>
#include <cmath>

#include "common.cuh"
#include "tc_prims.cuh"

namespace c3b {

namespace rot {

enum { STATUS_APPEND = 40 };

struct Args {
  const void* in;       // [tokens, hq + hk + hv, d]
  void* out[3];         // q, k, v heads: first head of the first token / sequence
  const float* w[2];    // norm weights of q, k (null: ones)
  int w_stride[2];      // elements from one head's weights to the next (0: shared)
  const void* pos;
  const long long* steps;
  const int* lengths;   // committed rows of each cache, or null when k and v are written like q
  int64_t tokens;
  int64_t capacity;
  int64_t pos_stride;   // positions from one sequence to the next (0: shared)
  int seq, heads[3], d, rotary, pos64, interleaved, normalize, copy_v;
  int64_t out_stride;   // elements from one token to the next in out[0] (and in out[1], out[2] without lengths)
  int chunks, chunk_heads;
  float scale, eps, inv_d;
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// N consecutive elements moved as one 4-, 8- or 16-byte word.
template <int BYTES> struct Word;
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<16> { typedef uint4 type; };
template <typename T, int N> struct Piece {
  typedef typename Word<N * sizeof(T)>::type W;
  union {
    W w;
    T v[N];
  };
  __device__ __forceinline__ Piece() {}
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = w; }
};

__device__ __forceinline__ long long position(const Args& a, int64_t b, int64_t t) {
  const int64_t i = b * a.pos_stride + t;
  return a.pos64 ? static_cast<const long long*>(a.pos)[i] : (long long)static_cast<const int*>(a.pos)[i];
}

// scale * (cos, sin) of position * step turns.
__device__ __forceinline__ void turn(long long pos, long long step, float scale, float& c, float& s) {
  const unsigned long long phase = (unsigned long long)pos * (unsigned long long)step;
  const float x = (float)(int)(phase >> 32) * 4.656612873077392578125e-10f;  // 2^-31: half turns in [-1, 1]
  sincospif(x, &s, &c);
  c *= scale;
  s *= scale;
}

// Where head h of the token goes; null: nowhere.  `role` is 0 (q), 1 (k) or 2 (v).
template <typename T>
__device__ __forceinline__ T* destination(const Args& a, int role, int h, int64_t token, int64_t b, int64_t row) {
  T* base = static_cast<T*>(a.out[role]);
  if (role == 0 || !a.lengths) return base + token * a.out_stride + (int64_t)h * a.d;
  if (row < 0) return nullptr;
  return base + ((b * a.heads[role] + h) * a.capacity + row) * a.d;
}

// The token's row in the caches; -1 where its sequence does not fit.
__device__ __forceinline__ int64_t cache_row(const Args& a, int64_t b, int64_t t) {
  if (!a.lengths) return -1;
  const int n = a.lengths[b];
  if (n < 0 || (int64_t)n + a.seq > a.capacity) {
    atomicExch(&g_status, STATUS_APPEND);
    return -1;
  }
  return n + t;
}

// Two values at a time, so that conversions and products come in pairs.
template <typename T> __device__ __forceinline__ float2 pair_of(const T* v) { return make_float2(to_f32(v[0]), to_f32(v[1])); }
template <> __device__ __forceinline__ float2 pair_of(const __nv_bfloat16* v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(v));
}
template <> __device__ __forceinline__ float2 pair_of(const __half* v) { return __half22float2(*reinterpret_cast<const __half2*>(v)); }
template <typename T> __device__ __forceinline__ void set_pair(T* v, float2 x) { v[0] = x.x, v[1] = x.y; }
template <> __device__ __forceinline__ void set_pair(__nv_bfloat16* v, float2 x) {
  *reinterpret_cast<__nv_bfloat162*>(v) = __float22bfloat162_rn(x);
}
template <> __device__ __forceinline__ void set_pair(__half* v, float2 x) { *reinterpret_cast<__half2*>(v) = __float22half2_rn(x); }

// What is done to a head besides the rotation.
enum { PLAIN = 0, NORM = 1 /* weights shared by the heads, or none */, NORM_EACH = 2 /* weights of each head */ };

// A lane's part in the heads of one token: a unit of 2 * VEC elements, VEC pairs
// or 2 * VEC elements behind the rotated part.  LANES lanes (a power of two; 0:
// known at run time) share a head, and the heads of a warp share the work on the
// sines.  These, multiplied by the norm's weights where all heads
// share them, serve every head:
//   a' = inv (a (w_a cos) - b (w_b sin)),  b' = inv (b (w_b cos) + a (w_a sin)).
template <typename T, int VEC, int MODE, bool INTERLEAVED, int LANES>
struct Unit {
  int sub, off0, off1;  // the unit's two pieces of VEC elements
  bool active, turned;
  int lanes, own, role; // own: which head of the warp's; role: whose coefficients are held, -1: none
  static constexpr int SHARE = LANES == 0 ? 1 : 32 / LANES < VEC ? 32 / LANES : VEC;
  long long steps[LANES ? VEC / SHARE : 1];  // of the pairs the lane works out: pair i * SHARE + g is the warp's head g's
  float c[VEC], s[VEC];
  float ca[VEC], sb[VEC], cb[VEC], sa[VEC];  // pair j: a' = a ca + b sb, b' = b cb + a sa

  __device__ __forceinline__ Unit(const Args& a, int lane, int lanes_) {
    lanes = LANES ? LANES : lanes_;
    sub = lane & (lanes - 1), own = lane / lanes;
    active = sub < a.d / (2 * VEC), turned = sub < a.rotary / (2 * VEC);
    // a piece of each half of the rotated part, or of each half of what is behind it: lanes side by side, pieces too
    off0 = turned ? sub * VEC : a.rotary / 2 + sub * VEC;
    off1 = off0 + (turned ? a.rotary : a.d - a.rotary) / 2;
    if constexpr (LANES > 0) {
#pragma unroll
      for (int i = 0; i < VEC / SHARE; ++i) steps[i] = a.steps[turned ? pair_index(a, i * SHARE + own % SHARE) : 0];
    }
  }

  // The frequency of pair j: (off0 + j, off1 + j), or, interleaved, one of the pairs within the pieces.
  __device__ __forceinline__ int pair_index(const Args& a, int j) const {
    return !INTERLEAVED ? sub * VEC + j : j < VEC / 2 ? sub * (VEC / 2) + j : a.rotary / 4 + sub * (VEC / 2) + j - VEC / 2;
  }

  __device__ __forceinline__ void set_token(const Args& a, long long pos) {
    role = -1;
    if constexpr (LANES > 0) {
#pragma unroll
      for (int i = 0; i < VEC / SHARE; ++i) {
        float x, y;
        turn(pos, steps[i], a.scale, x, y);
#pragma unroll
        for (int g = 0; g < SHARE; ++g) {
          c[i * SHARE + g] = __shfl_sync(0xffffffffu, x, sub + g * LANES);
          s[i * SHARE + g] = __shfl_sync(0xffffffffu, y, sub + g * LANES);
        }
      }
    } else if (turned) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) turn(pos, a.steps[pair_index(a, j)], a.scale, c[j], s[j]);
    }
    if (!turned) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) c[j] = 1.f, s[j] = 0.f;
    }
  }

  // The same from a token's cosines and sines, worked out before.
  __device__ __forceinline__ void take_token(const Args& a, const float* cosines, const float* sines) {
    role = -1;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int p = turned ? pair_index(a, j) : 0;
      c[j] = turned ? cosines[p] : 1.f;
      s[j] = turned ? sines[p] : 0.f;
    }
  }

  __device__ __forceinline__ void set_role(const Args& a, int r) {
    if (r == role || r == 2) return;
    role = r;
    if (MODE == NORM_EACH) return;
    const float* w = MODE == NORM ? a.w[r] : nullptr;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float wa = 1.f, wb = 1.f;
      if (w && active) {
        const float* pair = j < VEC / 2 ? w + off0 + 2 * j : w + off1 + 2 * j - VEC;
        wa = INTERLEAVED ? pair[0] : w[off0 + j];
        wb = INTERLEAVED ? pair[1] : w[off1 + j];
      }
      ca[j] = wa * c[j], sb[j] = -wb * s[j], cb[j] = wb * c[j], sa[j] = wa * s[j];
    }
  }

  // Head h of the q (r = 0) or k (r = 1) heads, in place; the whole warp calls, `on` where the lane has a part.
  __device__ __forceinline__ void head(const Args& a, int r, int h, bool on, Piece<T, VEC>& p0, Piece<T, VEC>& p1) const {
    // two pairs at a time (half layout) or one (interleaved)
    float2 x[VEC / 2], y[VEC / 2];
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      x[j] = pair_of(p0.v + 2 * j);
      y[j] = pair_of(p1.v + 2 * j);
    }
    float inv = 1.f;
    if (MODE != PLAIN) {
      float2 q = make_float2(0.f, 0.f);
      if (on) {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          q = __ffma2_rn(x[j], x[j], q);
          q = __ffma2_rn(y[j], y[j], q);
        }
      }
      float total = q.x + q.y;
      if constexpr (LANES > 0) {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      } else {
        for (int o = lanes / 2; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      }
      inv = rsqrtf(fmaf(total, a.inv_d, a.eps));
    }
    if (MODE == NORM_EACH && on) {
      const float* w = a.w[r];
      if (w) {
        w += (int64_t)h * a.w_stride[r];
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          x[j] = __fmul2_rn(x[j], make_float2(w[off0 + 2 * j], w[off0 + 2 * j + 1]));
          y[j] = __fmul2_rn(y[j], make_float2(w[off1 + 2 * j], w[off1 + 2 * j + 1]));
        }
      }
    }
    const float2 inv2 = make_float2(inv, inv);
    auto A = [&](int j) { return MODE == NORM_EACH ? c[j] : ca[j]; };
    auto B = [&](int j) { return MODE == NORM_EACH ? -s[j] : sb[j]; };
    auto C = [&](int j) { return MODE == NORM_EACH ? c[j] : cb[j]; };
    auto D = [&](int j) { return MODE == NORM_EACH ? s[j] : sa[j]; };
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      float2 u, v;
      if (INTERLEAVED) {
        // x[j] is pair j of the unit, y[j] pair VEC / 2 + j
        const int k = VEC / 2 + j;
        u = __fmul2_rn(x[j], make_float2(A(j), C(j)));
        v = __fmul2_rn(y[j], make_float2(A(k), C(k)));
        if (turned) {  // behind the rotated part nothing of a neighbour is added, not even 0 times it
          u = __ffma2_rn(make_float2(x[j].y, x[j].x), make_float2(B(j), D(j)), u);
          v = __ffma2_rn(make_float2(y[j].y, y[j].x), make_float2(B(k), D(k)), v);
        }
      } else {
        u = __fmul2_rn(x[j], make_float2(A(2 * j), A(2 * j + 1)));
        v = __fmul2_rn(y[j], make_float2(C(2 * j), C(2 * j + 1)));
        if (turned) {
          u = __ffma2_rn(y[j], make_float2(B(2 * j), B(2 * j + 1)), u);
          v = __ffma2_rn(x[j], make_float2(D(2 * j), D(2 * j + 1)), v);
        }
      }
      if (MODE != PLAIN) u = __fmul2_rn(u, inv2), v = __fmul2_rn(v, inv2);
      set_pair(p0.v + 2 * j, u);
      set_pair(p1.v + 2 * j, v);
    }
  }
};

// Where a role's heads of the token go, and how far one is from the next; null: nowhere.
template <typename T>
__device__ __forceinline__ T* heads_of(const Args& a, int role, int token, int b, int64_t row, int64_t& pitch) {
  const bool cached = role > 0 && a.lengths;
  pitch = cached ? a.capacity * a.d : a.d;
  if (cached && row < 0) return nullptr;
  return static_cast<T*>(a.out[role]) +
         (cached ? ((int64_t)b * a.heads[role] * a.capacity + row) * a.d : (int64_t)token * a.out_stride);
}

// Narrower pieces than 16 bytes, or weights of each head: a warp takes one token and
// chunk_heads of its heads; NB heads are loaded before the first is stored.
// 16 x 512 tokens, 32 + 8 + 8 heads of 128 in bf16, norm and turn (rotary_bulk_kernel: 45 us, floor 31): weights of each
// head 80 us, which each lane reads for each head; 8-byte pieces 61 us, 4-byte pieces 90 us.
template <typename T, int VEC, int MODE, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(const Args a, const int lanes) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int NB = 2;
  const int lane = threadIdx.x & 31, hpw = 32 / lanes, own = lane / lanes;
  const int item = (int)(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5));  // threads may pass 32 bits, warps do not
  const int token = item / a.chunks;
  if (token >= a.tokens) return;
  const int b = token / a.seq, t = token - b * a.seq;
  const int width = a.heads[0] + a.heads[1] + a.heads[2];
  const int first = (item - token * a.chunks) * a.chunk_heads;
  const int last = min(width - (a.copy_v ? 0 : a.heads[2]), first + a.chunk_heads);
  Unit<T, VEC, MODE, INTERLEAVED, 0> unit(a, lane, lanes);
  unit.set_token(a, position(a, b, t));
  const int64_t row = cache_row(a, b, t);
  const T* src = static_cast<const T*>(a.in) + (int64_t)token * width * a.d;
  int begin = 0;
#pragma unroll 1
  for (int role = 0; role < 3; begin += a.heads[role], ++role) {
    const int lo = max(first, begin), hi = min(last, begin + a.heads[role]);
    int64_t pitch;
    T* dst = heads_of<T>(a, role, token, b, row, pitch);
    if (lo >= hi || !dst) continue;
    unit.set_role(a, role);
#pragma unroll 1
    for (int h0 = lo; h0 < hi; h0 += hpw * NB) {
      Piece<T, VEC> p0[NB], p1[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int h = h0 + i * hpw + own;
        if (unit.active && h < hi) {
          p0[i].load(src + (int64_t)h * a.d + unit.off0);
          p1[i].load(src + (int64_t)h * a.d + unit.off1);
        }
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int h = h0 + i * hpw + own - begin;
        const bool on = unit.active && h + begin < hi;
        if (role < 2) unit.head(a, role, h, on, p0[i], p1[i]);
        if (on) {
          p0[i].store(dst + h * pitch + unit.off0);
          p1[i].store(dst + h * pitch + unit.off1);
        }
      }
    }
  }
}

// Tokens of few heads: heads of several tokens share a warp.  SHARED: the block
// first works out the sines of its tokens, each once, into shared memory; else
// each lane those of its pairs.
template <typename T, int MODE, bool INTERLEAVED, bool SHARED>
__global__ void __launch_bounds__(256) rotary_few_kernel(const Args a, const int lanes, const int64_t items) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int VEC = 16 / sizeof(T);
  constexpr int MOST = SHARED ? 256 * VEC / 3 : 0;  // pairs of a block's tokens
  __shared__ __align__(16) float cosines[MOST + 1], sines[MOST + 1];
  __shared__ long long positions[SHARED ? 64 : 1];  // a block takes at most 8 * 32 / 4 heads
  const int lane = threadIdx.x & 31;
  Unit<T, VEC, MODE, INTERLEAVED, 0> unit(a, lane, lanes);
  const int width = a.heads[0] + a.heads[1] + a.heads[2], total = width - (a.copy_v ? 0 : a.heads[2]);
  const int per_block = 8 * (32 / lanes), half = a.rotary / 2, item = (threadIdx.x >> 5) * (32 / lanes) + unit.own;
  const int64_t first = (int64_t)blockIdx.x * per_block;
  const bool on = unit.active && first + item < items;
  int token0 = 0, tokens = 0, token, h;
  if constexpr (SHARED) {  // the block's heads: of tokens token0 .. token0 + tokens - 1, from head h0 of the first
    token0 = items >> 31 ? (int)(first / total) : (int)((uint32_t)first / (uint32_t)total);
    const int h0 = (int)(first - (int64_t)token0 * total), here = items - first < per_block ? (int)(items - first) : per_block;
    tokens = (h0 + here - 1) / total + 1;
    const int nth = (h0 + item) / total;
    token = on ? token0 + nth : token0, h = on ? h0 + item - nth * total : 0;
  } else {
    token = on ? (int)((first + item) / total) : 0, h = on ? (int)(first + item - (int64_t)token * total) : 0;
  }
  const int b = token / a.seq, t = token - b * a.seq;
  const int role = h < a.heads[0] ? 0 : h < a.heads[0] + a.heads[1] ? 1 : 2;
  const int head = h - (role == 0 ? 0 : role == 1 ? a.heads[0] : a.heads[0] + a.heads[1]);
  Piece<T, VEC> p0, p1;
  if (on) {
    const T* src = static_cast<const T*>(a.in) + ((int64_t)token * width + h) * a.d;
    p0.load(src + unit.off0), p1.load(src + unit.off1);
  }
  if (SHARED) {
    if (threadIdx.x < tokens) {
      const int tk = token0 + threadIdx.x, bb = tk / a.seq;
      positions[threadIdx.x] = position(a, bb, tk - bb * a.seq);
    }
    int p = threadIdx.x % half, i = threadIdx.x / half;
    const int dp = 256 % half, di = 256 / half;
    __syncthreads();
    for (; i < tokens; p += dp, i += di) {
      if (p >= half && ++i >= tokens) break;
      if (p >= half) p -= half;
      turn(positions[i], a.steps[p], a.scale, cosines[i * half + p], sines[i * half + p]);
    }
  }
  int64_t pitch;
  T* dst = heads_of<T>(a, role, token, b, on ? cache_row(a, b, t) : -1, pitch);
  if (SHARED) {
    __syncthreads();
    unit.take_token(a, cosines + (token - token0) * half, sines + (token - token0) * half);
  } else {
    unit.set_token(a, position(a, b, t));
  }
  const Piece<T, VEC> v0 = p0, v1 = p1;
  unit.set_role(a, role);
  unit.head(a, role < 2 ? role : 0, head, on, p0, p1);
  if (on && dst) {
    dst += head * pitch;
    if (role == 2) p0 = v0, p1 = v1;
    p0.store(dst + unit.off0), p1.store(dst + unit.off1);
  }
}

// The common case, 16-byte pieces.  HBM bounds it, so the loads need no
// registers: a warp brings its heads, which lie side by side, into shared memory
// by bulk copies of up to 4 KB of q, k or v heads, as many ahead of its work as
// fit its 12 KB, across tokens: 12 pieces of up to 1 KB, 6 of 2 KB or 3 of 4 KB.
// A warp takes items (a token and chunk_heads of its heads) W apart.
constexpr int WARPS = 8, RING = 12288, MAX_STAGES = 12;
constexpr uint32_t BULK_SMEM = WARPS * RING;

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   tc::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
               : "memory");
}

template <typename T, int MODE, bool INTERLEAVED, int LANES>
__global__ void __launch_bounds__(32 * WARPS, 2) rotary_bulk_kernel(const Args a, const int items, const int piece) {
  constexpr int VEC = 16 / sizeof(T), HPW = 32 / LANES;
  extern __shared__ __align__(128) uint8_t ring_sm[];
  __shared__ uint64_t bars[WARPS][MAX_STAGES];
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stages = RING / piece;
  uint8_t* ring = ring_sm + warp * RING;
  uint64_t* full = bars[warp];
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0) {
    for (int i = 0; i < stages; ++i) tc::mbar_init(&full[i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tc::fence_proxy_async();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int k0 = a.heads[0], v0 = k0 + a.heads[1], width = v0 + a.heads[2], total = a.copy_v ? width : v0;
  const int per = piece / (a.d * (int)sizeof(T)) / HPW * HPW;  // heads of a piece, at most
  const int step = (int)gridDim.x * WARPS;
  // heads of the piece that begins at head h of a chunk that ends at `last`: all q, all k or all v
  auto heads_from = [&](int h, int last) { return min(per, min(last, h < k0 ? k0 : h < v0 ? v0 : width) - h); };

  // the next piece to bring: an item, and a head
  int next_item = (int)blockIdx.x * WARPS + warp, next_head = -1, next_last = 0;
  const T* next_src = nullptr;
  auto bring = [&](int st) {
    if (next_item >= items) return;
    if (next_head < 0) {
      const int token = next_item / a.chunks;
      next_head = (next_item - token * a.chunks) * a.chunk_heads;
      next_last = min(total, next_head + a.chunk_heads);
      next_src = static_cast<const T*>(a.in) + (int64_t)token * width * a.d;
    }
    const int n = heads_from(next_head, next_last);
    if (lane == 0) {
      const uint32_t bytes = (uint32_t)(n * a.d * (int)sizeof(T));
      tc::mbar_arrive_tx(&full[st], bytes);
      bulk_load(ring + st * piece, next_src + next_head * a.d, bytes, &full[st]);
    }
    next_head += n;
    if (next_head >= next_last) next_head = -1, next_item += step;
  };
  for (int i = 0; i < stages; ++i) bring(i);

  Unit<T, VEC, MODE, INTERLEAVED, LANES> unit(a, lane, LANES);
  int st = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int item = (int)blockIdx.x * WARPS + warp; item < items && ok; item += step) {
    const int token = item / a.chunks, first = (item - token * a.chunks) * a.chunk_heads;
    const int last = min(total, first + a.chunk_heads);
    const int b = token / a.seq, t = token - b * a.seq;
    const int64_t row = cache_row(a, b, t);
    unit.set_token(a, position(a, b, t));
    for (int h0 = first; h0 < last;) {
      const int n = heads_from(h0, last);
      const int role = h0 < k0 ? 0 : h0 < v0 ? 1 : 2, head = h0 - (role == 0 ? 0 : role == 1 ? k0 : v0);
      h0 += n;
      if (!tc::mbar_wait(&full[st], phase, &abort_flag, 51)) {
        ok = false;
        break;
      }
      int64_t pitch;
      T* dst = heads_of<T>(a, role, token, b, row, pitch);
      if (dst) {
        unit.set_role(a, role);
        dst += (head + unit.own) * pitch;
        const T* src = reinterpret_cast<const T*>(ring + st * piece) + unit.own * a.d;
        if (role == 2) {
#pragma unroll 2
          for (int h = unit.own; h < n; h += HPW, src += HPW * a.d, dst += HPW * pitch) {
            if (!unit.active) continue;
            Piece<T, VEC> p0, p1;
            p0.load(src + unit.off0), p1.load(src + unit.off1);
            p0.store(dst + unit.off0), p1.store(dst + unit.off1);
          }
        } else {
#pragma unroll 2
          for (int h = 0; h < n; h += HPW, src += HPW * a.d, dst += HPW * pitch) {
            const bool on = unit.active && h + unit.own < n;
            Piece<T, VEC> p0, p1;
            if (on) p0.load(src + unit.off0), p1.load(src + unit.off1);
            unit.head(a, role, 0, on, p0, p1);
            if (on) p0.store(dst + unit.off0), p1.store(dst + unit.off1);
          }
        }
      }
      __syncwarp();  // every lane has read the piece
      bring(st);
      if (++st == stages) st = 0, phase ^= 1;
    }
  }
  if (!ok)  // copies still in flight land before the block's shared memory is given back
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

// Any even rotary size, head size and alignment: a warp per head, one pair a lane.  The call above, one element off
// alignment: 221 us; 32 heads of 50, 10 turned, 16 x 512 tokens: 125 us for a floor of 8.
template <typename T>
__global__ void __launch_bounds__(256) rotary_any_kernel(const Args a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int total = a.heads[0] + a.heads[1] + (a.copy_v ? a.heads[2] : 0);
  const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int64_t token = item / total;
  if (token >= a.tokens) return;
  const int h = (int)(item - token * total);
  const int64_t b = token / a.seq, t = token - b * a.seq;
  const int role = h < a.heads[0] ? 0 : h < a.heads[0] + a.heads[1] ? 1 : 2;
  const int hh = h - (role > 0 ? a.heads[0] : 0) - (role > 1 ? a.heads[1] : 0);
  const T* src = static_cast<const T*>(a.in) + (token * (a.heads[0] + a.heads[1] + a.heads[2]) + h) * a.d;
  T* dst = destination<T>(a, role, hh, token, b, cache_row(a, b, t));
  if (!dst) return;
  if (role == 2) {
    for (int i = lane; i < a.d; i += 32) dst[i] = src[i];
    return;
  }
  float inv = 1.f;
  const float* w = nullptr;
  if (a.normalize) {
    float q = 0.f;
    for (int i = lane; i < a.d; i += 32) {
      const float x = to_f32(src[i]);
      q = fmaf(x, x, q);
    }
    inv = rsqrtf(warp_sum(q) / (float)a.d + a.eps);
    if (a.w[role]) w = a.w[role] + (int64_t)hh * a.w_stride[role];
  }
  const long long pos = position(a, b, t);
  for (int p = lane; p < a.rotary / 2; p += 32) {
    const int i = a.interleaved ? 2 * p : p, j = a.interleaved ? 2 * p + 1 : p + a.rotary / 2;
    float c, s;
    turn(pos, a.steps[p], a.scale, c, s);
    const float u = to_f32(src[i]) * (w ? inv * w[i] : inv), v = to_f32(src[j]) * (w ? inv * w[j] : inv);
    dst[i] = from_f32<T>(u * c - v * s);
    dst[j] = from_f32<T>(v * c + u * s);
  }
  for (int i = a.rotary + lane; i < a.d; i += 32) dst[i] = from_f32<T>(to_f32(src[i]) * (w ? inv * w[i] : inv));
}

template <typename T, int MODE, bool INTERLEAVED, int LANES>
static int launch_bulk(const Args& a, int items, cudaStream_t s) {
  const int blocks = (items + WARPS - 1) / WARPS, most = 2 * sm_count();  // two an SM are resident
  auto kernel = rotary_bulk_kernel<T, MODE, INTERLEAVED, LANES>;
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_smem(kernel, (int)BULK_SMEM, done)) return rc;
  // the largest piece there is: a role's heads, or a chunk's
  const int heads = a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1];
  const int64_t bytes = (int64_t)(heads < a.chunk_heads ? heads : a.chunk_heads) * a.d * sizeof(T);
  const int piece = bytes <= 1024 ? 1024 : bytes <= 2048 ? 2048 : 4096;
  return launch_pdl(kernel, blocks < most ? blocks : most, 32 * WARPS, BULK_SMEM, s, a, items, piece);
}

template <typename T, int VEC, int MODE, bool INTERLEAVED>
static int launch(const Args& a, int lanes, int items, cudaStream_t s) {
  if constexpr (VEC * sizeof(T) == 16 && MODE != NORM_EACH) {
    const int total = a.heads[0] + a.heads[1] + (a.copy_v ? a.heads[2] : 0), hpw = 32 / lanes;
    // 12 heads of 64 (eight a round) 30 us against 35, 5 of 96 11 against 18; from two rounds on the bulk copies win:
    // 8 heads of 128 38 us against 41, 24 of 64 42 against 55
    if (total < 2 * hpw) {
      const int64_t heads = a.tokens * total;
      const int per_block = 8 * hpw, blocks = (int)((heads + per_block - 1) / per_block);
      // Sines worked out once for a block cost as much as two and a half times as many of a lane's own:
      // 4 heads of 64 45 us against 48, 3 heads 48 either way, 2 heads 54 against 48.
      const int most = total == 1 ? per_block : (per_block - 2) / total + 2;  // tokens that a block's heads touch
      const bool shared = 3 * most * (a.rotary / 2) <= 256 * VEC;
      return launch_pdl(shared ? rotary_few_kernel<T, MODE, INTERLEAVED, true> : rotary_few_kernel<T, MODE, INTERLEAVED, false>,
                        blocks, 256, 0, s, a, lanes, heads);
    }
    switch (lanes) {
      case 4: return launch_bulk<T, MODE, INTERLEAVED, 4>(a, items, s);
      case 8: return launch_bulk<T, MODE, INTERLEAVED, 8>(a, items, s);
      case 16: return launch_bulk<T, MODE, INTERLEAVED, 16>(a, items, s);
      default: return launch_bulk<T, MODE, INTERLEAVED, 32>(a, items, s);
    }
  } else {
    return launch_pdl(rotary_kernel<T, VEC, MODE, INTERLEAVED>, (items + 7) / 8, 256, 0, s, a, lanes);
  }
}

template <typename T, int VEC>
static int run(Args a, cudaStream_t s) {
  const int units = a.d / (2 * VEC), lanes = units <= 4 ? 4 : units <= 8 ? 8 : units <= 16 ? 16 : 32, hpw = 32 / lanes;
  const int total = a.heads[0] + a.heads[1] + (a.copy_v ? a.heads[2] : 0);
  const int rounds = (total + hpw - 1) / hpw;
  // A token's heads are split over warps where that shortens the way of the
  // longest warp: waves of 16 warps an SM, each as long as its rounds of heads
  // and about three more for the token's positions and sines.
  const int64_t wave = (int64_t)sm_count() * 16;
  int64_t best = 0;
  for (int chunks = 1; chunks <= rounds && chunks <= 64; ++chunks) {
    const int each = (rounds + chunks - 1) / chunks;
    const int64_t cost = (a.tokens * chunks + wave - 1) / wave * (each + 3);
    if (chunks == 1 || cost < best) best = cost, a.chunk_heads = each * hpw;
  }
  a.chunks = (total + a.chunk_heads - 1) / a.chunk_heads;
  C3B_REQUIRE(a.tokens * a.chunks < ((int64_t)1 << 31) - 8, "rotary: too many tokens");
  const int items = (int)(a.tokens * a.chunks);
  const int mode = !a.normalize ? PLAIN : a.w_stride[0] || a.w_stride[1] ? NORM_EACH : NORM;
#define C3B_ROT(M) (a.interleaved ? launch<T, VEC, M, true>(a, lanes, items, s) : launch<T, VEC, M, false>(a, lanes, items, s))
  return mode == PLAIN ? C3B_ROT(PLAIN) : mode == NORM ? C3B_ROT(NORM) : C3B_ROT(NORM_EACH);
#undef C3B_ROT
}

template <typename T>
static int run_type(Args a, cudaStream_t s) {
  a.inv_d = 1.f / (float)a.d;
  const int total = a.heads[0] + a.heads[1] + (a.copy_v ? a.heads[2] : 0);
  if (a.tokens == 0 || total == 0 || a.d == 0) return C3B_OK;
  // Widest piece (16, 8 or 4 bytes) that divides the rotated part's halves, the
  // head and every pointer, and leaves at most 32 units a head.
  uintptr_t at = (uintptr_t)a.in | (uintptr_t)a.out[0] | (uintptr_t)a.out[1] | (uintptr_t)a.out[2];
  auto fits = [&](int vec) {
    return a.tokens < (1ll << 31) && a.rotary % (2 * vec) == 0 && a.d % (2 * vec) == 0 && a.d <= 64 * vec && at % (vec * sizeof(T)) == 0;
  };
  if constexpr (sizeof(T) == 2) {
    if (fits(8)) return run<T, 8>(a, s);
  }
  if (fits(4)) return run<T, 4>(a, s);
  if (fits(2)) return run<T, 2>(a, s);
  const int64_t blocks = (a.tokens * total + 7) / 8;
  C3B_REQUIRE(blocks < ((int64_t)1 << 31), "rotary: too many heads");
  return launch_pdl(rotary_any_kernel<T>, (int)blocks, 256, 0, s, a);
}

static int run_any(const Args& a, int dtype, cudaStream_t s) {
  switch (dtype) {
    case C3B_F32: return run_type<float>(a, s);
    case C3B_BF16: return run_type<__nv_bfloat16>(a, s);
    default: return run_type<__half>(a, s);
  }
}

// Positions and phase steps, shared by the three entry points.
static int take_positions(Args& a, const c3b_tensor& pos, const c3b_tensor& steps, int64_t batch, int64_t seq,
                          int rotary, const char* who) {
  const std::string w(who);
  C3B_REQUIRE(rotary >= 2 && rotary % 2 == 0 && rotary <= a.d, w + ": rotary_dim is even, 2 to head_dim");
  C3B_REQUIRE(steps.dtype == C3B_I64 && numel(steps) == rotary / 2, w + ": phase steps are int64 [rotary_dim / 2]");
  C3B_REQUIRE(pos.dtype == C3B_I64 || pos.dtype == C3B_I32, w + ": positions are int64 or int32");
  const bool shared = pos.ndim == 1 && pos.shape[0] == seq;
  C3B_REQUIRE(shared || (pos.ndim == 2 && pos.shape[0] == batch && pos.shape[1] == seq),
              w + ": positions are [batch, tokens] or [tokens]");
  a.pos = pos.ptr;
  a.pos64 = pos.dtype == C3B_I64;
  a.pos_stride = shared ? 0 : seq;
  a.steps = (const long long*)steps.ptr;
  a.rotary = rotary;
  return C3B_OK;
}

}  // namespace rot

int launch_rotary(const c3b_tensor* in, const c3b_tensor& out, const c3b_rotary_params& p, cudaStream_t s) {
  using namespace rot;
  const c3b_tensor &x = in[0], &pos = in[1], &steps = in[2];
  C3B_REQUIRE(std::isfinite(p.scale), "rotary: the scale is not finite");
  C3B_REQUIRE(is_float(x.dtype) && out.dtype == x.dtype, "rotary: f32, bf16 or fp16, the same in and out");
  C3B_REQUIRE(x.ndim == 4, "rotary: x is [batch, tokens, heads, head_dim]");
  C3B_REQUIRE(numel(out) == numel(x), "rotary: the output is shaped like x");
  C3B_REQUIRE(x.shape[1] < (1ll << 31) && x.shape[2] < (1 << 24) && x.shape[3] <= 65536 &&
                  x.shape[2] * x.shape[3] < (1ll << 31),
              "rotary: extents too large");
  C3B_REQUIRE((x.ptr == out.ptr || !overlaps(x, out)) && !overlaps(pos, out) && !overlaps(steps, out),
              "rotary: x and the output are the same buffer or do not overlap, nor does another input");
  Args a = {};
  a.in = x.ptr;
  a.out[0] = out.ptr;
  a.tokens = x.shape[0] * x.shape[1];
  a.seq = (int)x.shape[1];
  a.heads[0] = (int)x.shape[2];
  a.d = (int)x.shape[3];
  a.out_stride = x.shape[2] * x.shape[3];
  a.interleaved = p.interleaved != 0;
  a.scale = p.scale;
  if (int rc = take_positions(a, pos, steps, x.shape[0], x.shape[1], p.rotary_dim, "rotary")) return rc;
  return run_any(a, x.dtype, s);
}

// in: qkv, [q weight], [k weight], positions, phase steps, [lengths when appending]
int launch_qk_norm_rotary(const c3b_tensor* in, int n_in, const c3b_tensor* out, int n_out, bool append,
                          const c3b_qk_norm_params& p, cudaStream_t s) {
  using namespace rot;
  const char* who = append ? "qk norm rotary append" : "qk norm rotary";
  const std::string w(who);
  const int n_w = (p.has_q_weight ? 1 : 0) + (p.has_k_weight ? 1 : 0);
  C3B_REQUIRE(n_in == 3 + n_w + (append ? 1 : 0) && n_out == (append ? 3 : 1), w + ": wrong number of tensors");
  const c3b_tensor& x = in[0];
  const c3b_tensor &pos = in[1 + n_w], &steps = in[2 + n_w];
  C3B_REQUIRE(p.batch >= 0 && p.seq >= 0 && p.heads >= 0 && p.kv_heads >= 0 && p.head_dim > 0 && p.head_dim <= 65536,
              w + ": bad extents");
  const int64_t width = p.heads + 2ll * p.kv_heads;
  C3B_REQUIRE(p.seq < (1ll << 31) && p.heads < (1 << 24) && p.kv_heads < (1 << 24) && width * p.head_dim < (1ll << 31),
              w + ": extents too large");
  C3B_REQUIRE(is_float(x.dtype), w + ": f32, bf16 or fp16");
  C3B_REQUIRE(numel(x) == p.batch * p.seq * width * p.head_dim, w + ": qkv is [batch, tokens, heads + 2 kv_heads, head_dim]");
  C3B_REQUIRE(std::isfinite(p.scale) && p.epsilon >= 0.f, w + ": the scale is finite, epsilon at least 0");
  C3B_REQUIRE(p.normalize || n_w == 0, w + ": weights without normalisation");
  for (int i = 0; i < n_out; ++i) {
    C3B_REQUIRE(out[i].dtype == x.dtype, w + ": outputs have the type of qkv");
    for (int j = 1; j < n_in; ++j) C3B_REQUIRE(!overlaps(out[i], in[j]), w + ": an output overlaps an input");
  }
  Args a = {};
  a.in = x.ptr;
  a.tokens = p.batch * p.seq;
  a.seq = (int)p.seq;
  a.heads[0] = p.heads;
  a.heads[1] = a.heads[2] = p.kv_heads;
  a.d = p.head_dim;
  a.interleaved = p.interleaved != 0;
  a.normalize = p.normalize != 0;
  a.scale = p.scale;
  a.eps = p.epsilon;
  int at = 1;
  for (int role = 0; role < 2; ++role) {
    if (!(role ? p.has_k_weight : p.has_q_weight)) continue;
    const c3b_tensor& t = in[at++];
    const int64_t each = (int64_t)a.heads[role] * a.d;
    C3B_REQUIRE(t.dtype == C3B_F32 && (numel(t) == a.d || numel(t) == each),
                w + ": norm weights are f32 [head_dim] or [heads, head_dim]");
    a.w[role] = (const float*)t.ptr;
    a.w_stride[role] = numel(t) == a.d ? 0 : a.d;
  }
  if (int rc = take_positions(a, pos, steps, p.batch, p.seq, p.rotary_dim, who)) return rc;
  const size_t es = dtype_size(x.dtype);
  if (!append) {
    C3B_REQUIRE(numel(out[0]) == numel(x), w + ": the output is shaped like qkv");
    C3B_REQUIRE(x.ptr == out[0].ptr || !overlaps(x, out[0]), w + ": qkv and the output are the same buffer or do not overlap");
    a.out_stride = width * p.head_dim;
    a.copy_v = x.ptr != out[0].ptr;  // in place, the values already stand where they belong
    for (int i = 0; i < 3; ++i)
      a.out[i] = (char*)out[0].ptr + (size_t)(i > 0 ? p.heads : 0) * p.head_dim * es +
                 (size_t)(i > 1 ? p.kv_heads : 0) * p.head_dim * es;
    return run_any(a, x.dtype, s);
  }
  const c3b_tensor& lengths = in[3 + n_w];
  C3B_REQUIRE(lengths.dtype == C3B_I32 && numel(lengths) == p.batch, w + ": lengths are int32 [batch]");
  C3B_REQUIRE(p.capacity >= 0 && p.capacity < (1ll << 31), w + ": bad capacity");
  C3B_REQUIRE(numel(out[0]) == a.tokens * p.heads * p.head_dim, w + ": the first output is q [batch, tokens, heads, head_dim]");
  for (int i = 1; i < 3; ++i)
    C3B_REQUIRE(numel(out[i]) == p.batch * p.kv_heads * p.capacity * p.head_dim,
                w + ": caches are [batch, kv_heads, capacity, head_dim]");
  C3B_REQUIRE(!overlaps(out[0], out[1]) && !overlaps(out[0], out[2]) && !overlaps(out[1], out[2]) &&
                  !overlaps(x, out[0]) && !overlaps(x, out[1]) && !overlaps(x, out[2]),
              w + ": qkv, q and the caches do not overlap");
  a.lengths = (const int*)lengths.ptr;
  a.capacity = p.capacity;
  a.out_stride = (int64_t)p.heads * p.head_dim;
  a.copy_v = 1;
  for (int i = 0; i < 3; ++i) a.out[i] = out[i].ptr;
  return run_any(a, x.dtype, s);
}

}  // namespace c3b
