// Rotation of queries and keys by their positions, alone or behind an RMS norm of every head, and the gradients.
//   forward    y = R(pos) (x rstd w),  rstd = rsqrt(mean(x^2) + eps)          (without the norm: y = R(pos) x)
//   backward   g = R(pos)^T dy,  dw = sum g xhat,  dx = rstd (g w - xhat mean(g w xhat)),  xhat = x rstd
// R turns the first `rotary_dim` features pair by pair and multiplies them with a magnitude; the others pass as they are.
//
// Angles.  A frequency is held as a 64-bit fraction of a turn per position, so position times frequency is an integer
// product whose overflow drops whole turns: nothing is lost but what the fraction itself is off by (2^-52 of a frequency that was a
// double: 2^-52 radians a position at most, 10^-7 at 4 * 10^8), where a product in fp32 is off by 0.03 radians at position 10^6.  Sines
// and cosines of the phase are good to 2 * 10^-7 at any position.
// Angles are formed in the kernel: one set per token serves all its heads, so there is no table to build, keep or read.
//
// Work.  A row (one head of one token) belongs to 2^k neighbouring lanes, a lane to `units` of two vectors of W elements, whose
// elements are W pairs (u, v): with the half layout u from one vector and v from the other, else even and odd elements of both.
// A group of lanes goes through up to `per_slot` heads of a token (a slot: heads of the queries or of the keys), kBatch of them in
// flight, two values an instruction.  With the norm, rows come through thread-private places in shared memory, some heads ahead:
// registers go to the factors.
// What bounds it is the traffic: x (and dy) in, y (or dx) out.  bf16: rotation of 65536 x 72 heads of 128 365 us, 6.6 TB/s (the copy's
// rate); with the norm 16383 x 72 of 128 100 us, 6.1 TB/s; its backward for 32768 x 36 of 64 81 us, 5.6 TB/s, half of the issue slots
// busy with 16 warps an SM.

#include "nsa_common.cuh"
#include "nsa_kernels.h"
#include "nsa_sm100_ptx.cuh"

namespace nsa {

namespace heads {

// 128 threads, four blocks an SM: the registers for sixteen values, their factors and four rows under way (256 and two: 65536 x 72 heads
// of 128 368 instead of 365 us, the gradients of 3063 x 10 of 80 36 instead of 27, for their fewer blocks).
constexpr int kThreads = 128, kBlocksPerSM = 4;
// Heads of a slot: angles are formed once for them (8: 16383 x 72 heads of 128 117 us, 32: 102).
constexpr int kMostHeads = 32;
// Few tokens: slots are cut until there are this many blocks for each of the 148 SMs (twelve: 2 x 16384 x 20 heads of 64 86 us, six: 67).
constexpr int kEnoughBlocks = 6;
// Partial weight gradients come from this many blocks for each SM: twice what is resident, so that the last ones even out (four: 161 us
// for 4 x 8192 x 36 heads of 64 with gradients, eight: 152, sixteen: 155).
constexpr int kPartialBlocks = 8;
constexpr int kSMs = 148;
enum { kNone = 0, kShared = 1, kPerHead = 2 };

template <int BYTES> struct RawOf;
template <> struct RawOf<16> { typedef uint4 type; };
template <> struct RawOf<8> { typedef uint2 type; };
template <> struct RawOf<4> { typedef uint32_t type; };
template <> struct RawOf<2> { typedef uint16_t type; };

template <typename T, int W>
struct Vec {
  typedef typename RawOf<W * (int)sizeof(T)>::type Raw;
  __device__ static Raw load(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  __device__ static void widen(const Raw& raw, float* out) {
    const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] = Elem<T>::to_float(v[i]);
  }
  __device__ static void store(T* p, const float* in) {
    Raw raw;
    T* v = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = Elem<T>::from_float(in[i]);
    *reinterpret_cast<Raw*>(p) = raw;
  }
};

// Where a unit's two vectors lie in the row (-1: not there), the frequencies of their first pairs, and whether they are rotated
struct Unit {
  int a, b, freq_a, freq_b;
  bool rot_a, rot_b;
};

template <int W, bool HALF>
__device__ __forceinline__ Unit unit_at(const HeadsParams& P, int u) {
  Unit t;
  if (HALF) {
    const int rot = P.rotary_dim / 2 / W;
    t.rot_a = t.rot_b = u < rot;
    t.a = u < rot ? u * W : P.rotary_dim + 2 * (u - rot) * W;
    t.b = u < rot ? P.rotary_dim / 2 + u * W : t.a + W;
    t.freq_a = t.freq_b = u * W;
  } else if (W == 1) {
    t.a = 2 * u; t.b = 2 * u + 1;
    t.freq_a = t.freq_b = u;
    t.rot_a = t.rot_b = 2 * u < P.rotary_dim;
  } else {             // neighbouring lanes take neighbouring vectors
    t.a = u * W;
    t.b = t.a + (P.d / W + 1) / 2 * W;
    if (t.a >= (P.d / W + 1) / 2 * W) t.a = t.b = P.d;
    t.freq_a = t.a / 2; t.freq_b = t.b / 2;
    t.rot_a = t.a < P.rotary_dim; t.rot_b = t.b < P.rotary_dim;
  }
  if (t.a >= P.d) { t.a = -1; t.rot_a = false; }
  if (t.b >= P.d) { t.b = -1; t.rot_b = HALF && t.rot_a; }
  return t;
}

// The first pairs of a unit lie in its first vector (half layout: all of them in both)
template <int W, bool HALF>
__host__ __device__ constexpr int first_pairs() { return HALF || W == 1 ? W : W / 2; }

template <typename T, int W, bool HALF>
__device__ __forceinline__ void split(const typename Vec<T, W>::Raw& a, const typename Vec<T, W>::Raw& b, float* u, float* v) {
  float x[W], y[W];
  Vec<T, W>::widen(a, x);
  Vec<T, W>::widen(b, y);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (HALF || W == 1) {
      u[i] = x[i]; v[i] = y[i];
    } else {
      u[i] = 2 * i < W ? x[(2 * i) % W] : y[(2 * i) % W];
      v[i] = 2 * i < W ? x[(2 * i + 1) % W] : y[(2 * i + 1) % W];
    }
  }
}
// A unit's weights, of head h where there is a row per head (rows lie on the vectors' boundaries, see vector_width)
template <typename T, int W, bool HALF>
__device__ __forceinline__ void load_weight(const HeadsParams& P, const HeadRows& R, const Unit& t, int h, float* wu, float* wv) {
  const int64_t row = P.weight_per_head ? (int64_t)h * P.d : 0;
  float x[W], y[W];
  auto vector = [&](int at, float* out) {
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] = 0.f;
    if (at < 0) return;
    if (!P.weight_f32) {
      Vec<T, W>::widen(Vec<T, W>::load((const T*)R.weight + row + at), out);
    } else {
      constexpr int F = W < 4 ? W : 4;
#pragma unroll
      for (int i = 0; i < W; i += F) Vec<float, F>::widen(Vec<float, F>::load((const float*)R.weight + row + at + i), out + i);
    }
  };
  vector(t.a, x);
  vector(t.b, y);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    wu[i] = HALF || W == 1 ? x[i] : (2 * i < W ? x[(2 * i) % W] : y[(2 * i) % W]);
    wv[i] = HALF || W == 1 ? y[i] : (2 * i < W ? x[(2 * i + 1) % W] : y[(2 * i + 1) % W]);
  }
}
template <typename T, int W, bool HALF, bool FULL>
__device__ __forceinline__ void store(const Unit& t, T* row, const float* u, const float* v) {
  float x[W], y[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (HALF || W == 1) {
      x[i] = u[i]; y[i] = v[i];
    } else if (2 * i < W) {
      x[(2 * i) % W] = u[i]; x[(2 * i + 1) % W] = v[i];
    } else {
      y[(2 * i) % W] = u[i]; y[(2 * i + 1) % W] = v[i];
    }
  }
  if (FULL || t.a >= 0) Vec<T, W>::store(row + t.a, x);
  if (FULL || t.b >= 0) Vec<T, W>::store(row + t.b, y);
}

// Products and sums over W values, two an instruction (each rounded as a single one)
template <int W>
__device__ __forceinline__ void mul(const float* a, const float* b, float* r) {
  if constexpr (W == 1) r[0] = a[0] * b[0];
  else
#pragma unroll
    for (int i = 0; i < W; i += 2) ptx::unpack2(ptx::mul2(ptx::pack2(a[i], a[i + 1]), ptx::pack2(b[i], b[i + 1])), r[i], r[i + 1]);
}
template <int W>
__device__ __forceinline__ void fma(const float* a, const float* b, const float* c, float* r) {
  if constexpr (W == 1) r[0] = a[0] * b[0] + c[0];
  else
#pragma unroll
    for (int i = 0; i < W; i += 2)
      ptx::unpack2(ptx::fma2(ptx::pack2(a[i], a[i + 1]), ptx::pack2(b[i], b[i + 1]), ptx::pack2(c[i], c[i + 1])), r[i], r[i + 1]);
}
template <int W>
__device__ __forceinline__ void scale(float b, float* r) {
  if constexpr (W == 1) r[0] *= b;
  else
#pragma unroll
    for (int i = 0; i < W; i += 2) ptx::unpack2(ptx::mul2(ptx::pack2(r[i], r[i + 1]), ptx::pack2(b, b)), r[i], r[i + 1]);
}
// r += a b
template <int W>
__device__ __forceinline__ void add_scaled(const float* a, float b, float* r) {
  if constexpr (W == 1) r[0] += a[0] * b;
  else
#pragma unroll
    for (int i = 0; i < W; i += 2) ptx::unpack2(ptx::fma2(ptx::pack2(a[i], a[i + 1]), ptx::pack2(b, b), ptx::pack2(r[i], r[i + 1])), r[i], r[i + 1]);
}
// sum += a b, even and odd places apart
template <int W>
__device__ __forceinline__ void add_dot(const float* a, const float* b, float (&sum)[2]) {
  if constexpr (W == 1) sum[0] += a[0] * b[0];
  else
#pragma unroll
    for (int i = 0; i < W; i += 2)
      ptx::unpack2(ptx::fma2(ptx::pack2(a[i], a[i + 1]), ptx::pack2(b[i], b[i + 1]), ptx::pack2(sum[0], sum[1])), sum[0], sum[1]);
}

// (u, v) -> (u cu + v cv, v dv + u du): N pairs
template <int N>
__device__ __forceinline__ void rotate(float* u, float* v, const float* cu, const float* cv, const float* dv, const float* du) {
  float a[N], b[N];
  mul<N>(v, cv, a);
  mul<N>(u, du, b);
  fma<N>(u, cu, a, u);
  fma<N>(v, dv, b, v);
}

// Sine and cosine of a phase, 2^64 to the turn.  The nearest quarter turn is taken off in integers; what is left, at most pi / 4, goes
// into the Taylor series up to x^9 and x^8, whose next terms are below 2e-9 and 2.5e-8 (half a unit of a cosine above 0.7 is 3e-8).
// Its 30 bits as fp32 are off by 2^-25 of pi / 4 at most.
__device__ __forceinline__ void sine_cosine(uint64_t phase, float& si, float& co) {
  const uint32_t top = (uint32_t)((phase + 0x80000000ull) >> 32), quarter = (top + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(top - (quarter << 30)) * 1.4629180792671596e-9f;      // 2 pi / 2^32
  const float y = x * x;
  const float s = x + x * y * (-1.f / 6 + y * (1.f / 120 + y * (-1.f / 5040 + y * (1.f / 362880))));
  const float c = 1.f + y * (-0.5f + y * (1.f / 24 + y * (-1.f / 720 + y * (1.f / 40320))));
  si = __uint_as_float(__float_as_uint(quarter & 1 ? c : s) ^ (quarter & 2) << 30);
  co = __uint_as_float(__float_as_uint(quarter & 1 ? s : c) ^ ((quarter + 1) & 2) << 30);
}

// Sum over the lanes of a row
__device__ __forceinline__ float row_sum(float v, int lanes) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
    if (o < lanes) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}

}  // namespace heads

// W: elements of a vector; UPL: units of a lane; HALF: the layout
// WEIGHTS: kNone (no norm), kShared, kPerHead
// FULL: every lane has both vectors of every unit
template <typename T, int W, int UPL, bool HALF, int WEIGHTS, bool BWD, bool FULL>
__global__ void __launch_bounds__(heads::kThreads, heads::kBlocksPerSM) heads_kernel(const HeadsParams P) {
  using namespace heads;
  using V = Vec<T, W>;
  typedef typename V::Raw Raw;
  constexpr bool NORM = WEIGHTS != kNone;
  constexpr bool XIN = !BWD || NORM;                              // x is read
  constexpr bool FOLD = WEIGHTS == kShared && !BWD;               // the weights are part of the rotation's factors
  constexpr bool ONE = WEIGHTS == kPerHead && BWD;                // one head a slot, whose weight gradient stays in registers
  constexpr bool RING = FULL && NORM;                             // rows come through shared memory
  constexpr int kVecs = BWD ? 4 : 2, kStages = RING ? (BWD ? 3 : 5) : 1;     // (three forward: 111 us for 16383 x 72 heads of 128, five: 103)
  constexpr int kBatch = UPL > 1 || RING || (BWD && NORM) ? 1 : 4;     // heads in flight, in registers (two for 65536 x 72 of 128: 390 us, four: 369)
  constexpr int FIRST = first_pairs<W, HALF>();
  __shared__ float fold[NORM && BWD ? kThreads / 32 : 1][NORM && BWD ? kHeadsMaxDim : 1];
  __shared__ __align__(16) float held[NORM && BWD ? 32 * UPL : 1][NORM && BWD ? 2 * W : 1];   // the backward's weights, unit by unit

  // every thread's own places: 16 bytes of each vector of kStages rows
  __shared__ __align__(16) uint4 places[RING ? kStages * kVecs * kThreads : 1];

  ptx::grid_allow_next();
  const int lanes = 1 << P.lane_shift, lane = threadIdx.x & (lanes - 1);
  const int group = threadIdx.x >> P.lane_shift, groups = kThreads >> P.lane_shift;
  // blocks of the queries' slots, then of the keys'
  const bool keys = (int)blockIdx.x >= P.slots[0] * P.blocks[0];
  const HeadRows& R = P.part[keys];
  const int block = (int)blockIdx.x - (keys ? P.slots[0] * P.blocks[0] : 0), blocks = P.blocks[keys];
  const int slot = block / blocks, at_block = block - slot * blocks;
  const int h0 = slot * P.per_slot, h1 = min(R.heads, h0 + P.per_slot);

  Unit unit[UPL];
  float wu[FOLD ? UPL : 1][W], wv[FOLD ? UPL : 1][W], acc_u[UPL][W], acc_v[UPL][W];
#pragma unroll
  for (int k = 0; k < UPL; ++k) {
    unit[k] = unit_at<W, HALF>(P, lane + k * lanes);
    if (FOLD) load_weight<T, W, HALF>(P, R, unit[k], 0, wu[FOLD ? k : 0], wv[FOLD ? k : 0]);
    if (NORM && BWD) {
      if (group == 0) load_weight<T, W, HALF>(P, R, unit[k], h0, held[lane + k * lanes], held[lane + k * lanes] + W);
#pragma unroll
      for (int i = 0; i < W; ++i) acc_u[k][i] = acc_v[k][i] = 0.f;
    }
  }
  if (NORM && BWD) __syncthreads();

  const unsigned tokens = (unsigned)P.batch * (unsigned)P.seq;
  const float inv_d = 1.f / (float)P.d;
  const unsigned step = (unsigned)blocks * groups, begin = (unsigned)at_block * groups;
  auto position = [&](unsigned token) {
    const unsigned b = token / (unsigned)P.seq, n = token - b * (unsigned)P.seq;
    if (P.positions == nullptr) return P.offset + n;
    const int64_t at = (int64_t)b * P.pos_sb + n;
    return P.offset + (P.pos_i64 ? ((const int64_t*)P.positions)[at] : (int64_t)((const int32_t*)P.positions)[at]);
  };
  auto row_at = [&](const void* base, int64_t sb, int64_t sh, int64_t sn, unsigned token) {     // the slot's first head
    const unsigned b = token / (unsigned)P.seq, n = token - b * (unsigned)P.seq;
    return (T*)base + (int64_t)b * sb + (int64_t)n * sn + (int64_t)h0 * sh;
  };

  // RING: rows are on their way kStages - 1 heads ahead, past the end of a token into the next one
  const uint32_t place = ptx::smem_u32(places + threadIdx.x);
  unsigned far_token = begin + group;
  int far_head = h0, far_stage = 0, stage = 0;
  const T *far_x = nullptr, *far_g = nullptr;
  auto far_locate = [&]() {
    if (far_token >= tokens) return;
    far_x = row_at(R.x, R.x_sb, R.x_sh, R.x_sn, far_token);
    if (BWD) far_g = row_at(R.dy, R.dy_sb, R.dy_sh, R.dy_sn, far_token);
  };
  auto far_fetch = [&]() {
    if (far_token < tokens) {
      const uint32_t at = place + far_stage * (kVecs * kThreads * 16);
      ptx::cp_async16(at, far_x + unit[0].a, 16);
      ptx::cp_async16(at + kThreads * 16, far_x + unit[0].b, 16);
      if (BWD) {
        ptx::cp_async16(at + 2 * kThreads * 16, far_g + unit[0].a, 16);
        ptx::cp_async16(at + 3 * kThreads * 16, far_g + unit[0].b, 16);
      }
    }
    ptx::cp_async_commit();
    far_stage = far_stage + 1 == kStages ? 0 : far_stage + 1;
    if (++far_head < h1) {
      far_x += R.x_sh;
      if (BWD) far_g += R.dy_sh;
    } else {
      far_head = h0;
      far_token += step;
      far_locate();
    }
  };
  if (RING) {
    far_locate();
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) far_fetch();
  }
  int64_t next_pos = position(min(begin + group, tokens - 1));

  // every lane of a warp takes part in the sums over a row: groups without a token go along with nothing to load
  for (unsigned first = begin; first < tokens; first += step) {
    const unsigned token = first + group;
    const bool live = token < tokens;
    const T* xp = XIN && !RING ? row_at(R.x, R.x_sb, R.x_sh, R.x_sn, live ? token : 0) : nullptr;
    const T* gp = BWD && !RING ? row_at(R.dy, R.dy_sb, R.dy_sh, R.dy_sn, live ? token : 0) : nullptr;
    T* op = row_at(R.out, R.o_sb, R.o_sh, R.o_sn, live ? token : 0);
    Raw xr[kBatch][UPL][2], gr[BWD ? kBatch : 1][UPL][2];
    // the next head's values into place j; beyond the slot's heads (and, with FULL, for groups without a token) those of the last
    // one, of which nothing is kept
    int ahead = h0;
    auto fetch = [&](int j) {
#pragma unroll
      for (int k = 0; k < UPL; ++k) {
        const bool a = FULL || (live && unit[k].a >= 0), b = FULL || (live && unit[k].b >= 0);
        if (XIN) {
          xr[j][k][0] = a ? V::load(xp + unit[k].a) : Raw{};
          xr[j][k][1] = b ? V::load(xp + unit[k].b) : Raw{};
        }
        if (BWD) {
          gr[j][k][0] = a ? V::load(gp + unit[k].a) : Raw{};
          gr[j][k][1] = b ? V::load(gp + unit[k].b) : Raw{};
        }
      }
      if (++ahead < h1) {
        if (XIN) xp += R.x_sh;
        if (BWD) gp += R.dy_sh;
      }
    };
    if (!RING)
#pragma unroll
      for (int j = 0; j < kBatch; ++j) fetch(j);               // under way while the angles are formed
    const int64_t pos = next_pos;
    if (first + step < tokens) next_pos = position(min(token + step, tokens - 1));
    // factors of the rotation: u' = u cu + v cv, v' = v dv + u du, with the weights in them (FOLD; else dv = cu)
    float cu[UPL][W], cv[UPL][W], dv[FOLD ? UPL : 1][W], du[UPL][W];
#pragma unroll
    for (int k = 0; k < UPL; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float co = 1.f, si = 0.f;
        if (i < FIRST ? unit[k].rot_a : unit[k].rot_b) {
          sine_cosine((uint64_t)pos * __ldg(P.steps + (i < FIRST ? unit[k].freq_a + i : unit[k].freq_b + i - FIRST)), si, co);
          co *= P.magnitude;
          si *= BWD ? -P.magnitude : P.magnitude;
        }
        cu[k][i] = co; cv[k][i] = -si; du[k][i] = si;
        if (FOLD) {
          const int f = FOLD ? k : 0;
          dv[f][i] = wv[f][i] * co;
          cu[k][i] *= wu[f][i]; cv[k][i] *= wv[f][i]; du[k][i] *= wu[f][i];
        }
      }
    for (int h = h0; h < h1; h += kBatch) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const bool ok = live && h + j < h1;
        float u[UPL][W], v[UPL][W], gu[BWD ? UPL : 1][W], gv[BWD ? UPL : 1][W];          // x, dy; then what is stored
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
          if constexpr (RING) {
            ptx::cp_async_wait<kStages - 2>();
            const uint32_t at = place + stage * (kVecs * kThreads * 16);
            uint4 raw[kVecs];
#pragma unroll
            for (int i = 0; i < kVecs; ++i) raw[i] = ptx::lds_v4(at + i * (kThreads * 16));
            split<T, W, HALF>(reinterpret_cast<const Raw&>(raw[0]), reinterpret_cast<const Raw&>(raw[1]), u[k], v[k]);
            if (BWD) split<T, W, HALF>(reinterpret_cast<const Raw&>(raw[kVecs - 2]), reinterpret_cast<const Raw&>(raw[kVecs - 1]), gu[k], gv[k]);
            stage = stage + 1 == kStages ? 0 : stage + 1;
          } else {
            if (XIN) split<T, W, HALF>(xr[j][k][0], xr[j][k][1], u[k], v[k]);
            if (BWD) split<T, W, HALF>(gr[j][k][0], gr[j][k][1], gu[k], gv[k]);
          }
        }
        // the place is free: the next head's values are on their way meanwhile
        if (RING) far_fetch();
        else if (!ONE) fetch(j);
        float rstd = 1.f;
        if (NORM) {
          float ss[2] = {0.f, 0.f};
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
            add_dot<W>(u[k], u[k], ss);
            add_dot<W>(v[k], v[k], ss);
          }
          rstd = rsqrtf(row_sum(ss[0] + ss[1], lanes) * inv_d + P.eps);
        }
        auto turn = [&](int k, float* p, float* q) {
          const float* d = FOLD ? dv[FOLD ? k : 0] : cu[k];
          if (unit[k].rot_a && unit[k].rot_b) rotate<W>(p, q, cu[k], cv[k], d, du[k]);
          else {                             // a pair that is not rotated must not be multiplied with the other's zero
            if (unit[k].rot_a) rotate<FIRST>(p, q, cu[k], cv[k], d, du[k]);
            if constexpr (FIRST < W) {
              if (unit[k].rot_b) rotate<W - FIRST>(p + FIRST, q + FIRST, cu[k] + FIRST, cv[k] + FIRST, d + FIRST, du[k] + FIRST);
            }
            if (FOLD)
#pragma unroll
              for (int i = 0; i < W; ++i)
                if (!(i < FIRST ? unit[k].rot_a : unit[k].rot_b)) { p[i] *= cu[k][i]; q[i] *= d[i]; }
          }
        };
        if (!BWD) {
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
            if (NORM) {
              scale<W>(rstd, u[k]);
              scale<W>(rstd, v[k]);
            }
            if (WEIGHTS == kPerHead) {
              float pu[W], pv[W];
              load_weight<T, W, HALF>(P, R, unit[k], min(h + j, h1 - 1), pu, pv);
              mul<W>(u[k], pu, u[k]);
              mul<W>(v[k], pv, v[k]);
            }
            turn(k, u[k], v[k]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < UPL; ++k) turn(k, gu[k], gv[k]);
          if (NORM) {
            // g rstd in place of g: dw += g x, dx = g w - x rstd^2 mean(g w x)
            float dot[2] = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < UPL; ++k) {
              const float* w = held[lane + k * lanes];
              scale<W>(rstd, gu[k]);
              scale<W>(rstd, gv[k]);
              if (ok) {
                fma<W>(gu[k], u[k], acc_u[k], acc_u[k]);
                fma<W>(gv[k], v[k], acc_v[k], acc_v[k]);
              }
              mul<W>(gu[k], w, gu[k]);
              mul<W>(gv[k], w + W, gv[k]);
              add_dot<W>(gu[k], u[k], dot);
              add_dot<W>(gv[k], v[k], dot);
            }
            const float c = -rstd * rstd * (row_sum(dot[0] + dot[1], lanes) * inv_d);
#pragma unroll
            for (int k = 0; k < UPL; ++k) {
              add_scaled<W>(u[k], c, gu[k]);
              add_scaled<W>(v[k], c, gv[k]);
            }
          }
        }
        if (ok) {
#pragma unroll
          for (int k = 0; k < UPL; ++k) store<T, W, HALF, FULL>(unit[k], op, BWD ? gu[k] : u[k], BWD ? gv[k] : v[k]);
          op += R.o_sh;
        }
      }
    }
  }

  if (NORM && BWD) {
    // the weight gradient of this block's rows: groups of a warp by shuffles, warps through shared memory, in a fixed order
    const int wib = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < UPL; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float su = acc_u[k][i], sv = acc_v[k][i];
        for (int o = 16; o >= lanes; o >>= 1) {
          su += __shfl_xor_sync(kFullMask, su, o);
          sv += __shfl_xor_sync(kFullMask, sv, o);
        }
        int eu = unit[k].a + i, ev = unit[k].b + i;
        if (!HALF && W > 1) {
          eu = i < FIRST ? unit[k].a + 2 * i : unit[k].b + 2 * (i - FIRST);
          ev = eu + 1;
        }
        const bool has_u = (HALF || i < FIRST ? unit[k].a : unit[k].b) >= 0, has_v = (!HALF && W > 1 ? has_u : unit[k].b >= 0);
        if ((threadIdx.x & 31) < lanes) {
          if (has_u) fold[wib][eu] = su;
          if (has_v) fold[wib][ev] = sv;
        }
      }
    __syncthreads();
    float* partial = P.partial + (int64_t)blockIdx.x * P.d;
    for (int e = threadIdx.x; e < P.d; e += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k) s += fold[k][e];
      partial[e] = s;
    }
  }
}

// dw of a weight row: the sum of its slots' partials over their blocks, in a fixed order.  blockIdx.y: the weight row (queries'
// rows first); eight elements a block, 128 threads an element: the thousand partials of a row are nine loads deep (1155 partials of
// 64 and 64 elements: 7.8 us with 32 elements a block).
template <typename T>
__global__ void __launch_bounds__(1024) heads_dweight_kernel(const HeadsParams P) {
  __shared__ float fold[8][129];
  const int rows_q = P.weight_per_head ? P.part[0].heads : (P.part[0].heads > 0 ? 1 : 0);
  const bool keys = (int)blockIdx.y >= rows_q;
  const int row = (int)blockIdx.y - (keys ? rows_q : 0), blocks = P.blocks[keys];
  const int64_t first = (keys ? (int64_t)P.slots[0] * P.blocks[0] : 0) + (P.weight_per_head ? (int64_t)row * blocks : 0);
  const int count = (P.weight_per_head ? 1 : P.slots[keys]) * blocks;
  const int e = blockIdx.x * 8 + (threadIdx.x & 7), part = threadIdx.x >> 3;
  float s = 0.f;
  ptx::grid_wait();
  if (e < P.d) {
    const float* src = P.partial + first * P.d + e;
#pragma unroll 10
    for (int r = part; r < count; r += 128) s += src[(int64_t)r * P.d];
  }
  fold[threadIdx.x & 7][part] = s;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, out = blockIdx.x * 8 + warp;
  if (warp >= 8) return;
  s = warp_sum((fold[warp][lane] + fold[warp][lane + 32]) + (fold[warp][lane + 64] + fold[warp][lane + 96]));
  if (lane == 0 && out < P.d) {
    void* dw = P.part[keys].dweight;
    const int64_t at = (int64_t)row * P.d + out;
    if (P.weight_f32) ((float*)dw)[at] = s;
    else ((T*)dw)[at] = Elem<T>::from_float(s);
  }
}

// Widest vector that every row's start, the row length and the rotated part allow
static int vector_width(const HeadsParams& P, int size, bool backward) {
  uint64_t all = (uint64_t)16 | (uint64_t)P.d * size;
  all |= (uint64_t)(P.half ? P.rotary_dim / 2 : P.rotary_dim) * size;
  for (const HeadRows& r : P.part) {
    if (r.heads == 0) continue;
    all |= reinterpret_cast<uintptr_t>(r.out) | (uint64_t)(r.o_sb | r.o_sh | r.o_sn) * size;
    if (P.norm) {        // fp32 weights are read four at a time beside bf16 rows
      const uintptr_t at = reinterpret_cast<uintptr_t>(r.weight) & 15;
      all |= P.weight_f32 && size == 2 ? (at & 4 ? 2 : at & 8 ? 4 : 0) : at;
    }
    if (r.x != nullptr) all |= reinterpret_cast<uintptr_t>(r.x) | (uint64_t)(r.x_sb | r.x_sh | r.x_sn) * size;
    if (backward) all |= reinterpret_cast<uintptr_t>(r.dy) | (uint64_t)(r.dy_sb | r.dy_sh | r.dy_sn) * size;
  }
  const uint64_t bytes = all & (~all + 1);
  return (int)(bytes / size);
}

// Heads a slot, and blocks over the tokens for the slots of the queries and of the keys.  `one`: a head a slot.
static int heads_grid(HeadsParams& P, bool persistent, bool one, int groups) {
  using namespace heads;
  const int64_t all = ((int64_t)P.batch * P.seq + groups - 1) / groups;
  int per = one ? 1 : kMostHeads;
  auto slots = [&](int p) { return (int64_t)(P.part[0].heads + p - 1) / p + (P.part[1].heads + p - 1) / p; };
  // one set of angles serves a slot's heads; few tokens: heads go to blocks of their own until every SM has several
  while (per > 1 && all * slots(per) < (persistent ? kPartialBlocks : kEnoughBlocks) * kSMs) per /= 2;
  int64_t total = 0;
  for (int i = 0; i < 2; ++i) {
    P.slots[i] = (P.part[i].heads + per - 1) / per;
    // with partial weight gradients a set number of blocks, by the parts' share of the heads
    const int64_t share = (int64_t)kPartialBlocks * kSMs * P.part[i].heads / (P.part[0].heads + P.part[1].heads);
    const int64_t most = P.slots[i] > 0 ? (share + P.slots[i] - 1) / P.slots[i] : 1;
    const int64_t blocks = persistent && all > most ? (most > 0 ? most : 1) : all;
    if (blocks > 0x7fffffffLL) return fail(NSA_ERR_SHAPE, "heads: too many tokens for one launch");
    P.blocks[i] = (int)blocks;
    total += blocks * P.slots[i];
  }
  P.per_slot = per;
  if (total > 0x7fffffffLL) return fail(NSA_ERR_SHAPE, "heads: too many heads and tokens for one launch");
  return NSA_OK;
}

static int lane_shift(const HeadsParams& P, int W, int* units_per_lane) {
  const int units = P.half ? P.rotary_dim / 2 / W + ((P.d - P.rotary_dim) / W + 1) / 2 : (P.d + 2 * W - 1) / (2 * W);
  int shift = 0;
  while ((1 << shift) < units && shift < 5) ++shift;
  *units_per_lane = (units + (1 << shift) - 1) >> shift;
  return shift;
}

int64_t heads_partial_floats(const HeadsParams& P0) {
  if (!P0.norm) return 0;
  // blocks: the share of each part, rounded up once for each slot
  return (heads::kPartialBlocks * heads::kSMs + 2 * ((int64_t)P0.part[0].heads + P0.part[1].heads)) * P0.d;
}

template <typename T, int W, int UPL, int WEIGHTS, bool BWD>
static int launch_heads_w(HeadsParams& P, cudaStream_t stream) {
  using heads::kNone;
  int units = 0;
  P.lane_shift = lane_shift(P, W, &units);
  if (units > UPL) return fail(NSA_ERR_UNSUPPORTED, "heads: dim_head is too large for rows that lie on such boundaries");
  constexpr bool partials = WEIGHTS != kNone && BWD;
  const int rc = heads_grid(P, partials, partials && WEIGHTS == heads::kPerHead, heads::kThreads >> P.lane_shift);
  if (rc != NSA_OK) return rc;
  const unsigned grid = (unsigned)(P.slots[0] * P.blocks[0] + P.slots[1] * P.blocks[1]);
  const int rows = P.weight_per_head ? P.part[0].heads + P.part[1].heads : (P.part[0].heads > 0) + (P.part[1].heads > 0);
  if (partials && rows > 65535) return fail(NSA_ERR_SHAPE, "heads: more than 65535 weight rows");
  const bool full = W * (int)sizeof(T) == 16 && P.d == (2 * W << P.lane_shift);      // the usual heads, in the widest vectors
  constexpr bool wide = W * sizeof(T) == 16;
  if (full && P.half) heads_kernel<T, W, UPL, true, WEIGHTS, BWD, wide><<<grid, heads::kThreads, 0, stream>>>(P);
  else if (full) heads_kernel<T, W, UPL, false, WEIGHTS, BWD, wide><<<grid, heads::kThreads, 0, stream>>>(P);
  else if (P.half) heads_kernel<T, W, UPL, true, WEIGHTS, BWD, false><<<grid, heads::kThreads, 0, stream>>>(P);
  else heads_kernel<T, W, UPL, false, WEIGHTS, BWD, false><<<grid, heads::kThreads, 0, stream>>>(P);
  cudaError_t err = cudaGetLastError();
  if (partials && err == cudaSuccess) {
    cudaLaunchConfig_t config = {};      // starts while the last blocks of the kernel before it are at work
    config.gridDim = dim3((unsigned)(P.d + 7) / 8, (unsigned)rows);
    config.blockDim = dim3(1024);
    config.stream = stream;
    cudaLaunchAttribute overlap = {};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &overlap;
    config.numAttrs = 1;
    err = cudaLaunchKernelEx(&config, heads_dweight_kernel<T>, P);
  }
  if (err != cudaSuccess) return fail((int)err, cudaGetErrorString(err));
  count_launches(partials ? 2 : 1);
  return NSA_OK;
}

template <typename T, int WEIGHTS, bool BWD>
static int launch_heads_typed(HeadsParams& P, cudaStream_t stream) {
  constexpr int kMost = 16 / (int)sizeof(T);
  const int W = vector_width(P, sizeof(T), BWD);
  if (W >= kMost) return launch_heads_w<T, kMost, 1, WEIGHTS, BWD>(P, stream);
  if (W >= kMost / 2) return launch_heads_w<T, kMost / 2, kMost / 2 >= 4 ? 1 : 2, WEIGHTS, BWD>(P, stream);
  if (kMost / 4 > 1 && W >= kMost / 4) return launch_heads_w<T, kMost / 4 < 2 ? 2 : kMost / 4, 2, WEIGHTS, BWD>(P, stream);
  return launch_heads_w<T, 1, 4, WEIGHTS, BWD>(P, stream);
}

template <typename T>
static int launch_heads_dir(HeadsParams& P, bool backward, cudaStream_t stream) {
  using namespace heads;
  if (!P.norm) return backward ? launch_heads_typed<T, kNone, true>(P, stream) : launch_heads_typed<T, kNone, false>(P, stream);
  if (!P.weight_per_head) return backward ? launch_heads_typed<T, kShared, true>(P, stream) : launch_heads_typed<T, kShared, false>(P, stream);
  return backward ? launch_heads_typed<T, kPerHead, true>(P, stream) : launch_heads_typed<T, kPerHead, false>(P, stream);
}

int launch_heads(HeadsParams& P, int dtype, bool backward, cudaStream_t stream) {
  if ((int64_t)P.batch * P.seq == 0) {
    if (!backward || !P.norm) return NSA_OK;
    for (const HeadRows& r : P.part) {
      if (r.heads == 0) continue;
      const size_t size = (size_t)(P.weight_per_head ? r.heads : 1) * P.d * (P.weight_f32 || dtype == NSA_F32 ? 4 : 2);
      const cudaError_t err = cudaMemsetAsync(r.dweight, 0, size, stream);
      if (err != cudaSuccess) return fail((int)err, cudaGetErrorString(err));
    }
    return NSA_OK;
  }
  return dtype == NSA_F32 ? launch_heads_dir<float>(P, backward, stream) : launch_heads_dir<__nv_bfloat16>(P, backward, stream);
}

}  // namespace nsa
