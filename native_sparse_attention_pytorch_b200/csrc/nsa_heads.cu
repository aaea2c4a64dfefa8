// Rotation of queries and keys by their positions, alone or behind an RMS norm of every head, and the gradients.
//   forward    y = R(pos) (x rstd w),  rstd = rsqrt(mean(x^2) + eps)          (without the norm: y = R(pos) x)
//   backward   g = R(pos)^T dy,  dw = sum g xhat,  dx = rstd (g w - xhat mean(g w xhat)),  xhat = x rstd
// R turns the first `rotary_dim` features pair by pair and multiplies them with a magnitude; the others pass as they are.
//
// Angles.  A frequency is held as a 64-bit fraction of a turn per position, so position times frequency is an integer
// product whose overflow drops whole turns: the phase is exact to pos * 2^-65 turns, where a product in fp32 is off by 0.03
// radians at position 10^6.  Its upper 32 bits, as fp32 in [-1, 1) half turns, go to sincospif: 10^-7 in the end.
// Angles are formed in the kernel: one set per token serves all its heads, so there is no table to build, keep or read.
//
// Work.  A row (one head of one token) belongs to 2^k neighbouring lanes, a lane to `units` of two vectors of W elements:
// with the half layout the two vectors whose elements form pairs, else two neighbouring vectors.  A group of lanes goes
// through up to `per_slot` heads of a token (a slot: heads of the queries or of the keys), kBatch of them in flight.
// What bounds it is the traffic: x (and dy) in, y (or dx) out.

#include "nsa_common.cuh"
#include "nsa_kernels.h"
#include "nsa_sm100_ptx.cuh"

namespace nsa {

namespace heads {

constexpr int kThreads = 256;

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

// Where a unit's two vectors lie in the row (-1: not there), and which of its W pairs are rotated by which frequencies
struct Unit {
  int a, b;        // first elements
  int freq;        // frequency of the first pair
  int pairs;       // rotated pairs
};

template <int W>
__device__ __forceinline__ Unit unit_at(const HeadsParams& P, int u) {
  Unit t;
  if (P.half) {
    const int rot = P.rotary_dim / 2 / W;
    if (u < rot) {
      t.a = u * W; t.b = P.rotary_dim / 2 + u * W; t.freq = u * W; t.pairs = W;
      return t;
    }
    t.a = P.rotary_dim + 2 * (u - rot) * W; t.freq = 0; t.pairs = 0;
  } else {
    t.a = 2 * u * W; t.freq = u * W;
    t.pairs = max(0, min(W, P.rotary_dim / 2 - u * W));
  }
  t.b = t.a + W < P.d ? t.a + W : -1;
  if (t.a >= P.d) t.a = -1;
  return t;
}

// The rotation of a unit's values, a and b; sine negated for the way back
template <int W>
__device__ __forceinline__ void turn(bool half, int pairs, const float* co, const float* si, float* a, float* b) {
#pragma unroll
  for (int i = 0; i < W; ++i) {
    // half (and single elements): a[i] with b[i]; else neighbours inside the 2 W elements of a, b
    float* x = (half || W == 1) ? a + i : (2 * i < W ? a + 2 * i : b + 2 * i - W);
    float* z = (half || W == 1) ? b + i : x + 1;
    if (i < pairs) {
      const float x0 = *x, z0 = *z;
      *x = x0 * co[i] - z0 * si[i];
      *z = z0 * co[i] + x0 * si[i];
    }
  }
}

}  // namespace heads

// W: elements of a vector; UPL: units of a lane; HALF: the layout
template <typename T, int W, int UPL, bool HALF, bool NORM, bool BWD>
__global__ void __launch_bounds__(heads::kThreads, 2) heads_kernel(const HeadsParams P) {
  using namespace heads;
  using V = Vec<T, W>;
  typedef typename V::Raw Raw;
  constexpr bool XIN = !BWD || NORM;                 // x is read
  constexpr int kBatch = UPL > 1 ? 1 : (BWD && NORM ? 2 : 4);   // heads in flight
  __shared__ float fold[NORM && BWD ? kThreads / 32 : 1][NORM && BWD ? kHeadsMaxDim : 1];

  const int lanes = 1 << P.lane_shift, lane = threadIdx.x & (lanes - 1);
  const int group = threadIdx.x >> P.lane_shift, groups = kThreads >> P.lane_shift;
  const bool keys = (int)blockIdx.y >= P.slots[0];
  const HeadRows& R = P.part[keys];
  const int slot = (int)blockIdx.y - (keys ? P.slots[0] : 0);
  const int h0 = slot * P.per_slot, h1 = min(R.heads, h0 + P.per_slot);

  Unit unit[UPL];
  float w[UPL][2 * W], acc[UPL][2 * W];
#pragma unroll
  for (int k = 0; k < UPL; ++k) {
    unit[k] = unit_at<W>(P, lane + k * lanes);
    if (NORM) {
      const int64_t row = P.weight_per_head ? (int64_t)h0 * P.d : 0;    // per head: one head a slot
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int ea = unit[k].a + i, eb = unit[k].b + i;
        w[k][i] = unit[k].a < 0 ? 0.f : P.weight_f32 ? ((const float*)R.weight)[row + ea] : Elem<T>::to_float(((const T*)R.weight)[row + ea]);
        w[k][W + i] = unit[k].b < 0 ? 0.f : P.weight_f32 ? ((const float*)R.weight)[row + eb] : Elem<T>::to_float(((const T*)R.weight)[row + eb]);
        acc[k][i] = acc[k][W + i] = 0.f;
      }
    }
  }

  const unsigned tokens = (unsigned)P.batch * (unsigned)P.seq;
  const float inv_d = 1.f / (float)P.d;
  // every lane of a warp takes part in the sums over a row: groups without a token go along with nothing to load
  for (unsigned first = blockIdx.x * groups; first < tokens; first += gridDim.x * groups) {
    const unsigned token = first + group;
    const bool live = token < tokens;
    const unsigned b = live ? token / (unsigned)P.seq : 0, n = live ? token - b * (unsigned)P.seq : 0;
    int64_t pos = P.offset + n;
    if (P.positions != nullptr) {
      const int64_t at = (int64_t)b * P.pos_sb + n;
      pos = P.offset + (P.pos_i64 ? ((const int64_t*)P.positions)[at] : (int64_t)((const int32_t*)P.positions)[at]);
    }
    float co[UPL][W], si[UPL][W];
#pragma unroll
    for (int k = 0; k < UPL; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i) {
        co[k][i] = 1.f; si[k][i] = 0.f;
        if (i < unit[k].pairs) {
          const uint64_t phase = (uint64_t)pos * __ldg(P.steps + unit[k].freq + i);
          const int32_t top = (int32_t)((phase + 0x80000000ull) >> 32);
          sincospif((float)top * 4.656612873077393e-10f, &si[k][i], &co[k][i]);    // 2^-31: a turn is two half turns
          co[k][i] *= P.magnitude;
          si[k][i] *= BWD ? -P.magnitude : P.magnitude;
        }
      }
    const T* xp = XIN ? (const T*)R.x + (int64_t)b * R.x_sb + (int64_t)n * R.x_sn : nullptr;
    const T* gp = BWD ? (const T*)R.dy + (int64_t)b * R.dy_sb + (int64_t)n * R.dy_sn : nullptr;
    T* op = (T*)R.out + (int64_t)b * R.o_sb + (int64_t)n * R.o_sn;
    for (int h = h0; h < h1; h += kBatch) {
      Raw xr[kBatch][UPL][2], gr[BWD ? kBatch : 1][UPL][2];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
          const bool ok = live && h + j < h1;
          if (XIN) {
            xr[j][k][0] = ok && unit[k].a >= 0 ? V::load(xp + (h + j) * R.x_sh + unit[k].a) : Raw{};
            xr[j][k][1] = ok && unit[k].b >= 0 ? V::load(xp + (h + j) * R.x_sh + unit[k].b) : Raw{};
          }
          if (BWD) {
            gr[j][k][0] = ok && unit[k].a >= 0 ? V::load(gp + (h + j) * R.dy_sh + unit[k].a) : Raw{};
            gr[j][k][1] = ok && unit[k].b >= 0 ? V::load(gp + (h + j) * R.dy_sh + unit[k].b) : Raw{};
          }
        }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const bool ok = live && h + j < h1;
        float x[UPL][2 * W], g[UPL][2 * W];
        float rstd = 1.f, c = 0.f;
        if (NORM) {
          float ss = 0.f;
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
            V::widen(xr[j][k][0], x[k]);
            V::widen(xr[j][k][1], x[k] + W);
#pragma unroll
            for (int i = 0; i < 2 * W; ++i) ss += x[k][i] * x[k][i];
          }
          for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(kFullMask, ss, o);
          rstd = rsqrtf(ss * inv_d + P.eps);
        } else if (!BWD) {
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
            V::widen(xr[j][k][0], x[k]);
            V::widen(xr[j][k][1], x[k] + W);
          }
        }
        if (BWD) {
          float dot = 0.f;
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
            V::widen(gr[j][k][0], g[k]);
            V::widen(gr[j][k][1], g[k] + W);
            turn<W>(HALF, unit[k].pairs, co[k], si[k], g[k], g[k] + W);
            if (NORM) {
#pragma unroll
              for (int i = 0; i < 2 * W; ++i) {
                const float xh = x[k][i] * rstd;
                if (ok) acc[k][i] += g[k][i] * xh;
                g[k][i] *= w[k][i];
                dot += g[k][i] * xh;
                x[k][i] = xh;
              }
            }
          }
          if (NORM) {
            for (int o = lanes >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(kFullMask, dot, o);
            c = dot * inv_d;
#pragma unroll
            for (int k = 0; k < UPL; ++k)
#pragma unroll
              for (int i = 0; i < 2 * W; ++i) g[k][i] = rstd * (g[k][i] - x[k][i] * c);
          }
        } else {
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
            if (NORM) {
#pragma unroll
              for (int i = 0; i < 2 * W; ++i) x[k][i] = x[k][i] * rstd * w[k][i];
            }
            turn<W>(HALF, unit[k].pairs, co[k], si[k], x[k], x[k] + W);
          }
        }
        if (ok) {
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
            const float* y = BWD ? g[k] : x[k];
            if (unit[k].a >= 0) V::store(op + (h + j) * R.o_sh + unit[k].a, y);
            if (unit[k].b >= 0) V::store(op + (h + j) * R.o_sh + unit[k].b, y + W);
          }
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
      for (int i = 0; i < 2 * W; ++i) {
        float s = acc[k][i];
        for (int o = 16; o >= lanes; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
        const int e = i < W ? unit[k].a : unit[k].b;
        if ((threadIdx.x & 31) < lanes && e >= 0) fold[wib][e + (i < W ? i : i - W)] = s;
      }
    __syncthreads();
    float* partial = P.partial + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * P.d;
    for (int e = threadIdx.x; e < P.d; e += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k) s += fold[k][e];
      partial[e] = s;
    }
  }
}

// dw of a weight row: the sum of its slots' partials over the blocks, in a fixed order.  blockIdx.y: the weight row (queries'
// rows first); 32 elements a block, eight threads an element.
template <typename T>
__global__ void __launch_bounds__(256) heads_dweight_kernel(const HeadsParams P, int blocks) {
  __shared__ float fold[8][33];
  const int rows_q = P.weight_per_head ? P.part[0].heads : (P.part[0].heads > 0 ? 1 : 0);
  const bool keys = (int)blockIdx.y >= rows_q;
  const int row = (int)blockIdx.y - (keys ? rows_q : 0);
  const int first = (keys ? P.slots[0] : 0) + (P.weight_per_head ? row : 0);      // per head: one head a slot
  const int64_t count = (int64_t)(P.weight_per_head ? 1 : P.slots[keys]) * blocks;
  const int e = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
  float s = 0.f;
  if (e < P.d) {
    const float* src = P.partial + (int64_t)first * blocks * P.d + e;
#pragma unroll 8
    for (int64_t r = part; r < count; r += 8) s += src[r * P.d];
  }
  fold[part][threadIdx.x & 31] = s;
  __syncthreads();
  if (part == 0 && e < P.d) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += fold[k][threadIdx.x & 31];
    void* dw = P.part[keys].dweight;
    const int64_t at = (int64_t)row * P.d + e;
    if (P.weight_f32) ((float*)dw)[at] = s;
    else ((T*)dw)[at] = Elem<T>::from_float(s);
  }
}

// Widest vector that every row's start, the row length and the layout's second half allow
static int vector_width(const HeadsParams& P, int size, bool backward) {
  uint64_t all = (uint64_t)16 | (uint64_t)P.d * size;
  if (P.half) all |= (uint64_t)P.rotary_dim / 2 * size;
  for (const HeadRows& r : P.part) {
    if (r.heads == 0) continue;
    all |= reinterpret_cast<uintptr_t>(r.out) | (uint64_t)(r.o_sb | r.o_sh | r.o_sn) * size;
    if (r.x != nullptr) all |= reinterpret_cast<uintptr_t>(r.x) | (uint64_t)(r.x_sb | r.x_sh | r.x_sn) * size;
    if (backward) all |= reinterpret_cast<uintptr_t>(r.dy) | (uint64_t)(r.dy_sb | r.dy_sh | r.dy_sn) * size;
  }
  const uint64_t bytes = all & (~all + 1);
  return (int)(bytes / size);
}

// Blocks over the tokens and heads a slot
static void heads_grid(const HeadsParams& P, bool backward, int groups, int* per_slot, int64_t* blocks) {
  const int64_t all = ((int64_t)P.batch * P.seq + groups - 1) / groups;
  int per = P.norm && P.weight_per_head ? 1 : 8;
  auto slots = [&](int p) { return (int64_t)(P.part[0].heads + p - 1) / p + (P.part[1].heads + p - 1) / p; };
  // few tokens: heads go to blocks of their own until every SM has two
  while (per > 1 && all * slots(per) < 2 * 148) per /= 2;
  *per_slot = per;
  *blocks = all;
  if (P.norm && backward) {           // as many blocks as are resident, each with a partial weight gradient
    const int64_t most = (2 * 148 + slots(per) - 1) / slots(per);
    if (*blocks > most) *blocks = most;
  }
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
  // the most that any vector width asks for: 256 groups a block give the fewest blocks, 8 the most
  const int64_t slots = P0.part[0].heads + P0.part[1].heads;
  return (2 * 148 + slots) * P0.d;
}

template <typename T, int W, int UPL, bool NORM, bool BWD>
static int launch_heads_w(HeadsParams& P, cudaStream_t stream) {
  int units = 0, per = 0;
  int64_t blocks = 0;
  P.lane_shift = lane_shift(P, W, &units);
  if (units > UPL) return fail(NSA_ERR_UNSUPPORTED, "heads: dim_head is too large for rows that lie on such boundaries");
  heads_grid(P, BWD, heads::kThreads >> P.lane_shift, &per, &blocks);
  P.per_slot = per;
  for (int i = 0; i < 2; ++i) P.slots[i] = (P.part[i].heads + per - 1) / per;
  const int slots = P.slots[0] + P.slots[1];
  if (blocks > 0x7fffffffLL || slots > 65535) return fail(NSA_ERR_SHAPE, "heads: too many heads or tokens for one launch");
  const dim3 grid((unsigned)blocks, (unsigned)slots);
  if (P.half) heads_kernel<T, W, UPL, true, NORM, BWD><<<grid, heads::kThreads, 0, stream>>>(P);
  else heads_kernel<T, W, UPL, false, NORM, BWD><<<grid, heads::kThreads, 0, stream>>>(P);
  count_launches(1);
  if (NORM && BWD) {
    const int rows = P.weight_per_head ? P.part[0].heads + P.part[1].heads : (P.part[0].heads > 0) + (P.part[1].heads > 0);
    heads_dweight_kernel<T><<<dim3((unsigned)(P.d + 31) / 32, (unsigned)rows), 256, 0, stream>>>(P, (int)blocks);
    count_launches(1);
  }
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? NSA_OK : fail((int)err, cudaGetErrorString(err));
}

template <typename T, bool NORM, bool BWD>
static int launch_heads_typed(HeadsParams& P, cudaStream_t stream) {
  constexpr int kMost = 16 / (int)sizeof(T);
  const int W = vector_width(P, sizeof(T), BWD);
  if (W >= kMost) return launch_heads_w<T, kMost, 1, NORM, BWD>(P, stream);
  if (W >= kMost / 2) return launch_heads_w<T, kMost / 2, kMost / 2 >= 4 ? 1 : 2, NORM, BWD>(P, stream);
  return launch_heads_w<T, 1, 4, NORM, BWD>(P, stream);
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
  if (dtype == NSA_F32) {
    if (P.norm) return backward ? launch_heads_typed<float, true, true>(P, stream) : launch_heads_typed<float, true, false>(P, stream);
    return backward ? launch_heads_typed<float, false, true>(P, stream) : launch_heads_typed<float, false, false>(P, stream);
  }
  if (P.norm) return backward ? launch_heads_typed<__nv_bfloat16, true, true>(P, stream) : launch_heads_typed<__nv_bfloat16, true, false>(P, stream);
  return backward ? launch_heads_typed<__nv_bfloat16, false, true>(P, stream) : launch_heads_typed<__nv_bfloat16, false, false>(P, stream);
}

}  // namespace nsa
