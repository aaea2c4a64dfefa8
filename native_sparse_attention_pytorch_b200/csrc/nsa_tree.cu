// Attention of drafted tokens over a cache: sum_j p_j v_j with p = softmax(scale q . k_j) over the cached rows and, by a mask,
// the drafted ones.  One pass over the keys with the running maximum and sum of the softmax, both in fp32 and base 2.
//
// Rows.  The tokens times the query heads of a KV head are the rows that share its keys: row = token * G + head.  They are cut
// into tiles; a tile goes through blocks of keys, first those of the cache (up to the sequence's length), then the drafted ones.
//
// Sharing the keys out.  Lengths are known on the device only, and one long sequence among short ones must not leave the others'
// CTAs idle.  So all key blocks of all (sequence, KV head) units stand in one row, which is cut into equal pieces: group g of CTAs
// takes the blocks [g total / groups, (g+1) total / groups), a CTA of the group one row tile of them.  A piece may begin and end in
// the middle of a unit; what it has there leaves as a partial result (unnormalised sum, maximum, sum of exponentials), at most two
// per CTA: slot 0 where the piece begins inside the unit, slot 1 where it begins with it.  tree_merge_kernel joins a unit's
// partials, whose groups follow from the same arithmetic, in the order of the keys.
//
// Rows behind a length are never read.  A drafted value that is not finite would reach tokens which do not see it (0 times
// infinity is NaN): such values are left out of the products, and added behind them for the tokens that see them.

#include "nsa_common.cuh"
#include "nsa_kernels.h"
#include "nsa_sm100_ptx.cuh"

namespace nsa {

namespace tree {

__device__ __forceinline__ int length_of(const TreeParams& P, int b) {
  const int n = P.lengths != nullptr ? __ldg(P.lengths + b) : P.length;
  return max(0, min(n, P.capacity));
}

__device__ __forceinline__ int warp_add(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}

// Key blocks of one KV head of a sequence
template <int KB>
__device__ __forceinline__ int cache_blocks(const TreeParams& P, int b) { return (length_of(P, b) + KB - 1) / KB; }
template <int KB>
__device__ __forceinline__ int draft_blocks(const TreeParams& P) { return (P.tokens + KB - 1) / KB; }

// Blocks of all units, by a whole warp
template <int KB>
__device__ int64_t total_blocks(const TreeParams& P, int lane, int upto) {
  int64_t sum = 0;
  for (int b0 = 0; b0 < upto; b0 += 32) {
    const int b = b0 + lane;
    int64_t n = b < upto ? (int64_t)cache_blocks<KB>(P, b) + draft_blocks<KB>(P) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(kFullMask, n, o);
    sum += n;
  }
  return sum * P.kv_heads;
}

// Where a piece of the row of blocks begins: sequence and its first block
struct Place { int b; int64_t base; };
template <int KB>
__device__ Place place_of(const TreeParams& P, int lane, int64_t block) {
  Place at = {0, 0};
  for (int b0 = 0; b0 < P.batch; b0 += 32) {
    const int b = b0 + lane;
    const int64_t n = b < P.batch ? ((int64_t)cache_blocks<KB>(P, b) + draft_blocks<KB>(P)) * P.kv_heads : 0;
    int64_t upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(kFullMask, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned past = __ballot_sync(kFullMask, at.base + upto > block && b < P.batch);
    if (past) {
      const int first = __ffs(past) - 1;
      at.b = b0 + first;
      at.base += __shfl_sync(kFullMask, upto - n, first);
      return at;
    }
    at.base += __shfl_sync(kFullMask, upto, 31);
  }
  at.b = P.batch;
  return at;
}

__device__ __forceinline__ int64_t piece_begin(int64_t total, int g, int groups) { return total * g / groups; }

__device__ __forceinline__ bool sees(const TreeParams& P, int b, int t, int u) {
  return P.mask != nullptr ? P.mask[b * P.m_sb + t * P.m_st + u] != 0 : u <= t;
}

template <typename T>
__device__ __forceinline__ const T* row_of(const RowView& r, int b, int h, int64_t n) {
  return (const T*)r.p + b * r.sb + h * r.sh + n * r.sn;
}

}  // namespace tree

// ---- any type and alignment, on the CUDA cores -------------------------------------------

namespace tree_simt {
constexpr int kKeys = 64, kThreads = 256;
template <int DP, int RT>
struct Shape {
  static constexpr int kRow = DP + 4;                       // padded: four neighbouring rows on different banks
  static constexpr int kScore = kKeys + 4;
  static constexpr int TX = RT == 32 ? 16 : 64, TY = kThreads / TX;
  static constexpr int KPT = kKeys / TX, RPT = RT / TY;     // keys and rows of a thread
  static constexpr int CPT = DP / TX;                       // output columns of a thread
  static constexpr int kFloats = RT * kRow + 2 * kKeys * kRow + RT * kScore + 3 * RT;
};
}  // namespace tree_simt

// DP: dim_head padded to 64 or 128; RT: rows of a tile
template <typename T, int DP, int RT>
__global__ void __launch_bounds__(tree_simt::kThreads, 2) tree_simt_kernel(const TreeParams P, const int vec) {
  using namespace tree;
  using namespace tree_simt;
  using S = Shape<DP, RT>;
  constexpr int V = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) float tree_smem[];
  float* const qs = tree_smem;
  float* const ks = qs + RT * S::kRow;
  float* const vs = ks + kKeys * S::kRow;
  float* const ss = vs + kKeys * S::kRow;
  float* const row_m = ss + RT * S::kScore;
  float* const row_l = row_m + RT;
  float* const row_a = row_l + RT;
  __shared__ int odd_values;       // a drafted value of this unit is not finite
  const int tid = threadIdx.x, lane = tid & 31;
  const int tx = tid % S::TX, ty = tid / S::TX;
  const int tile = blockIdx.x % P.tiles, group = blockIdx.x / P.tiles;
  const int rows = P.tokens * P.G, row0 = tile * RT;

  const int64_t total = total_blocks<kKeys>(P, lane, P.batch);
  const int64_t begin = piece_begin(total, group, P.groups), end = piece_begin(total, group + 1, P.groups);
  if (begin >= end) return;
  Place at = place_of<kKeys>(P, lane, begin);
  const float scale2 = P.scale * kLog2e;

  // 16 bytes (or, where rows do not lie on such boundaries, one element) a thread and step; rows from `n` on are zero
  auto load_rows = [&](float* dst, const T* src, int64_t stride, int n, int count, bool mend) {
    if (vec) {
      const int per = P.d / V;
      for (int e = tid; e < count * (DP / V); e += kThreads) {
        const int r = e / (DP / V), c = e - r * (DP / V);
        float x[V];
        if (r < n && c < per) Elem<T>::load_vec(src + r * stride + c * V, x);
        else
#pragma unroll
          for (int i = 0; i < V; ++i) x[i] = 0.f;
        if (mend)
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (!isfinite(x[i])) { x[i] = 0.f; odd_values = 1; }
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(dst + r * S::kRow + c * V + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      }
    } else {
      for (int e = tid; e < count * DP; e += kThreads) {
        const int r = e / DP, c = e - r * DP;
        float x = r < n && c < P.d ? Elem<T>::to_float(src[r * stride + c]) : 0.f;
        if (mend && !isfinite(x)) { x = 0.f; odd_values = 1; }
        dst[r * S::kRow + c] = x;
      }
    }
  };

  for (int64_t at_block = begin; at_block < end;) {
    // the unit at_block lies in, and this piece's blocks of it
    const int cached = cache_blocks<kKeys>(P, at.b), per_unit = cached + draft_blocks<kKeys>(P), length = length_of(P, at.b);
    const int h = (int)((at_block - at.base) / per_unit);
    const int64_t unit0 = at.base + (int64_t)h * per_unit;
    const int j0 = (int)(at_block - unit0), j1 = (int)min((int64_t)per_unit, end - unit0);

    __syncthreads();
    if (tid == 0) odd_values = 0;
    for (int e = tid; e < RT * DP; e += kThreads) {
      const int r = e / DP, c = e - r * DP, row = row0 + r;
      const int t = row / P.G, g = row - t * P.G;
      qs[r * S::kRow + c] = row < rows && c < P.d ? Elem<T>::to_float(row_of<T>(P.q, at.b, h * P.G + g, t)[c]) : 0.f;
    }
    if (tid < RT) { row_m[tid] = -INFINITY; row_l[tid] = 0.f; }
    float o[S::RPT][S::CPT];
#pragma unroll
    for (int r = 0; r < S::RPT; ++r)
#pragma unroll
      for (int c = 0; c < S::CPT; ++c) o[r][c] = 0.f;

    for (int j = j0; j < j1; ++j) {
      const bool draft = j >= cached;
      const int first = (draft ? j - cached : j) * kKeys, n = min(kKeys, (draft ? P.tokens : length) - first);
      __syncthreads();   // the tiles and scores of the block before have been read
      load_rows(ks, row_of<T>(draft ? P.k : P.kc, at.b, h, first), draft ? P.k.sn : P.kc.sn, n, kKeys, false);
      load_rows(vs, row_of<T>(draft ? P.v : P.vc, at.b, h, first), draft ? P.v.sn : P.vc.sn, n, kKeys, draft);
      __syncthreads();

      // scores: keys tx + TX k, rows ty RPT + r
      float s[S::RPT][S::KPT];
#pragma unroll
      for (int r = 0; r < S::RPT; ++r)
#pragma unroll
        for (int k = 0; k < S::KPT; ++k) s[r][k] = 0.f;
#pragma unroll 4
      for (int c = 0; c < DP; c += 4) {
        float4 kv[S::KPT], qv[S::RPT];
#pragma unroll
        for (int k = 0; k < S::KPT; ++k) kv[k] = *reinterpret_cast<const float4*>(ks + (tx + S::TX * k) * S::kRow + c);
#pragma unroll
        for (int r = 0; r < S::RPT; ++r) qv[r] = *reinterpret_cast<const float4*>(qs + (ty * S::RPT + r) * S::kRow + c);
#pragma unroll
        for (int r = 0; r < S::RPT; ++r)
#pragma unroll
          for (int k = 0; k < S::KPT; ++k)
            s[r][k] += qv[r].x * kv[k].x + qv[r].y * kv[k].y + qv[r].z * kv[k].z + qv[r].w * kv[k].w;
      }
#pragma unroll
      for (int r = 0; r < S::RPT; ++r)
#pragma unroll
        for (int k = 0; k < S::KPT; ++k) {
          const int key = tx + S::TX * k, row = row0 + ty * S::RPT + r;
          const bool ok = key < n && row < rows && (!draft || sees(P, at.b, row / P.G, first + key));
          ss[(ty * S::RPT + r) * S::kScore + key] = ok ? s[r][k] * scale2 : -INFINITY;
        }
      __syncthreads();

      // softmax: kThreads / RT lanes share a row
      {
        constexpr int L = kThreads / RT, E = kKeys / L;
        const int r = tid / L, l = tid % L;
        float x[E], m = -INFINITY;
#pragma unroll
        for (int i = 0; i < E; ++i) { x[i] = ss[r * S::kScore + l + i * L]; m = fmaxf(m, x[i]); }
#pragma unroll
        for (int off = L / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, off));
        const float m_old = row_m[r], m_new = fmaxf(m_old, m), ref = m_new == -INFINITY ? 0.f : m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float p = exp2f(x[i] - ref);
          ss[r * S::kScore + l + i * L] = p;
          sum += p;
        }
#pragma unroll
        for (int off = L / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(kFullMask, sum, off);
        __syncwarp();
        if (l == 0) {
          const float a = exp2f(m_old - ref);      // 0 where nothing was seen before
          row_a[r] = a;
          row_m[r] = m_new;
          row_l[r] = row_l[r] * a + sum;
        }
      }
      __syncthreads();

      // output columns tx CPT + c
#pragma unroll
      for (int r = 0; r < S::RPT; ++r) {
        const float a = row_a[ty * S::RPT + r];
#pragma unroll
        for (int c = 0; c < S::CPT; ++c) o[r][c] *= a;
      }
#pragma unroll 4
      for (int k = 0; k < kKeys; ++k) {
        float p[S::RPT];
#pragma unroll
        for (int r = 0; r < S::RPT; ++r) p[r] = ss[(ty * S::RPT + r) * S::kScore + k];
#pragma unroll
        for (int c = 0; c < S::CPT; ++c) {
          const float v = vs[k * S::kRow + tx * S::CPT + c];
#pragma unroll
          for (int r = 0; r < S::RPT; ++r) o[r][c] += p[r] * v;
        }
      }
    }

    if (odd_values) {
      const int u0 = max(0, j0 - cached) * kKeys, u1 = min(P.tokens, (j1 - cached) * kKeys);
#pragma unroll
      for (int r = 0; r < S::RPT; ++r) {
        const int row = row0 + ty * S::RPT + r;
        for (int u = u0; u < u1; ++u) {
          if (row >= rows || !sees(P, at.b, row / P.G, u)) continue;
#pragma unroll
          for (int c = 0; c < S::CPT; ++c) {
            const int col = tx * S::CPT + c;
            const float v = col < P.d ? Elem<T>::to_float(row_of<T>(P.v, at.b, h, u)[col]) : 0.f;
            if (!isfinite(v)) o[r][c] += v;
          }
        }
      }
    }
    const bool whole = j0 == 0 && j1 == per_unit;
    const int64_t slot = (int64_t)blockIdx.x * 2 + (j0 == 0 ? 1 : 0);
#pragma unroll
    for (int r = 0; r < S::RPT; ++r) {
      const int local = ty * S::RPT + r, row = row0 + local;
      if (row >= rows) continue;
      const int t = row / P.G, g = row - t * P.G;
      const float l = row_l[local];
      if (whole) {
        T* out = const_cast<T*>(row_of<T>(P.out, at.b, h * P.G + g, t));
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);      // a sum that is NaN stays NaN
#pragma unroll
        for (int c = 0; c < S::CPT; ++c)
          if (tx * S::CPT + c < P.d) out[tx * S::CPT + c] = Elem<T>::from_float(o[r][c] * inv);
        if (tx == 0 && P.lse != nullptr)
          P.lse[((int64_t)at.b * P.q_heads + h * P.G + g) * P.tokens + t] = l == 0.f ? -INFINITY : (row_m[local] + log2f(l)) * kLn2;
      } else {
#pragma unroll
        for (int c = 0; c < S::CPT; ++c) P.partial[(slot * RT + local) * DP + tx * S::CPT + c] = o[r][c];
        if (tx == 0) P.stats[slot * RT + local] = make_float2(row_m[local], l);
      }
    }
    at_block = unit0 + j1;
    if (at_block - at.base == (int64_t)per_unit * P.kv_heads) {
      at.base = at_block;
      ++at.b;
    }
  }
}

// ---- joining the partial results -----------------------------------------------------------

// A warp per row of a unit that more than one group of CTAs worked on
template <typename T, int DP, int RT, int KB>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeParams P) {
  using namespace tree;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = P.tokens * P.G, row = blockIdx.x * 8 + warp;
  const int b = blockIdx.y / P.kv_heads, h = blockIdx.y - b * P.kv_heads;
  ptx::grid_wait();
  if (row >= rows) return;
  const int64_t total = total_blocks<KB>(P, lane, P.batch);
  const int per_unit = cache_blocks<KB>(P, b) + draft_blocks<KB>(P);
  const int64_t unit0 = total_blocks<KB>(P, lane, b) + (int64_t)h * per_unit;
  // the group that has block x: the last whose piece begins at or before it
  auto group_of = [&](int64_t x) { return (int)(((x + 1) * P.groups - 1) / total); };
  const int g0 = group_of(unit0), g1 = group_of(unit0 + per_unit - 1);
  if (g0 == g1) return;
  const int tile = row / RT, local = row - tile * RT;
  auto slot_of = [&](int g) { return ((int64_t)g * P.tiles + tile) * 2 + (g == g0 ? 1 : 0); };

  // two passes over the statistics: the largest maximum, then sums; lanes take groups side by side
  float top = -INFINITY;
  for (int g = g0 + lane; g <= g1; g += 32) {
    // a group without blocks has no piece, its place lies between those of its neighbours
    if (piece_begin(total, g, P.groups) < piece_begin(total, g + 1, P.groups)) top = fmaxf(top, P.stats[slot_of(g) * RT + local].x);
  }
  top = warp_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  constexpr int C = DP / 32;
  float o[C], l = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = 0.f;
  for (int first = g0; first <= g1; first += 32) {
    const int g = first + lane;
    float w = 0.f;
    const bool there = g <= g1 && piece_begin(total, g, P.groups) < piece_begin(total, g + 1, P.groups);
    if (there) {
      const float2 st = P.stats[slot_of(g) * RT + local];
      w = exp2f(st.x - ref);
      l += st.y * w;
    }
    unsigned todo = __ballot_sync(kFullMask, there);
    while (todo) {
      const int k = __ffs(todo) - 1;
      todo &= todo - 1;
      const float wk = __shfl_sync(kFullMask, w, k);
      const float* src = P.partial + (slot_of(first + k) * RT + local) * DP + lane * C;
      __align__(16) float v[C];
      if constexpr (C == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
      else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] += v[c] * wk;
    }
  }
  l = warp_sum(l);
  const int t = row / P.G, g = row - t * P.G;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  T* out = const_cast<T*>(row_of<T>(P.out, b, h * P.G + g, t));
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (lane * C + c < P.d) out[lane * C + c] = Elem<T>::from_float(o[c] * inv);
  if (lane == 0 && P.lse != nullptr)
    P.lse[((int64_t)b * P.q_heads + h * P.G + g) * P.tokens + t] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
}

// ---- host ------------------------------------------------------------------------------------

struct TreePlan {
  bool tensor_cores;
  int DP, RT, KB, ctas;      // padded dim_head, rows of a tile, keys of a block, CTAs the device holds at once
  int tiles, groups;
  int64_t partial_bytes, bytes;
};

static TreePlan plan_tree(const TreeParams& P, int dtype, int impl) {
  (void)dtype; (void)impl;
  TreePlan p = {};
  const int64_t rows = (int64_t)P.tokens * P.G;
  p.DP = P.d <= 64 ? 64 : 128;
  p.RT = rows <= 8 ? 8 : 32;
  p.KB = tree_simt::kKeys;
  p.ctas = 2 * 148;
  p.tiles = (int)((rows + p.RT - 1) / p.RT);
  p.groups = p.tiles >= p.ctas ? 1 : p.ctas / p.tiles;
  // no more groups than there can be blocks
  const int64_t most = (int64_t)P.batch * P.kv_heads * (((int64_t)P.capacity + p.KB - 1) / p.KB + (P.tokens + p.KB - 1) / p.KB);
  if (p.groups > most) p.groups = (int)most;
  const int64_t slots = (int64_t)p.groups * p.tiles * 2;
  p.partial_bytes = slots * p.RT * p.DP * (int64_t)sizeof(float);
  p.bytes = p.groups > 1 ? p.partial_bytes + slots * p.RT * (int64_t)sizeof(float2) : 0;
  return p;
}

int64_t tree_workspace_bytes(const TreeParams& P, int dtype, int impl) {
  return plan_tree(P, dtype, impl).bytes;
}

template <typename T, int DP, int RT>
static int run_simt(const TreeParams& P, const TreePlan& p, cudaStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T);
  auto wide = [](const RowView& r) { return (reinterpret_cast<uintptr_t>(r.p) & 15u) == 0 && r.sb % V == 0 && r.sh % V == 0 && r.sn % V == 0; };
  const int vec = wide(P.k) && wide(P.v) && (P.capacity == 0 || (wide(P.kc) && wide(P.vc)));
  const int smem = tree_simt::Shape<DP, RT>::kFloats * (int)sizeof(float);
  cudaError_t err = allow_shared_memory<tree_simt_kernel<T, DP, RT>>();
  if (err != cudaSuccess) return fail((int)err, cudaGetErrorString(err));
  tree_simt_kernel<T, DP, RT><<<(unsigned)(p.groups * p.tiles), tree_simt::kThreads, smem, stream>>>(P, vec);
  if (p.groups > 1) {
    const dim3 grid((unsigned)(((int64_t)P.tokens * P.G + 7) / 8), (unsigned)(P.batch * P.kv_heads));
    tree_merge_kernel<T, DP, RT, tree_simt::kKeys><<<grid, 256, 0, stream>>>(P);
  }
  count_launches(p.groups > 1 ? 2 : 1);
  err = cudaGetLastError();
  return err == cudaSuccess ? NSA_OK : fail((int)err, cudaGetErrorString(err));
}

template <typename T>
static int run_simt_typed(const TreeParams& P, const TreePlan& p, cudaStream_t stream) {
  if (p.DP == 64) return p.RT == 8 ? run_simt<T, 64, 8>(P, p, stream) : run_simt<T, 64, 32>(P, p, stream);
  return p.RT == 8 ? run_simt<T, 128, 8>(P, p, stream) : run_simt<T, 128, 32>(P, p, stream);
}

int launch_tree(TreeParams& P, int dtype, int impl, uint8_t* workspace, cudaStream_t stream) {
  const TreePlan p = plan_tree(P, dtype, impl);
  if (impl == NSA_IMPL_SM100) return fail(NSA_ERR_UNSUPPORTED, "tree: not served by the tensor-core kernel");
  if ((int64_t)p.groups * p.tiles > 0x7fffffffLL || (int64_t)P.batch * P.kv_heads > 65535)
    return fail(NSA_ERR_SHAPE, "tree: too many rows, or more than 65535 KV heads over the batch");
  P.tiles = p.tiles; P.groups = p.groups;
  P.partial = reinterpret_cast<float*>(workspace);
  P.stats = reinterpret_cast<float2*>(workspace + p.partial_bytes);
  return dtype == NSA_F32 ? run_simt_typed<float>(P, p, stream) : run_simt_typed<__nv_bfloat16>(P, p, stream);
}

}  // namespace nsa
