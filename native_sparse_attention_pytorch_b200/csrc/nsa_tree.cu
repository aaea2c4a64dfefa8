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
// Rows behind a length leave no trace.  The CUDA cores do not read them; the tensor cores' kernels fetch a sequence's last block whole,
// mask the logits of the rows behind and clear their values before the products.  A drafted value that is not finite would reach
// tokens which do not see it (0 times infinity is NaN): such values are left out of the products, and added behind them for the
// tokens that see them.

#include "nsa_common.cuh"
#include "nsa_kernels.h"
#include "nsa_sm100_ptx.cuh"

namespace nsa {

namespace tree {

__device__ __forceinline__ int length_of(const TreeParams& P, int b) {
  const int n = P.lengths != nullptr ? __ldg(P.lengths + b) : P.length;
  return max(0, min(n, P.capacity));
}

// Key blocks of one KV head of a sequence.  (Unsigned: a length may lie less than a block below 2^31.)
template <int KB>
__device__ __forceinline__ int blocks_of(int rows) { return (int)(((unsigned)rows + KB - 1) / KB); }
template <int KB>
__device__ __forceinline__ int cache_blocks(const TreeParams& P, int b) { return blocks_of<KB>(length_of(P, b)); }
template <int KB>
__device__ __forceinline__ int draft_blocks(const TreeParams& P) { return blocks_of<KB>(P.tokens); }

// Blocks of the units of the sequences before `upto`, and of all, by a whole warp
template <int KB>
__device__ void count_blocks(const TreeParams& P, int lane, int upto, int64_t& before, int64_t& total) {
  int64_t all = 0, some = 0;
  for (int b = lane; b < P.batch; b += 32) {
    const int n = cache_blocks<KB>(P, b) + draft_blocks<KB>(P);
    all += n;
    some += b < upto ? n : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(kFullMask, all, o);
    some += __shfl_xor_sync(kFullMask, some, o);
  }
  total = all * P.kv_heads;
  before = some * P.kv_heads;
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

// The groups that have blocks: no more than there are blocks, so that none of them is without
__device__ __forceinline__ int busy_groups(const TreeParams& P, int64_t total) { return (int)min((int64_t)P.groups, total); }
// x / y; a division of 64-bit numbers takes some hundred instructions
__device__ __forceinline__ int64_t quotient(int64_t x, int y) {
  return (uint64_t)x >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
}
__device__ __forceinline__ int64_t piece_begin(int64_t total, int g, int groups) { return quotient(total * g, groups); }
// The group that has block x: the last whose piece begins at or before it
__device__ __forceinline__ int group_of(int64_t total, int64_t x, int groups) {
  const int64_t y = (x + 1) * groups - 1;
  return (uint64_t)(y | total) >> 32 ? (int)(y / total) : (int)((uint32_t)y / (uint32_t)total);
}

// A reference maximum (base 2) beyond this is `far`.  The product logit * scale, less the reference, is one fused operation on the tensor
// cores' kernels; the reference is a product rounded to fp32, so that the difference of the largest logit from itself is not zero but up
// to half a unit of the reference's last place: 2^-8 here, a factor of 2^128 and more from 2^31 on.  Far logits are multiplied first.
constexpr float kFar = 65536.f;
__device__ __forceinline__ bool is_far(float ref) { return fabsf(ref) > kFar && fabsf(ref) != INFINITY; }

__device__ __forceinline__ bool sees(const TreeParams& P, int b, int t, int u) {
  return P.mask != nullptr ? P.mask[b * P.m_sb + t * P.m_st + u] != 0 : u <= t;
}

// Which of 32 drafted rows from `first` on token t sees, `row` its row of the mask (or NULL); and which of N rows (token, head) from
// `first` on see drafted row u: bits.  The loads do not depend on one another, so that they are under way all at once; a call of its
// own, because they would take registers from the loop over the cached keys.
__device__ __noinline__ uint32_t seen_from(const uint8_t* row, int t, int first, int tokens) {
  uint32_t bits = 0;
  if (row == nullptr) {
#pragma unroll
    for (int i = 0; i < 32; ++i) bits |= (first + i <= t ? 1u : 0u) << i;
    return bits;
  }
  uint8_t v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = row[min(first + i, tokens - 1)];
#pragma unroll
  for (int i = 0; i < 32; ++i) bits |= (v[i] != 0 && first + i < tokens ? 1u : 0u) << i;
  return bits;
}
template <int N>
__device__ __forceinline__ uint32_t seen_by(const TreeParams& P, int b, int first, int u) {
  uint32_t bits = 0;
  if (u >= P.tokens) return 0;
  int t[N], g = first % P.G;
  t[0] = first / P.G;
#pragma unroll
  for (int i = 1; i < N; ++i) {
    const bool next = ++g == P.G;
    t[i] = t[i - 1] + next;
    if (next) g = 0;
  }
  if (P.mask == nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) bits |= (u <= t[i] && t[i] < P.tokens ? 1u : 0u) << i;
    return bits;
  }
  const uint8_t* m = P.mask + b * P.m_sb + u;
  uint8_t v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = m[min(t[i], P.tokens - 1) * P.m_st];
#pragma unroll
  for (int i = 0; i < N; ++i) bits |= (v[i] != 0 && t[i] < P.tokens ? 1u : 0u) << i;
  return bits;
}

template <typename T>
__device__ __forceinline__ const T* row_of(const RowView& r, int b, int h, int64_t n) {
  return (const T*)r.p + b * r.sb + h * r.sh + n * r.sn;
}

}  // namespace tree

// ---- any type and alignment, on the CUDA cores -------------------------------------------

// fp32, and bf16 rows that TMA cannot fetch.  256 threads share a tile of 8, 32 or 64 rows: scores of a block into shared memory, softmax
// by 32, 8 or 4 lanes a row, values times weights in registers.  Bound by shared memory and issue: with 64 rows of 128 a thread has 4 rows
// x 2 keys and four features, then 4 x 8 columns and four keys: six and twelve 16-byte reads for 32 and 128 fused multiplications of a
// step.  fp32 rows arrive a block ahead.
// 4 x 64 tokens over 4096 rows, 64 / 8 heads of 128: 1111 us, 31 TFLOP/s (over half to all of them: 967; tiles of 32 rows, loads in turn,
// columns read one by one: 1712); 16 x one token over 8192 rows, 32 / 4 heads of 128: 162 us, 3.3 TB/s (over half to all of them: 127; two
// rows x one key a thread: 167).

namespace tree_simt {
constexpr int kThreads = 256;
template <int DP, int RT>
struct Shape {
  static constexpr int kKeys = RT == 8 ? 64 : 32;           // of a block; two are in shared memory
  static constexpr int kRow = DP + 4;                       // padded: four neighbouring rows on different banks
  static constexpr int kScore = kKeys + 4;
  static constexpr int TX = RT == 8 ? 32 : 16, TY = kThreads / TX;
  static constexpr int KPT = kKeys / TX, RPT = RT / TY;     // keys and rows of a thread
  static constexpr int kPlanes = RT == 8 ? 4 : 1;           // eight rows: scores by quarters of the features
  static constexpr int CPT = DP / TX;                       // output columns of a thread, VC neighbours every VC TX
  static constexpr int VC = CPT < 4 ? CPT : 4;
  static constexpr int kFloats = RT * kRow + 4 * kKeys * kRow + kPlanes * RT * kScore + 3 * RT;
  static constexpr int kPerSM = kFloats * 4 <= 113 * 1024 ? 2 : 1;          // CTAs
};
}  // namespace tree_simt

// DP: dim_head padded to 64 or 128; RT: rows of a tile
template <typename T, int DP, int RT>
__global__ void __launch_bounds__(tree_simt::kThreads, tree_simt::Shape<DP, RT>::kPerSM) tree_simt_kernel(const TreeParams P, const int vec) {
  using namespace tree;
  using namespace tree_simt;
  using S = Shape<DP, RT>;
  constexpr int V = 16 / (int)sizeof(T), kKeys = S::kKeys;
  extern __shared__ __align__(16) float tree_smem[];
  float* const qs = tree_smem;
  float* const tiles = qs + RT * S::kRow;               // K and V of two blocks
  float* const ss = tiles + 4 * kKeys * S::kRow;
  float* const row_m = ss + S::kPlanes * RT * S::kScore;
  float* const row_l = row_m + RT;
  float* const row_a = row_l + RT;
  __shared__ int odd_values;       // a drafted value of this unit is not finite
  const int tid = threadIdx.x, lane = tid & 31;
  const int tx = tid % S::TX, ty = tid / S::TX;
  auto column = [&](int c) { return (c / S::VC * S::TX + tx) * S::VC + c % S::VC; };
  const int tile = blockIdx.x % P.tiles, group = blockIdx.x / P.tiles;
  const int rows = P.tokens * P.G, row0 = tile * RT;

  ptx::grid_allow_next();
  int64_t before, total;
  count_blocks<kKeys>(P, lane, 0, before, total);
  const int groups = busy_groups(P, total);
  if (group >= groups) return;
  const int64_t begin = piece_begin(total, group, groups), end = piece_begin(total, group + 1, groups);
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

  // fp32 rows on 16-byte boundaries come asynchronously, a block ahead
  const bool ahead = vec && sizeof(T) == 4;
  auto fetch_rows = [&](float* dst, const T* src, int64_t stride, int n) {
    const int per = P.d / V;
    const uint32_t to = ptx::smem_u32(dst);
    for (int e = tid; e < kKeys * (DP / V); e += kThreads) {
      const int r = e / (DP / V), c = e - r * (DP / V);
      const bool there = r < n && c < per;
      ptx::cp_async16(to + (r * S::kRow + c * V) * 4, there ? src + r * stride + c * V : src, there ? 16 : 0);
    }
  };

  for (int64_t at_block = begin; at_block < end;) {
    // the unit at_block lies in, and this piece's blocks of it
    const int cached = cache_blocks<kKeys>(P, at.b), per_unit = cached + draft_blocks<kKeys>(P), length = length_of(P, at.b);
    const int h = (int)quotient(at_block - at.base, per_unit);
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
    // Eight rows: a thread takes all of them, for one key and a quarter of the features, then for an eighth of the keys (its warp's) and
    // its columns, so that K and V are read from shared memory once; the warps' sums are added at the unit's end.
    constexpr int ROWS = RT == 8 ? 8 : S::RPT;
    float o[ROWS][S::CPT];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int c = 0; c < S::CPT; ++c) o[r][c] = 0.f;

    auto fetch_block = [&](int j) {
      const bool draft = j >= cached;
      const int first = (draft ? j - cached : j) * kKeys, n = min(kKeys, (draft ? P.tokens : length) - first);
      float* const to = tiles + (j & 1) * (2 * kKeys * S::kRow);
      fetch_rows(to, row_of<T>(draft ? P.k : P.kc, at.b, h, first), draft ? P.k.sn : P.kc.sn, n);
      fetch_rows(to + kKeys * S::kRow, row_of<T>(draft ? P.v : P.vc, at.b, h, first), draft ? P.v.sn : P.vc.sn, n);
    };
    if (ahead) {
      fetch_block(j0);          // (the barrier above: the tiles of the unit before have been read)
      ptx::cp_async_commit();
    }

    for (int j = j0; j < j1; ++j) {
      const bool draft = j >= cached;
      const int first = (draft ? j - cached : j) * kKeys, n = min(kKeys, (draft ? P.tokens : length) - first);
      float* const ks = tiles + (j & 1) * (2 * kKeys * S::kRow);
      float* const vs = ks + kKeys * S::kRow;
      __syncthreads();   // the tiles and scores of the block before have been read
      if (ahead) {
        if (j + 1 < j1) fetch_block(j + 1);
        ptx::cp_async_commit();
        ptx::cp_async_wait<1>();
        if (draft) {     // each thread mends what it fetched
          for (int e = tid; e < kKeys * (DP / V); e += kThreads) {
            const int r = e / (DP / V), c = e - r * (DP / V);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              float& x = vs[r * S::kRow + c * V + i];
              if (!isfinite(x)) { x = 0.f; odd_values = 1; }
            }
          }
        }
      } else {
        load_rows(ks, row_of<T>(draft ? P.k : P.kc, at.b, h, first), draft ? P.k.sn : P.kc.sn, n, kKeys, false);
        load_rows(vs, row_of<T>(draft ? P.v : P.vc, at.b, h, first), draft ? P.v.sn : P.vc.sn, n, kKeys, draft);
      }
      __syncthreads();

      if constexpr (RT == 8) {
        const int key = tid & 63, part = tid >> 6;
        float d[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) d[r] = 0.f;
#pragma unroll 4
        for (int c = part * (DP / 4); c < (part + 1) * (DP / 4); c += 4) {
          const float4 kv = *reinterpret_cast<const float4*>(ks + key * S::kRow + c);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const float4 qv = *reinterpret_cast<const float4*>(qs + r * S::kRow + c);
            d[r] += qv.x * kv.x + qv.y * kv.y + qv.z * kv.z + qv.w * kv.w;
          }
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) ss[(part * 8 + r) * S::kScore + key] = d[r];
      } else {
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
      }
      __syncthreads();

      // softmax: kThreads / RT lanes share a row
      {
        constexpr int L = kThreads / RT, E = kKeys / L;
        const int r = tid / L, l = tid % L;
        float x[E], m = -INFINITY;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          x[i] = ss[r * S::kScore + l + i * L];
          if constexpr (RT == 8) {
#pragma unroll
            for (int k = 1; k < 4; ++k) x[i] += ss[(k * 8 + r) * S::kScore + l + i * L];
            const int key = l + i * L;
            x[i] = key < n && r < rows && (!draft || sees(P, at.b, r / P.G, first + key)) ? x[i] * scale2 : -INFINITY;
          }
          m = fmaxf(m, x[i]);
        }
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

      // output columns: column(c)
      const int first_row = RT == 8 ? 0 : ty * S::RPT, first_key = RT == 8 ? ty * 8 : 0, last_key = RT == 8 ? first_key + 8 : kKeys;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float a = row_a[first_row + r];
#pragma unroll
        for (int c = 0; c < S::CPT; ++c) o[r][c] *= a;
      }
#pragma unroll 2
      for (int k = first_key; k < last_key; k += 4) {
        float4 p[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) p[r] = *reinterpret_cast<const float4*>(ss + (first_row + r) * S::kScore + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          float v[S::CPT];
#pragma unroll
          for (int c = 0; c < S::CPT; c += S::VC) {
            const float* at = vs + (k + kk) * S::kRow + column(c);
            if constexpr (S::VC == 4) {
              const float4 q = *reinterpret_cast<const float4*>(at);
              v[c] = q.x; v[c + 1] = q.y; v[c + 2] = q.z; v[c + 3] = q.w;
            } else if constexpr (S::VC == 2) {
              const float2 q = *reinterpret_cast<const float2*>(at);
              v[c] = q.x; v[c + 1] = q.y;
            } else {
              v[c] = *at;
            }
          }
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const float w = kk == 0 ? p[r].x : kk == 1 ? p[r].y : kk == 2 ? p[r].z : p[r].w;
#pragma unroll
            for (int c = 0; c < S::CPT; ++c) o[r][c] += w * v[c];
          }
        }
      }
    }
    if constexpr (RT == 8) {
      __syncthreads();           // the tiles have been read
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int c = 0; c < S::CPT; ++c) tiles[(ty * 8 + r) * DP + column(c)] = o[r][c];
      __syncthreads();
#pragma unroll
      for (int c = 0; c < S::CPT; ++c) {      // warp ty has row ty now
        o[0][c] = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[0][c] += tiles[(k * 8 + ty) * DP + column(c)];
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
            const int col = column(c);
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
          if (column(c) < P.d) out[column(c)] = Elem<T>::from_float(o[r][c] * inv);
        if (tx == 0 && P.lse != nullptr)
          P.lse[((int64_t)at.b * P.q_heads + h * P.G + g) * P.tokens + t] = l == 0.f ? -INFINITY : (row_m[local] + log2f(l)) * kLn2;
      } else {
#pragma unroll
        for (int c = 0; c < S::CPT; ++c) P.partial[(slot * RT + local) * DP + column(c)] = o[r][c];
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

// ---- bf16, on the tensor cores ---------------------------------------------------------------

// A persistent CTA per SM goes through its piece of the key blocks (128 keys, with two streams 64):
//   TMA warp        K and V blocks through a ring of slots (K, V, K, V, ...), across units and as far ahead as the ring holds
//   mending warp    clears the rows of a V block that lie behind the sequence, and drafted values that are not finite
//   MMA warp(s)     S = Q K^T, then O += P V with P from tensor memory; one per stream
//   softmax warps   S from tensor memory, maximum, exponentials, P back as bf16.  A warp reaches 32 lanes of tensor memory, 32 rows.
//                   One stream: two threads per row, half of a block's keys each, which exchange maxima.  Two streams: one thread (64
//                   tokens over 65536 rows, a block of 64 keys and two tiles: 1790 cycles, with two threads 2000).  P is rounded, up to
//                   2^-8 of a weight, as any bf16 tensor of weights would be; the sum adds the exponentials as they are.
// The accumulator O stays in tensor memory.  It is rescaled lazily: a row keeps its reference maximum until a block exceeds it by
// more than 2^8.
// What bounds it: the exponentials (16 a cycle and SM) and what else a warp does for a value beside them; then power.  64 tokens over 65536
// rows, 64 / 8 heads of 128: 393 us, 1170 TFLOP/s, in bursts of 30 passes, 461 us back to back (1.5 GHz at 990 W).
// STREAMS.  Above 128 rows two tiles share the K and V blocks; the softmax of one runs under the products of the other.  Blocks of 64
// keys, so that tensor memory holds two S buffers of either beside both O: with blocks of 128 and one buffer, S of the next block
// waited for the products of this one, which waited for its softmax (3800 cycles a block and pair of tiles, 2050 of them products).
namespace tree_tc {
constexpr int kRows = 128;
constexpr int keys(int streams) { return streams == 1 ? 128 : 64; }     // of a block
template <int D, int STREAMS>
struct Shape {
  static constexpr int KK = keys(STREAMS);
  static constexpr int NC = D / 64;                                // 64-column subtiles of a row
  static constexpr uint32_t kTileQ = NC * 16384, kSub = KK * 128, kTile = NC * kSub;
  static constexpr int kSlots = (14 * 16384 - STREAMS * kTileQ) / kTile;
  static constexpr uint32_t kBytes = STREAMS * kTileQ + kSlots * kTile;
  static constexpr int kHalves = STREAMS == 1 ? 2 : 1;             // threads of a row
  static constexpr int kWarps = 4 * kHalves * STREAMS + STREAMS + 2, kThreads = 32 * kWarps;
};
constexpr int kMostSlots = 24, kAhead = 16;
struct Bars {
  uint64_t full[kMostSlots], free[kMostSlots];
  uint64_t ready[kAhead];         // V blocks, by their number: the mending warp is never this many ahead of the products
  uint64_t q_full[2], s_full[2][2], p_full[2][2], pv_done[2][2], drain[2];
};
}  // namespace tree_tc

namespace tree {

// The units of a CTA's piece, one after the other; every warp walks by itself
template <int KB>
struct Walk {
  int b, h, length, cached, per_unit, j0, j1;
  int64_t base, at, end, unit0;
  // by a whole warp
  __device__ void ask(const TreeParams& P, int lane) { length = lane < P.batch ? length_of(P, lane) : 0; }
  __device__ void begin(const TreeParams& P, int lane, int group) {
    if (P.batch <= 32) {                  // one look at the lengths
      const int64_t n = lane < P.batch ? ((int64_t)blocks_of<KB>(length) + draft_blocks<KB>(P)) * P.kv_heads : 0;
      int64_t upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(kFullMask, upto, o);
        if (lane >= o) upto += v;
      }
      set_piece(P, __shfl_sync(kFullMask, upto, 31), group);
      const unsigned past = __ballot_sync(kFullMask, upto > at && lane < P.batch);
      b = past ? __ffs(past) - 1 : P.batch;
      base = __shfl_sync(kFullMask, upto - n, b & 31);
    } else {
      int64_t before, total;
      count_blocks<KB>(P, lane, 0, before, total);
      set_piece(P, total, group);
      const Place p = place_of<KB>(P, lane, at);
      b = p.b;
      base = p.base;
    }
  }
  __device__ void set_piece(const TreeParams& P, int64_t total, int group) {
    const int groups = busy_groups(P, total);
    at = group < groups ? piece_begin(total, group, groups) : 0;
    end = group < groups ? piece_begin(total, group + 1, groups) : 0;
  }
  // the unit the piece is at, if it is not at its end
  __device__ bool unit(const TreeParams& P) {
    if (at >= end) return false;
    length = length_of(P, b);
    cached = blocks_of<KB>(length);
    per_unit = cached + draft_blocks<KB>(P);
    h = (int)quotient(at - base, per_unit);
    unit0 = base + (int64_t)h * per_unit;
    j0 = (int)(at - unit0);
    j1 = (int)min((int64_t)per_unit, end - unit0);
    return true;
  }
  __device__ void next(const TreeParams& P) {
    at = unit0 + j1;
    if (at - base == (int64_t)per_unit * P.kv_heads) {
      base = at;
      ++b;
    }
  }
};

}  // namespace tree

// Which of a cache's axes the coordinates move along (an axis of stride zero is one entry in its tensor map)
struct TreeAxes { int kc_b, kc_h, vc_b, vc_h, k_b, k_h, v_b, v_h; };

// The role of the TMA warp: K and V blocks of all units into the ring, as far ahead as it holds
template <int D, int KK, int SLOTS>
__device__ __forceinline__ void fetch_blocks(const TreeParams& P, const TreeAxes& A, const CUtensorMap& tmKc, const CUtensorMap& tmVc, const CUtensorMap& tmK,
                                             const CUtensorMap& tmV, tree::Walk<KK>& walk, uint32_t ring, tree_tc::Bars& bars, int lane, volatile int* abort_flag) {
  using namespace ptx;
  constexpr int NC = D / 64;
  constexpr uint32_t kSub = KK * 128, kTile = NC * kSub;
  uint32_t i = 0;
  for (; walk.unit(P); walk.next(P)) {
    for (int j = walk.j0; j < walk.j1; ++j) {
      const bool draft = j >= walk.cached;
      const int first = (draft ? j - walk.cached : j) * KK;
#pragma unroll
      for (int v = 0; v < 2; ++v, ++i) {
        const uint32_t slot = i % SLOTS, round = i / SLOTS;
        if (round >= 1) mbar_wait_bounded(smem_u32(&bars.free[slot]), (round - 1) & 1, abort_flag);
        if (lane == 0) {
          const CUtensorMap* map = draft ? (v ? &tmV : &tmK) : (v ? &tmVc : &tmKc);
          const int bb = walk.b * (draft ? (v ? A.v_b : A.k_b) : (v ? A.vc_b : A.kc_b));
          const int hh = walk.h * (draft ? (v ? A.v_h : A.k_h) : (v ? A.vc_h : A.kc_h));
          mbar_arrive_expect_tx(smem_u32(&bars.full[slot]), kTile);
#pragma unroll
          for (int c = 0; c < NC; ++c) tma_load_4d(ring + slot * kTile + c * kSub, map, smem_u32(&bars.full[slot]), c * 64, first, hh, bb);
        }
        __syncwarp();
      }
    }
  }
  // every request must have landed before the block may exit (also when it gave up)
  for (uint32_t back = 1; back <= (uint32_t)SLOTS && back <= i; ++back)
    mbar_wait_drain(smem_u32(&bars.full[(i - back) % SLOTS]), ((i - back) / SLOTS) & 1);
}

// The role of the mending warp: rows of a V block behind the sequence are cleared, as are drafted values that are not finite.  It asks
// about every block in turn, and a barrier is asked by the parity of its phase: a slot must not be filled again before this warp has
// seen it full (the phase it asks for would be over, and the next one of that parity waits for this warp), and it must not ask about a
// phase before the one in front of it is over (a slot may hold K and V in turn).  So it waits for K as well, and gives slots back.
template <int D, int KK, int SLOTS>
__device__ __forceinline__ void mend_blocks(const TreeParams& P, tree::Walk<KK>& walk, uint32_t ring, tree_tc::Bars& bars, volatile int* odd_values, int lane,
                                            volatile int* abort_flag) {
  using namespace ptx;
  using tree_tc::kAhead;
  constexpr int NC = D / 64;
  constexpr uint32_t kSub = KK * 128, kTile = NC * kSub;
  uint32_t u = 0;
  for (int seq = 0; walk.unit(P); walk.next(P), ++seq) {
    int odd = 0;
    for (int j = walk.j0; j < walk.j1; ++j, ++u) {
      const uint32_t slot = (2 * u + 1) % SLOTS, round = (2 * u + 1) / SLOTS;
      const uint32_t at = ring + slot * kTile;
      mbar_wait_warp(smem_u32(&bars.full[2 * u % SLOTS]), (2 * u / SLOTS) & 1, abort_flag);
      if (lane == 0) mbar_arrive(smem_u32(&bars.free[2 * u % SLOTS]));
      mbar_wait_warp(smem_u32(&bars.full[slot]), round & 1, abort_flag);
      const bool draft = j >= walk.cached;
      const int n = min(KK, (draft ? P.tokens - (j - walk.cached) * KK : walk.length - j * KK));
      if (draft || n < KK) {
        if (!draft)       // behind the drafted rows the tile is zero as loaded
          for (int e = lane; e < (KK - n) * 8 * NC; e += 32)
            sts_v4(at + (e & (NC - 1)) * kSub + sw128_offset(n + (e / NC) / 8, (e / NC) & 7), make_uint4(0, 0, 0, 0));
        else
          for (int e = lane; e < n * 8 * NC; e += 32) {
            const uint32_t p = at + (e & (NC - 1)) * kSub + sw128_offset((e / NC) / 8, (e / NC) & 7);
            const uint4 v = lds_v4(p);
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            bool bad = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if ((w[k] & 0x7f80u) == 0x7f80u) { w[k] &= 0xffff0000u; bad = true; }
              if ((w[k] & 0x7f800000u) == 0x7f800000u) { w[k] &= 0xffffu; bad = true; }
            }
            if (bad) {
              sts_v4(p, make_uint4(w[0], w[1], w[2], w[3]));
              odd = 1;
            }
          }
        fence_proxy_async_smem();
        odd = __any_sync(kFullMask, odd);
      }
      __syncwarp();          // what all lanes wrote lies before the arrival
      if (lane == 0) {
        if (j == walk.j1 - 1) odd_values[seq & 15] = odd;
        mbar_arrive(smem_u32(&bars.ready[u % kAhead]));
        mbar_arrive(smem_u32(&bars.free[slot]));
      }
      __syncwarp();
    }
  }
}

template <int D, int STREAMS>
__global__ void __launch_bounds__(tree_tc::Shape<D, STREAMS>::kThreads, 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap tmKc, const __grid_constant__ CUtensorMap tmVc, const __grid_constant__ CUtensorMap tmK,
               const __grid_constant__ CUtensorMap tmV, const TreeParams P, const TreeAxes A, const int q_vec) {
  using namespace ptx;
  using namespace tree;
  using namespace tree_tc;
  using S = Shape<D, STREAMS>;
  constexpr int kKeys = S::KK, LOOK = 2;                // keys of a block; S is computed two blocks ahead of P V
  using Walker = Walk<kKeys>;
  typedef __nv_bfloat16 T;
  constexpr int kSlots = S::kSlots, HALVES = S::kHalves, SOFT = 4 * HALVES * STREAMS;
  constexpr int RT = STREAMS * kRows;                   // rows of the CTA's tile
  constexpr int CW = kKeys / HALVES, CH = 32, NCH = CW / CH;      // keys of a thread in a block, in pieces
  constexpr uint32_t kTile = S::kTile, kTileQ = S::kTileQ, kSub = S::kSub;
  constexpr uint32_t tO = 2 * kKeys;                    // tensor memory of a stream: two S buffers (P over the S it came from), O behind them
  extern __shared__ __align__(1024) uint8_t tree_tc_smem[];
  __shared__ int abort_flag;
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(8) Bars bars;
  __shared__ volatile int odd_values[16];               // by unit: a drafted value is not finite
  // maxima, and sums at a unit's end, of the two threads of a row
  __shared__ __align__(16) float xchg[HALVES > 1 ? STREAMS : 1][LOOK][2][HALVES > 1 ? kRows : 1];

  const uint32_t sQ0 = smem_u32(tree_tc_smem), sRing = sQ0 + STREAMS * kTileQ;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = blockIdx.x % P.tiles, group = blockIdx.x / P.tiles;
  const int rows = P.tokens * P.G, row0 = tile * RT, here = min(RT, rows - row0);     // this tile's rows
  const int streams = STREAMS == 2 && here > kRows ? 2 : 1;
  // quarters of the tensor-core tile with rows, of a stream
  auto active = [&](int s) { return max(0, min(4, (here - s * kRows + 31) / 32)); };

  if (tid == 0) {
    abort_flag = sQ0 & 1023u ? 1 : 0;                   // the tiles would be mis-swizzled: report instead of computing
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(smem_u32(&bars.full[i]), 1);
      mbar_init(smem_u32(&bars.free[i]), streams + 1);      // the products of each stream, the mending warp
    }
    for (int i = 0; i < kAhead; ++i) mbar_init(smem_u32(&bars.ready[i]), 1);
    for (int s = 0; s < streams; ++s) {
      mbar_init(smem_u32(&bars.q_full[s]), 32 * HALVES * active(s));
      for (int i = 0; i < LOOK; ++i) {
        mbar_init(smem_u32(&bars.s_full[s][i]), 1);
        mbar_init(smem_u32(&bars.p_full[s][i]), 32 * HALVES * active(s));
        mbar_init(smem_u32(&bars.pv_done[s][i]), 1);
      }
      mbar_init(smem_u32(&bars.drain[s]), 1);
    }
    fence_mbar_init();
    prefetch_tensormap(&tmKc);
    prefetch_tensormap(&tmVc);
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
  }
  grid_allow_next();
  Walker walk;
  walk.ask(P, lane);            // the lengths are on their way meanwhile
  if (warp == S::kWarps - 1) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  walk.begin(P, lane, group);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tm = tmem_slot;

  if (warp < SOFT) {
    // ------------------------------------------------------------------ softmax
    const int s = warp / (4 * HALVES), quarter = warp & 3, half = HALVES > 1 ? (warp >> 2) & 1 : 0;
    const int lane_row = quarter * 32 + lane;                                 // row of the tensor-core tile
    const int local = s * kRows + lane_row;                                   // row of the CTA's tile
    const int row = row0 + local, t = row / P.G, g = row - t * P.G;
    const bool valid = local < here;
    const uint32_t tm_lane = tm + s * 256 + ((uint32_t)(quarter * 32) << 16);
    const float scale2 = P.scale * kLog2e;
    auto pair_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + s * 4 + quarter), "n"(32 * HALVES) : "memory"); };
    const bool working = s < streams && local - lane < here;
    // Two streams: the two warps of a quarter, which share an exponential unit, take turns at it, so that one's maxima, waits and
    // transfers fall into the other's exponentials
    const bool turns = STREAMS == 2 && row0 + kRows + quarter * 32 < rows;
    auto my_turn = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + s * 4 + quarter) : "memory"); };
    auto your_turn = [&]() { asm volatile("bar.arrive %0, 64;" ::"r"(1 + (s ^ 1) * 4 + quarter) : "memory"); };
    uint32_t u = 0;
    for (int seq = 0; working && walk.unit(P); walk.next(P), ++seq) {
      // the query's row, swizzled as the products want it
      {
        const T* src = row_of<T>(P.q, walk.b, walk.h * P.G + g, t);
#pragma unroll
        for (int cc = 0; cc < D / 8 / HALVES; ++cc) {
          const int c = half * (D / 8 / HALVES) + cc;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (valid && c * 8 < P.d) {
            if (q_vec) v = *reinterpret_cast<const uint4*>(src + c * 8);
            else {
              __align__(16) T x[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) x[i] = src[c * 8 + i];
              v = *reinterpret_cast<const uint4*>(x);
            }
          }
          sts_v4(sQ0 + s * kTileQ + (c / 8) * 16384 + sw128_offset(lane_row, c & 7), v);
        }
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(&bars.q_full[s]));
      }
      // a lane without a row gives weights of zero: ones, of a query of zeros, would cost the products' power (64 / 8 heads of 128, 32
      // sequences of 16384, back to back: 274 -> 248 us)
      float m_ref = valid ? -INFINITY : INFINITY, l = 0.f;         // l: of this thread's keys
      for (int j = walk.j0; j < walk.j1; ++j, ++u) {
        const uint32_t buf = u % LOOK, phase = (u / LOOK) & 1;
        const uint32_t tS = tm_lane + buf * kKeys, tP = tS;
        const bool draft = j >= walk.cached;
        const int first = (draft ? j - walk.cached : j) * kKeys + half * CW, n = (draft ? P.tokens : walk.length) - first;
        float x[NCH][CH];
        mbar_wait_warp(smem_u32(&bars.s_full[s][buf]), phase, &abort_flag);
        tc_fence_after_sync();
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
          tmem_ld32(tS + half * CW + k * 32, x[k]);
        }
        tmem_ld_wait();
        if (draft) {
#pragma unroll
          for (int k = 0; k < NCH; ++k) {
            const uint32_t seen = valid ? seen_from(P.mask != nullptr ? P.mask + walk.b * P.m_sb + t * P.m_st : nullptr, t, first + k * CH, P.tokens) : 0;
#pragma unroll
            for (int i = 0; i < CH; ++i)
              if (!(seen >> i & 1)) x[k][i] = -INFINITY;
          }
        } else if (n < CW) {
#pragma unroll
          for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < CH; ++i)
              if (k * CH + i >= n) x[k][i] = -INFINITY;
        }
        float m = max_row<CH>(x[0]);
#pragma unroll
        for (int k = 1; k < NCH; ++k) m = fmaxf(m, max_row<CH>(x[k]));
        // the row's maximum over both threads; behind the barrier both have read their S columns
        if (HALVES > 1) {
          xchg[s][buf][half][lane_row] = m;
          pair_sync();
          m = fmaxf(m, xchg[s][buf][half ^ 1][lane_row]);
        }
        const float m2 = __fmul_rn(m, scale2);    // -inf: nothing seen
        bool need = false;
        float alpha = 1.f;
        if (m_ref == -INFINITY) {
          m_ref = m2;
        } else if (m2 > m_ref + 8.f) {
          alpha = ex2(m_ref - m2);
          m_ref = m2;
          l *= alpha;
          need = true;
        }
        float ref = m_ref == -INFINITY ? 0.f : m_ref;     // -inf - -inf must not be formed
        const bool far = is_far(ref);
        // both are rare and share a branch (far ones in one of their own: 64 tokens over 65536 rows 1.6 % slower, so 0.5 %)
        if (__any_sync(kFullMask, need || far)) {
          if (__any_sync(kFullMask, need)) {        // not in a unit's first block: there the reference was -inf
            mbar_wait_warp(smem_u32(&bars.pv_done[s][(u - 1) % LOOK]), ((u - 1) / LOOK) & 1, &abort_flag);
            tc_fence_after_sync();
#pragma unroll 1
            for (int c = half * (D / HALVES); c < (half + 1) * (D / HALVES); c += 16) {
              float o[16];
              tmem_ld16(tm_lane + tO + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= alpha;
              tmem_st16(tm_lane + tO + c, o);
            }
            tmem_st_wait();
          }
          if (far) {          // multiplied, less the reference, and back to what the exponentials multiply
            const float back = 1.f / scale2;
#pragma unroll
            for (int k = 0; k < NCH; ++k)
#pragma unroll
              for (int i = 0; i < CH; ++i) x[k][i] = __fmul_rn(__fsub_rn(__fmul_rn(x[k][i], scale2), ref), back);
            ref = 0.f;
          }
        }
        if (STREAMS == 2 && turns && (s == 1 || u > 0)) my_turn();
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
          uint32_t r[CH / 2];
          l += exp_pack_row(x[k], scale2, ref, r);       // a masked logit, -inf, gives 0
          if (STREAMS == 2 && turns && k == NCH - 1) your_turn();
          tmem_st_words(tP + half * (CW / 2) + k * 16, r);
        }
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive(smem_u32(&bars.p_full[s][buf]));
      }
      // the unit's end: O of this CTA's blocks, complete or a partial result
      mbar_wait_warp(smem_u32(&bars.pv_done[s][(u - 1) % LOOK]), ((u - 1) / LOOK) & 1, &abort_flag);
      tc_fence_after_sync();
      if (HALVES > 1) {                           // (all threads have given P of the last block, and so read its maxima)
        xchg[s][u % LOOK][half][lane_row] = l;
        pair_sync();
        l += xchg[s][u % LOOK][half ^ 1][lane_row];
      }
      const bool whole = walk.j0 == 0 && walk.j1 == walk.per_unit;
      const int64_t slot = (int64_t)blockIdx.x * 2 + (walk.j0 == 0 ? 1 : 0);
      const int u0 = max(0, walk.j0 - walk.cached) * kKeys, u1 = min(P.tokens, (walk.j1 - walk.cached) * kKeys);
      const bool odd = odd_values[seq & 15] != 0;
      // values that are not finite, of drafted rows that this row sees: columns c .. c + 7
      auto add_odd = [&](int token, int c, float* o) {
        for (int uu = u0; uu < u1; ++uu) {
          if (!sees(P, walk.b, token, uu)) continue;
          const T* v = row_of<T>(P.v, walk.b, walk.h, uu);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float z = c + i < P.d ? __bfloat162float(v[c + i]) : 0.f;
            if (!isfinite(z)) o[i] += z;
          }
        }
      };
      auto store8 = [&](int r, int token, int head, int c, float l_row, float* o) {       // columns c .. c + 7 of a row
        if (odd) add_odd(token, c, o);
        if (whole) {
          if (c < P.d) {
            const float inv = l_row > 0.f ? 1.f / l_row : (l_row == 0.f ? 0.f : l_row);      // a sum that is NaN stays NaN
            uint4 v;
            v.x = pack_bf16(o[0] * inv, o[1] * inv);
            v.y = pack_bf16(o[2] * inv, o[3] * inv);
            v.z = pack_bf16(o[4] * inv, o[5] * inv);
            v.w = pack_bf16(o[6] * inv, o[7] * inv);
            *reinterpret_cast<uint4*>(const_cast<T*>(row_of<T>(P.out, walk.b, head, token)) + c) = v;
          }
        } else {
          float4* dst = reinterpret_cast<float4*>(P.partial + (slot * RT + r) * D + c);
          dst[0] = make_float4(o[0], o[1], o[2], o[3]);
          dst[1] = make_float4(o[4], o[5], o[6], o[7]);
        }
      };
      auto store_stats = [&](int r, int token, int head, float m_row, float l_row) {
        if (!whole) P.stats[slot * RT + r] = make_float2(m_row, l_row);
        else if (P.lse != nullptr)
          P.lse[((int64_t)walk.b * P.q_heads + head) * P.tokens + token] = l_row == 0.f ? -INFINITY : (m_row + log2f(l_row)) * kLn2;
      };
#pragma unroll 1
      for (int c = half * (D / HALVES); c < (half + 1) * (D / HALVES); c += 32) {
        float o[32];
        tmem_ld32(tm_lane + tO + c, o);
        tmem_ld_wait();
        if (valid)
#pragma unroll
          for (int k = 0; k < 4; ++k) store8(local, t, walk.h * P.G + g, c + 8 * k, l, o + 8 * k);
        __syncwarp();
      }
      if (valid && half == 0) store_stats(local, t, walk.h * P.G + g, m_ref, l);
      if (HALVES > 1) pair_sync();        // both have read the sums: the next unit's first block may write the same place
    }
    if (STREAMS == 2 && turns && working && s == 0 && u > 0) my_turn();     // the last one that was given
  } else if (warp < SOFT + STREAMS) {
    // ------------------------------------------------------------------ MMA issuer of a stream
    const int s = warp - SOFT;
    if (s < streams) {
      constexpr uint32_t idS = instr_desc_bf16(128, kKeys, false, false);
      constexpr uint32_t idO = instr_desc_bf16(128, D, false, true);
      const uint32_t ts = tm + s * 256;
      const uint64_t dQ = smem_desc_sw128(sQ0 + s * kTileQ, 16);
      uint32_t u = 0, su = 0, units = 0;      // blocks whose P V, whose S has been issued
      auto issue_s = [&]() {
        const uint32_t slot = 2 * su % kSlots, round = 2 * su / kSlots;
        mbar_wait_bounded(smem_u32(&bars.full[slot]), round & 1, &abort_flag);
        __syncwarp();
        tc_fence_after_sync();
        const uint64_t dK = smem_desc_sw128(sRing + slot * kTile, 16);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_bf16_elect(ts + (su % LOOK) * kKeys, desc_advance(dQ, (k / 4) * 16384 + (k % 4) * 32),
                         desc_advance(dK, (k / 4) * kSub + (k % 4) * 32), idS, k > 0);
        mma_commit_elect(smem_u32(&bars.s_full[s][su % LOOK]));
        mma_commit_elect(smem_u32(&bars.free[slot]));
        ++su;
      };
      for (; walk.unit(P); walk.next(P), ++units) {
        const int nb = walk.j1 - walk.j0;
        mbar_wait_bounded(smem_u32(&bars.q_full[s]), units & 1, &abort_flag);
        for (int t = 0; t < LOOK && t < nb; ++t) issue_s();
        for (int t = 0; t < nb; ++t, ++u) {
          const uint32_t slot = (2 * u + 1) % kSlots;
          mbar_wait_bounded(smem_u32(&bars.ready[u % kAhead]), (u / kAhead) & 1, &abort_flag);
          mbar_wait_bounded(smem_u32(&bars.p_full[s][u % LOOK]), (u / LOOK) & 1, &abort_flag);
          __syncwarp();
          tc_fence_after_sync();
          const uint64_t dV = smem_desc_sw128(sRing + slot * kTile, kSub);
          const uint32_t tP = ts + (u % LOOK) * kKeys;
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k) mma_bf16_tmem_a_elect(ts + tO, tP + k * 8, desc_advance(dV, k * 2048), idO, t > 0 || k > 0);
          mma_commit_elect(smem_u32(&bars.pv_done[s][u % LOOK]));
          mma_commit_elect(smem_u32(&bars.free[slot]));
          if (t + LOOK < nb) issue_s();
        }
      }
      // nothing of this CTA may still be running on the tensor cores when tensor memory is freed
      mma_commit_elect(smem_u32(&bars.drain[s]));
      mbar_wait_drain(smem_u32(&bars.drain[s]), 0);
    }
  } else if (warp == SOFT + STREAMS) {
    fetch_blocks<D, kKeys, kSlots>(P, A, tmKc, tmVc, tmK, tmV, walk, sRing, bars, lane, &abort_flag);
  } else {
    mend_blocks<D, kKeys, kSlots>(P, walk, sRing, bars, odd_values, lane, &abort_flag);
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tm, 512);
  if (tid == 0 && abort_flag && P.status != nullptr) atomicOr(P.status, 1);
}

// ---- few rows: keys along the tensor-core tile's rows --------------------------------------------

// Up to 64 rows would leave most of a tile of 128 rows empty.  Here the keys of a block are its rows and the queries its columns (N, a
// multiple of 16): S^T = K Q^T [128 keys x N], O^T += V^T P^T [dim_head x N].  A thread has a key (two or four threads share one, eight or
// sixteen columns each) and exponentials for the rows there are; P^T goes through shared memory, K-major as the products want it.
//   * The reference maxima are one per column, the same for all threads, in shared memory.  While no logit exceeds its column's by
//     more than 2^8 (one vote of all softmax warps a block) nothing is reduced over the keys; else, for the first block of a unit, for
//     those behind it while a column has seen nothing but -inf or has a far reference, and for those of the drafted rows, the maxima
//     are taken, O^T and the sums rescaled.
//   * Sums stay with the threads, a key each, until a unit ends.
//   * The transposed accumulator leaves whole rows of the output side by side.
// Against the tile with rows as rows and copies of them over the keys, calls back to back: one token over 4096 rows 12.3 -> 11.6 us, 32
// x one token over 16384 (64 / 8 heads of 128) 248 -> 244 us, 8 x 16 tokens over 16384 (16 / 4 heads of 64) 39 us either way.
namespace tree_few {
constexpr int KK = 128;
template <int D, int N>
struct Shape {
  static constexpr int NC = D / 64, kParts = N == 64 ? 4 : 2;      // threads that share a key
  static constexpr int kSoftWarps = 4 * kParts, kSoft = 32 * kSoftWarps, kThreads = kSoft + 96;
  static constexpr uint32_t kTile = NC * KK * 128, kQ = NC * N * 128, kP = N * 256;      // K or V block; queries; P of a block
  static constexpr int kFit = (int)((14 * 16384 - kQ - 2 * kP) / kTile), kSlots = kFit < tree_tc::kMostSlots ? kFit : tree_tc::kMostSlots;
  static constexpr uint32_t kBytes = kSlots * kTile + kQ + 2 * kP;
};
}  // namespace tree_few

namespace tree_few {
// Over the lanes of a warp, the maximum (or the sum) of each of NT columns; lane c has that of column c (modulo NT).  Every step
// gives half of the columns away: 31 exchanges for 32 columns.
template <int NT, bool MAX>
__device__ __forceinline__ float reduce_columns(float (&v)[NT]) {
  const int lane = threadIdx.x & 31;
  auto join = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
#pragma unroll
  for (int o = NT / 2; o > 0; o >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = upper ? v[i + o] : v[i], give = upper ? v[i] : v[i + o];
      v[i] = join(keep, __shfl_xor_sync(kFullMask, give, o));
    }
  }
#pragma unroll
  for (int o = NT; o < 32; o <<= 1) v[0] = join(v[0], __shfl_xor_sync(kFullMask, v[0], o));
  return v[0];
}
}  // namespace tree_few

template <int D, int N>
__global__ void __launch_bounds__(tree_few::Shape<D, N>::kThreads, 1)
tree_few_kernel(const __grid_constant__ CUtensorMap tmKc, const __grid_constant__ CUtensorMap tmVc, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const TreeParams P, const TreeAxes A, const int q_vec) {
  using namespace ptx;
  using namespace tree;
  using tree_tc::Bars;
  using tree_tc::kAhead;
  using namespace tree_few;
  using S = Shape<D, N>;
  typedef __nv_bfloat16 T;
  constexpr int kSlots = S::kSlots, kSoftWarps = S::kSoftWarps, kSoft = S::kSoft, NT = N / S::kParts;      // NT: columns of a thread
  constexpr uint32_t kSub = KK * 128, kTile = S::kTile, tO = 2 * N;    // tensor memory: two S^T buffers, O^T
  extern __shared__ __align__(1024) uint8_t tree_few_smem[];
  __shared__ int abort_flag;
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(8) Bars bars;
  __shared__ volatile int odd_values[16];               // by unit: a drafted value is not finite
  // by column: the reference maximum (base 2; -inf: nothing seen yet), what is added to the logits (0 for that: they are all -inf, and
  // the next block's maxima are taken; -inf for a column without a row, whose weights are then zero), the factor of a rescaling, at a
  // unit's end the sum
  __shared__ __align__(16) float ref[N], off[N], factor[N], sums[N];
  __shared__ float found[4][N];                         // maxima, and sums at a unit's end, of the quarters of the keys

  const uint32_t sRing = smem_u32(tree_few_smem), sQ = sRing + kSlots * kTile, sP = sQ + S::kQ;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = blockIdx.x, here = P.tokens * P.G;   // one tile holds all rows

  if (tid == 0) {
    abort_flag = sRing & 1023u ? 1 : 0;                  // the tiles would be mis-swizzled: report instead of computing
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(smem_u32(&bars.full[i]), 1);
      mbar_init(smem_u32(&bars.free[i]), 2);                // the products, the mending warp
    }
    for (int i = 0; i < kAhead; ++i) mbar_init(smem_u32(&bars.ready[i]), 1);
    mbar_init(smem_u32(&bars.q_full[0]), kSoft);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.s_full[0][i]), 1);
      mbar_init(smem_u32(&bars.p_full[0][i]), kSoft);
      mbar_init(smem_u32(&bars.pv_done[0][i]), 1);
    }
    mbar_init(smem_u32(&bars.drain[0]), 1);
    fence_mbar_init();
    prefetch_tensormap(&tmKc);
    prefetch_tensormap(&tmVc);
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
  }
  grid_allow_next();
  Walk<KK> walk;
  walk.ask(P, lane);            // the lengths are on their way meanwhile
  if (warp == kSoftWarps) {
    tmem_alloc(smem_u32(&tmem_slot), 256);
    tmem_relinquish();
  }
  walk.begin(P, lane, group);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tm = tmem_slot;

  if (warp < kSoftWarps) {
    // ------------------------------------------------------------------ softmax
    const int quarter = warp & 3, key = quarter * 32 + lane, col0 = (warp >> 2) * NT;
    const uint32_t tm_lane = tm + ((uint32_t)(quarter * 32) << 16);
    const float scale2 = P.scale * kLog2e;
    const uint64_t scale = pack2(scale2, scale2);
    auto soft_sync = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(kSoft) : "memory"); };
    auto soft_any = [&](bool mine) {
      uint32_t any;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                   : "=r"(any) : "r"((uint32_t)mine), "n"(kSoft) : "memory");
      return any != 0;
    };
    // where this key's weight of column c lies in a P tile: rows of 64 keys, 16-byte pieces exchanged by row & 7
    uint32_t place[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) place[k] = sP + (quarter >> 1) * (N * 128) + ((((key & 63) >> 3) ^ k) << 4) + (key & 7) * 2;
    uint32_t u = 0;
    for (int seq = 0; walk.unit(P); walk.next(P), ++seq) {
      {
        constexpr int kPieces = (N * (D / 8) + kSoft - 1) / kSoft;
        uint4 v[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int e = tid + i * kSoft, r = e / (D / 8), c = e % (D / 8), t = r / P.G, g = r - t * P.G;
          v[i] = make_uint4(0, 0, 0, 0);
          if (r < here && c * 8 < P.d) {
            const T* src = row_of<T>(P.q, walk.b, walk.h * P.G + g, t) + c * 8;
            if (q_vec) v[i] = *reinterpret_cast<const uint4*>(src);
            else {
              __align__(16) T x[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] = src[k];
              v[i] = *reinterpret_cast<const uint4*>(x);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int e = tid + i * kSoft, r = e / (D / 8), c = e % (D / 8);
          if (r < N) sts_v4(sQ + (c / 8) * (N * 128) + sw128_offset(r, c & 7), v[i]);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(smem_u32(&bars.q_full[0]));
      if (tid < N) {
        ref[tid] = -INFINITY;
        off[tid] = tid < here ? 0.f : -INFINITY;
      }
      float l[NT];
#pragma unroll
      for (int c = 0; c < NT; ++c) l[c] = 0.f;
      // a column has no reference yet (all its logits were -inf), or a far one: the same for all softmax warps
      bool careful = true;
      for (int j = walk.j0; j < walk.j1; ++j, ++u) {
        const uint32_t buf = u & 1, phase = (u >> 1) & 1;
        const bool draft = j >= walk.cached;
        const int at = (draft ? j - walk.cached : j) * KK + key;       // row of the cache, or drafted row
        float x[NT];
        mbar_wait_warp(smem_u32(&bars.s_full[0][buf]), phase, &abort_flag);
        tc_fence_after_sync();
        if constexpr (NT == 8) tmem_ld8(tm_lane + buf * N + col0, x);
        else tmem_ld16(tm_lane + buf * N + col0, x);
        tmem_ld_wait();
        if (draft) {
          const uint32_t seen = seen_by<NT>(P, walk.b, col0, at);
#pragma unroll
          for (int c = 0; c < NT; ++c)
            if (!(seen >> c & 1)) x[c] = -INFINITY;
        } else if (at >= walk.length) {
#pragma unroll
          for (int c = 0; c < NT; ++c) x[c] = -INFINITY;
        }
        float y[NT];
        auto shift = [&]() {
#pragma unroll
          for (int c = 0; c < NT; c += 4) {
            const float4 o = *reinterpret_cast<const float4*>(off + col0 + c);
            unpack2(fma2(pack2(x[c], x[c + 1]), scale, pack2(o.x, o.y)), y[c], y[c + 1]);
            unpack2(fma2(pack2(x[c + 2], x[c + 3]), scale, pack2(o.z, o.w)), y[c + 2], y[c + 3]);
          }
        };
        bool renew = careful || draft;
        if (!renew) {
          shift();
          renew = soft_any(max_row<NT>(y) > 8.f);
        }
        if (renew) {
          // the columns' maxima over the keys; columns that outgrew their reference get a new one
#pragma unroll
          for (int c = 0; c < NT; ++c) y[c] = x[c];
          const float mine = reduce_columns<NT, true>(y);
          if (lane < NT) found[quarter][col0 + lane] = mine;
          soft_sync();
          if (tid < here) {
            const float m = fmaxf(fmaxf(found[0][tid], found[1][tid]), fmaxf(found[2][tid], found[3][tid]));
            const float m2 = __fmul_rn(m, scale2), old = ref[tid];
            const bool grown = old == -INFINITY ? m2 > old || m2 != m2 : m2 > old + 8.f;
            factor[tid] = grown && old != -INFINITY ? ex2(old - m2) : 1.f;
            if (grown) { ref[tid] = m2; off[tid] = -m2; }
          } else if (tid < N) {
            factor[tid] = 1.f;
          }
          careful = soft_any(tid < here && (ref[tid] == -INFINITY || is_far(ref[tid])));
#pragma unroll
          for (int c = 0; c < NT; ++c) l[c] *= factor[col0 + c];
          if (j > walk.j0) {
            mbar_wait_warp(smem_u32(&bars.pv_done[0][(u - 1) & 1]), ((u - 1) >> 1) & 1, &abort_flag);
            tc_fence_after_sync();
#pragma unroll
            for (int c = 0; c < NT; c += 8) {
              float o[8];
              tmem_ld8(tm_lane + tO + col0 + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] *= factor[col0 + c + i];
              tmem_st8(tm_lane + tO + col0 + c, o);
            }
            tmem_st_wait();
          }
          if (!careful) shift();
          else
#pragma unroll
            for (int c = 0; c < NT; ++c) y[c] = __fadd_rn(__fmul_rn(x[c], scale2), off[col0 + c]);
        }
#pragma unroll
        for (int c = 0; c < NT; ++c) y[c] = ex2(y[c]);
#pragma unroll
        for (int c = 0; c < NT; c += 2) {
          unpack2(add2(pack2(l[c], l[c + 1]), pack2(y[c], y[c + 1])), l[c], l[c + 1]);
          const uint32_t w = pack_bf16(y[c], y[c + 1]);
          sts_u16(place[c & 7] + buf * S::kP + (col0 + c) * 128, (uint16_t)w);
          sts_u16(place[(c + 1) & 7] + buf * S::kP + (col0 + c + 1) * 128, (uint16_t)(w >> 16));
        }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        mbar_arrive(smem_u32(&bars.p_full[0][buf]));
      }
      // the unit's end: sums over the keys, then O^T of this CTA's blocks, complete or a partial result
      const float mine = reduce_columns<NT, false>(l);
      if (lane < NT) found[quarter][col0 + lane] = mine;
      soft_sync();
      const bool whole = walk.j0 == 0 && walk.j1 == walk.per_unit;
      const int64_t slot = (int64_t)blockIdx.x * 2 + (walk.j0 == 0 ? 1 : 0);
      if (tid < here) {
        const float sum = (found[0][tid] + found[1][tid]) + (found[2][tid] + found[3][tid]);
        sums[tid] = sum;
        const int t = tid / P.G, g = tid - t * P.G;
        if (!whole) P.stats[slot * N + tid] = make_float2(ref[tid], sum);
        else if (P.lse != nullptr)
          P.lse[((int64_t)walk.b * P.q_heads + walk.h * P.G + g) * P.tokens + t] = sum == 0.f ? -INFINITY : (ref[tid] + log2f(sum)) * kLn2;
      }
      mbar_wait_warp(smem_u32(&bars.pv_done[0][(u - 1) & 1]), ((u - 1) >> 1) & 1, &abort_flag);
      tc_fence_after_sync();
      soft_sync();
      float o[NT];
      if constexpr (NT == 8) tmem_ld8(tm_lane + tO + col0, o);
      else tmem_ld16(tm_lane + tO + col0, o);
      tmem_ld_wait();
      // 128 features lie in 128 lanes, 64 in the first half of every quarter
      const int f = D == 128 ? key : quarter * 16 + lane;
      if (D == 128 || lane < 16) {
        const bool odd = odd_values[seq & 15] != 0;
        const int u0 = max(0, walk.j0 - walk.cached) * KK, u1 = min(P.tokens, (walk.j1 - walk.cached) * KK);
        if (odd) {           // values that are not finite, of drafted rows that a row sees
          for (int uu = u0; uu < u1; ++uu) {
            const float z = f < P.d ? __bfloat162float(row_of<T>(P.v, walk.b, walk.h, uu)[f]) : 0.f;
            if (isfinite(z)) continue;
#pragma unroll
            for (int c = 0; c < NT; ++c)
              if (col0 + c < here && sees(P, walk.b, (col0 + c) / P.G, uu)) o[c] += z;
          }
        }
        if (!whole) {
          float* dst = P.partial + (slot * N + col0) * D + f;
#pragma unroll
          for (int c = 0; c < NT; ++c)
            if (col0 + c < here) dst[c * D] = o[c];
        } else if (f < P.d) {
          int t = col0 / P.G, g = col0 - t * P.G;
          T* dst = const_cast<T*>(row_of<T>(P.out, walk.b, walk.h * P.G + g, t)) + f;
#pragma unroll
          for (int c = 0; c < NT; ++c) {
            if (col0 + c < here) {
              const float sum = sums[col0 + c], inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);      // a sum that is NaN stays NaN
              *dst = __float2bfloat16_rn(o[c] * inv);
            }
            dst += P.out.sh;
            if (++g == P.G) {            // the next token's first head
              g = 0;
              dst += P.out.sn - P.G * P.out.sh;
            }
          }
        }
      }
      soft_sync();        // sums and maxima have been read: the next unit may write the same places
    }
  } else if (warp == kSoftWarps) {
    // ------------------------------------------------------------------ MMA issuer
    constexpr uint32_t idS = instr_desc_bf16(128, N, false, false);
    constexpr uint32_t idO = instr_desc_bf16(D, N, true, false);
    const uint64_t dQ = smem_desc_sw128(sQ, 16);
    uint32_t u = 0, su = 0, units = 0;      // blocks whose O, whose S has been issued
    auto issue_s = [&]() {
      const uint32_t slot = 2 * su % kSlots, round = 2 * su / kSlots;
      mbar_wait_bounded(smem_u32(&bars.full[slot]), round & 1, &abort_flag);
      __syncwarp();
      tc_fence_after_sync();
      const uint64_t dK = smem_desc_sw128(sRing + slot * kTile, 16);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        mma_bf16_elect(tm + (su & 1) * N, desc_advance(dK, (k / 4) * kSub + (k % 4) * 32), desc_advance(dQ, (k / 4) * (N * 128) + (k % 4) * 32), idS, k > 0);
      mma_commit_elect(smem_u32(&bars.s_full[0][su & 1]));
      mma_commit_elect(smem_u32(&bars.free[slot]));
      ++su;
    };
    for (; walk.unit(P); walk.next(P), ++units) {
      const int nb = walk.j1 - walk.j0;
      mbar_wait_bounded(smem_u32(&bars.q_full[0]), units & 1, &abort_flag);
      for (int t = 0; t < 2 && t < nb; ++t) issue_s();
      for (int t = 0; t < nb; ++t, ++u) {
        const uint32_t slot = (2 * u + 1) % kSlots;
        mbar_wait_bounded(smem_u32(&bars.ready[u % kAhead]), (u / kAhead) & 1, &abort_flag);
        mbar_wait_bounded(smem_u32(&bars.p_full[0][u & 1]), (u >> 1) & 1, &abort_flag);
        __syncwarp();
        tc_fence_after_sync();
        const uint64_t dV = smem_desc_sw128(sRing + slot * kTile, kSub), dP = smem_desc_sw128(sP + (u & 1) * S::kP, 16);
#pragma unroll
        for (int k = 0; k < KK / 16; ++k)
          mma_bf16_elect(tm + tO, desc_advance(dV, k * 2048), desc_advance(dP, (k / 4) * (N * 128) + (k % 4) * 32), idO, t > 0 || k > 0);
        mma_commit_elect(smem_u32(&bars.pv_done[0][u & 1]));
        mma_commit_elect(smem_u32(&bars.free[slot]));
        if (t + 2 < nb) issue_s();
      }
    }
    // nothing of this CTA may still be running on the tensor cores when tensor memory is freed
    mma_commit_elect(smem_u32(&bars.drain[0]));
    mbar_wait_drain(smem_u32(&bars.drain[0]), 0);
  } else if (warp == kSoftWarps + 1) {
    fetch_blocks<D, KK, kSlots>(P, A, tmKc, tmVc, tmK, tmV, walk, sRing, bars, lane, &abort_flag);
  } else {
    mend_blocks<D, KK, kSlots>(P, walk, sRing, bars, odd_values, lane, &abort_flag);
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == kSoftWarps) tmem_dealloc(tm, 256);
  if (tid == 0 && abort_flag && P.status != nullptr) atomicOr(P.status, 1);
}

// ---- joining the partial results -----------------------------------------------------------

// WARPS warps per row of a unit that more than one group of CTAs worked on, each takes every WARPS-th group; eight warps a block.
// Few rows with many partials (one token over a long cache: 32 rows of 34 partials, 22 us with a warp a row) need all of a block's
// warps for a row, many rows have few partials each.
template <typename T, int DP, int RT, int KB, int WARPS>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeParams P) {
  using namespace tree;
  constexpr int C = DP / 32, ROWS = 8 / WARPS;
  __shared__ __align__(16) float sums[WARPS > 1 ? 8 : 1][DP];
  __shared__ float2 parts[WARPS > 1 ? 8 : 1];          // maximum, sum
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % WARPS;
  const int rows = P.tokens * P.G;
  const int b = blockIdx.y / P.kv_heads, h = blockIdx.y - b * P.kv_heads;
  int64_t before, total;
  count_blocks<KB>(P, lane, b, before, total);
  const int groups = busy_groups(P, total);
  const int per_unit = cache_blocks<KB>(P, b) + draft_blocks<KB>(P);
  const int64_t unit0 = before + (int64_t)h * per_unit;
  const int g0 = group_of(total, unit0, groups), g1 = group_of(total, unit0 + per_unit - 1, groups);
  ptx::grid_wait();                          // on every path: what follows in the stream waits for this kernel alone
  if (g0 == g1) return;                      // written as a whole (the same for all of a block)
  // (a block's warps stay together: with several of them a row there is a barrier in the loop)
  for (int row0 = blockIdx.x * ROWS; row0 < rows; row0 += gridDim.x * ROWS) {
    const int row = row0 + warp / WARPS;
    const bool there = row < rows;
    const int tile = (there ? row : 0) / RT, local = (there ? row : 0) - tile * RT;
    auto slot_of = [&](int g) { return ((int64_t)g * P.tiles + tile) * 2 + (g == g0 ? 1 : 0); };

    // four partials at a time, statistics and sums of all of them under way together, joined with a running maximum
    float o[C], l = 0.f, top = -INFINITY;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
#pragma unroll 1
    for (int first = g0 + part; first <= g1; first += 4 * WARPS) {
      float2 st[4];
      __align__(16) float v[4][C];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int g = first + k * WARPS;
        const int64_t at = slot_of(min(g, g1)) * RT + local;      // (the last one again where there are fewer)
        st[k] = P.stats[at];
        if constexpr (C == 4) *reinterpret_cast<float4*>(v[k]) = *reinterpret_cast<const float4*>(P.partial + at * DP + lane * C);
        else *reinterpret_cast<float2*>(v[k]) = *reinterpret_cast<const float2*>(P.partial + at * DP + lane * C);
      }
      const float before = top;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = fmaxf(top, st[k].x);
      const float ref = top == -INFINITY ? 0.f : top, a = exp2f(before - ref);
      l *= a;
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] *= a;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (first + k * WARPS > g1) break;
        const float w = exp2f(st[k].x - ref);
        l += st[k].y * w;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] += v[k][c] * w;
      }
    }
    if constexpr (WARPS > 1) {
#pragma unroll
      for (int c = 0; c < C; ++c) sums[warp][lane * C + c] = o[c];
      if (lane == 0) parts[warp] = make_float2(top, l);
      __syncthreads();
      if (part == 0) {
#pragma unroll
        for (int k = 1; k < WARPS; ++k) top = fmaxf(top, parts[warp + k].x);
        const float ref = top == -INFINITY ? 0.f : top;
        l = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
          const float w = exp2f(parts[warp + k].x - ref);
          l += parts[warp + k].y * w;
#pragma unroll
          for (int c = 0; c < C; ++c) o[c] += sums[warp + k][lane * C + c] * w;
        }
      }
      __syncthreads();
    }
    if (!there || part > 0) continue;
    const int t = row / P.G, g = row - t * P.G;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);      // a sum that is NaN stays NaN
    T* out = const_cast<T*>(row_of<T>(P.out, b, h * P.G + g, t));
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (lane * C + c < P.d) out[lane * C + c] = Elem<T>::from_float(o[c] * inv);
    if (lane == 0 && P.lse != nullptr)
      P.lse[((int64_t)b * P.q_heads + h * P.G + g) * P.tokens + t] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
  }
}

// ---- host ------------------------------------------------------------------------------------

struct TreePlan {
  bool tensor_cores;
  int DP, RT, KB;            // padded dim_head, rows of a tile, keys of a block
  int tiles, groups;
  int64_t partial_bytes, bytes;
};

// Rows that TMA can fetch: 16-byte boundaries, strides the tiled format holds
static bool tma_rows(const RowView& r, int64_t n) {
  auto fits = [](int64_t s) { return s >= 0 && s % 8 == 0 && s < (1LL << 38); };
  return (reinterpret_cast<uintptr_t>(r.p) & 15u) == 0 && fits(r.sb) && fits(r.sh) && fits(r.sn) && (r.sn > 0 || n <= 1);
}

static bool tc_serves(const TreeParams& P, int dtype) {
  return dtype == NSA_BF16 && P.scale >= 1e-30f && P.scale <= 1e30f && tma_rows(P.k, P.tokens) && tma_rows(P.v, P.tokens) &&
         (P.capacity == 0 || (tma_rows(P.kc, P.capacity) && tma_rows(P.vc, P.capacity))) &&
         (reinterpret_cast<uintptr_t>(P.out.p) & 15u) == 0 && P.out.sb % 8 == 0 && P.out.sh % 8 == 0 && P.out.sn % 8 == 0;
}

static TreePlan plan_tree(const TreeParams& P, int dtype, int impl) {
  TreePlan p = {};
  const int64_t rows = (int64_t)P.tokens * P.G;
  p.DP = P.d <= 64 ? 64 : 128;
  p.tensor_cores = impl != NSA_IMPL_SIMT && tc_serves(P, dtype);
  int64_t ctas = num_sms();
  if (p.tensor_cores) {
    p.RT = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    p.KB = p.RT <= 64 ? tree_few::KK : tree_tc::keys(p.RT <= 128 ? 1 : 2);
  } else {
    p.RT = rows <= 8 ? 8 : rows <= 32 ? 32 : 64;
    p.KB = p.RT == 8 ? 64 : 32;
    if (p.RT > 8 || p.DP == 64) ctas *= 2;           // Shape::kPerSM
  }
  p.tiles = (int)((rows + p.RT - 1) / p.RT);
  p.groups = p.tiles >= ctas ? 1 : (int)(ctas / p.tiles);
  // no more groups than there can be blocks
  const int64_t most = (int64_t)P.batch * P.kv_heads * (((int64_t)P.capacity + p.KB - 1) / p.KB + (P.tokens + p.KB - 1) / p.KB);
  if (p.groups > most) p.groups = (int)most;
  const int64_t slots = (int64_t)p.groups * p.tiles * 2;
  p.partial_bytes = slots * p.RT * p.DP * (int64_t)sizeof(float);
  p.bytes = p.groups > 1 ? p.partial_bytes + slots * p.RT * (int64_t)sizeof(float2) : 0;
  return p;
}

int64_t tree_workspace_bytes(const TreeParams& P, int dtype, int impl) { return plan_tree(P, dtype, impl).bytes; }

#define TREE_TRY(expr)                                                        \
  do {                                                                        \
    const cudaError_t e_ = (expr);                                            \
    if (e_ != cudaSuccess) return fail((int)e_, cudaGetErrorString(e_));     \
  } while (0)

// The merge starts while the last CTAs of the kernel before it are still at work, and waits for their results
template <typename T, int DP, int RT, int KB, int WARPS>
static cudaError_t launch_merge(const TreeParams& P, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  constexpr int ROWS = 8 / WARPS;
  // a block finds its unit's place once for the rows it goes through: no more blocks than are resident at once
  const int64_t all = ((int64_t)P.tokens * P.G + ROWS - 1) / ROWS, units = (int64_t)P.batch * P.kv_heads, most = (8 * (int64_t)num_sms() + units - 1) / units;
  config.gridDim = dim3((unsigned)(all < most ? all : most), (unsigned)units);
  config.blockDim = dim3(256);
  config.stream = stream;
  cudaLaunchAttribute overlap = {};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &overlap;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, tree_merge_kernel<T, DP, RT, KB, WARPS>, P);
}

template <typename T, int DP, int RT, int KB>
static int run_merge(const TreeParams& P, const TreePlan& p, cudaStream_t stream) {
  if (p.groups > 1) {
    // partials of a row if the sequences are alike: eight warps where there are more than four, as long as the rows are few
    const int64_t units = (int64_t)P.batch * P.kv_heads;
    const bool many = p.groups > 4 * units && units * P.tokens * P.G <= 8 * num_sms();
    TREE_TRY((many ? launch_merge<T, DP, RT, KB, 8>(P, stream) : launch_merge<T, DP, RT, KB, 1>(P, stream)));
  }
  TREE_TRY(cudaGetLastError());
  count_launches(p.groups > 1 ? 2 : 1);
  return NSA_OK;
}

template <typename T, int DP, int RT>
static int run_simt(const TreeParams& P, const TreePlan& p, cudaStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T);
  auto wide = [](const RowView& r) { return (reinterpret_cast<uintptr_t>(r.p) & 15u) == 0 && r.sb % V == 0 && r.sh % V == 0 && r.sn % V == 0; };
  const int vec = wide(P.k) && wide(P.v) && (P.capacity == 0 || (wide(P.kc) && wide(P.vc)));
  constexpr int smem = tree_simt::Shape<DP, RT>::kFloats * (int)sizeof(float);
  static_assert(tree_simt::Shape<DP, RT>::kPerSM == (RT > 8 || DP == 64 ? 2 : 1) && smem <= kMaxSharedBytes, "plan_tree");
  TREE_TRY((allow_shared_memory<tree_simt_kernel<T, DP, RT>>()));
  tree_simt_kernel<T, DP, RT><<<(unsigned)(p.groups * p.tiles), tree_simt::kThreads, smem, stream>>>(P, vec);
  return run_merge<T, DP, RT, tree_simt::Shape<DP, RT>::kKeys>(P, p, stream);
}

template <typename T>
static int run_simt_typed(const TreeParams& P, const TreePlan& p, cudaStream_t stream) {
  switch (p.RT) {
    case 8: return p.DP == 64 ? run_simt<T, 64, 8>(P, p, stream) : run_simt<T, 128, 8>(P, p, stream);
    case 32: return p.DP == 64 ? run_simt<T, 64, 32>(P, p, stream) : run_simt<T, 128, 32>(P, p, stream);
    default: return p.DP == 64 ? run_simt<T, 64, 64>(P, p, stream) : run_simt<T, 128, 64>(P, p, stream);
  }
}

// Boxes of 64 features x `rows` rows of one head.  An axis of one entry, or of stride zero, is one entry in the map; `step_b` and
// `step_h` say whether coordinates move along it.
static int make_tree_map(CUtensorMap* map, const RowView& r, int B, int H, int64_t N, int d, int rows, int* step_b, int* step_h) {
  *step_b = B > 1 && r.sb > 0;
  *step_h = H > 1 && r.sh > 0;
  const uint64_t row = N > 1 ? (uint64_t)r.sn * 2 : (uint64_t)d * 2;
  const uint64_t dims[4] = {(uint64_t)d, (uint64_t)N, (uint64_t)(*step_h ? H : 1), (uint64_t)(*step_b ? B : 1)};
  const uint64_t strides[3] = {row, *step_h ? (uint64_t)r.sh * 2 : row, *step_b ? (uint64_t)r.sb * 2 : row};
  const uint32_t box[4] = {64, (uint32_t)rows, 1, 1};
  return encode_bf16_tiles(map, r.p, dims, strides, box);
}

// The kernel with its tensor maps, for blocks of KEYS keys, then the merge
template <auto Kernel, int D, int RT, int KEYS>
static int run_tiles(const TreeParams& P, const TreePlan& p, int threads, int smem, cudaStream_t stream) {
  CUtensorMap tmKc, tmVc, tmK, tmV;
  TreeAxes A = {};
  int rc = make_tree_map(&tmK, P.k, P.batch, P.kv_heads, P.tokens, P.d, KEYS, &A.k_b, &A.k_h);
  if (rc == NSA_OK) rc = make_tree_map(&tmV, P.v, P.batch, P.kv_heads, P.tokens, P.d, KEYS, &A.v_b, &A.v_h);
  tmKc = tmK; tmVc = tmV;                 // an empty cache is never looked at
  if (rc == NSA_OK && P.capacity > 0) rc = make_tree_map(&tmKc, P.kc, P.batch, P.kv_heads, P.capacity, P.d, KEYS, &A.kc_b, &A.kc_h);
  if (rc == NSA_OK && P.capacity > 0) rc = make_tree_map(&tmVc, P.vc, P.batch, P.kv_heads, P.capacity, P.d, KEYS, &A.vc_b, &A.vc_h);
  if (rc != NSA_OK) return rc;
  const int q_vec = (reinterpret_cast<uintptr_t>(P.q.p) & 15u) == 0 && P.q.sb % 8 == 0 && P.q.sh % 8 == 0 && P.q.sn % 8 == 0;
  TREE_TRY(allow_shared_memory<Kernel>());
  Kernel<<<(unsigned)(p.groups * p.tiles), threads, smem, stream>>>(tmKc, tmVc, tmK, tmV, P, A, q_vec);
  return run_merge<__nv_bfloat16, D, RT, KEYS>(P, p, stream);
}

template <int D, int STREAMS>
static int run_tc(const TreeParams& P, const TreePlan& p, cudaStream_t stream) {
  using S = tree_tc::Shape<D, STREAMS>;
  return run_tiles<tree_tc_kernel<D, STREAMS>, D, STREAMS * tree_tc::kRows, S::KK>(P, p, S::kThreads, S::kBytes, stream);
}
template <int D, int N>
static int run_few(const TreeParams& P, const TreePlan& p, cudaStream_t stream) {
  return run_tiles<tree_few_kernel<D, N>, D, N, tree_few::KK>(P, p, tree_few::Shape<D, N>::kThreads, tree_few::Shape<D, N>::kBytes, stream);
}

template <int D>
static int run_tc_rows(const TreeParams& P, const TreePlan& p, cudaStream_t stream) {
  switch (p.RT) {
    case 16: return run_few<D, 16>(P, p, stream);
    case 32: return run_few<D, 32>(P, p, stream);
    case 64: return run_few<D, 64>(P, p, stream);
    case 128: return run_tc<D, 1>(P, p, stream);
    default: return run_tc<D, 2>(P, p, stream);
  }
}

int launch_tree(TreeParams& P, int dtype, int impl, uint8_t* workspace, cudaStream_t stream) {
  const TreePlan p = plan_tree(P, dtype, impl);
  if (impl == NSA_IMPL_SM100 && !p.tensor_cores) return fail(NSA_ERR_UNSUPPORTED, "tree: not served by the tensor-core kernel");
  if ((int64_t)p.groups * p.tiles > 0x7fffffffLL || (int64_t)P.batch * P.kv_heads > 65535)
    return fail(NSA_ERR_SHAPE, "tree: too many rows, or more than 65535 KV heads over the batch");
  P.tiles = p.tiles; P.groups = p.groups;
  P.partial = reinterpret_cast<float*>(workspace);
  P.stats = reinterpret_cast<float2*>(workspace + p.partial_bytes);
  if (p.tensor_cores) return p.DP == 64 ? run_tc_rows<64>(P, p, stream) : run_tc_rows<128>(P, p, stream);
  return dtype == NSA_F32 ? run_simt_typed<float>(P, p, stream) : run_simt_typed<__nv_bfloat16>(P, p, stream);
}

}  // namespace nsa
