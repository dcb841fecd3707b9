// Tokens sorted by expert, and rows weighted and summed back to tokens: the data movement around the routed experts of
// amct_pytorch/experimental/quantization/DeepSeekV3.2/cores/models/deepseek_v3_2/modeling_deepseek_v3_2.py:522-611
// (argsort of the expert numbers, gather, weighted sum), with gradients for the calibration that runs through it
// (cores/calibrator/dsv3_calib.py).
//
//   order     : stable by expert; assignment (t, j) = flat index t * topk + j.  row_map[t, j] is its row, -1 when its
//               expert number is outside [0, experts) (held elsewhere); offsets[e] the first row of expert e,
//               offsets[experts] the rows in use.  Rows from there on are zero.
//   permute   : rows[row_map[t, j]] = x[t]                       gradient: dx[t] = sum_j drows[row_map[t, j]]
//   unpermute : out[t] = sum_j w[t, j] * rows[row_map[t, j]]     gradients: drows[row_map[t, j]] = w[t, j] * dout[t],
//               dw[t, j] = dot(dout[t], rows[row_map[t, j]])
//
// The sums run over j in order, in fp32, and are rounded once; nothing is atomic, so results repeat bit for bit.
// All of it is HBM bound: a token is read once and written topk times (or the other way round).  8191 tokens x 8 experts x
// 7168 bf16: permute 189 us (floor at the copy rate 161), weighted sum 168 (161), its two gradients 332 (305).
//
// Ranking.  Up to kFewAssignments assignments need no sort: a warp counts, for one assignment, those that come before it
// (smaller expert, or the same expert and a smaller index), in the launch that also copies the token.  Beyond that a
// counting sort: one histogram for each chunk of assignments, then every chunk adds up the histograms before it and
// ranks its own assignments by 32 at a time (match_any) against per-warp running counts.  Two launches, then the copy.
#include "common.cuh"

namespace amct {
namespace moe {

constexpr int kThreads = 256;
constexpr int kFewAssignments = 1024;
constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kRounds = 2;
constexpr int kSubChunk = kSortThreads * kRounds;          // assignments ranked at a time
constexpr int kMaxChunks = 512;
constexpr int kMaxExperts = 1024, kMaxTopk = 1024;

// expert number of assignment i, -1 when there is none here
__device__ __forceinline__ int expert_at(const void* ids, int wide, int64_t i, int experts) {
  if (wide) {
    const long long v = __ldg(reinterpret_cast<const long long*>(ids) + i);
    return v >= 0 && v < experts ? (int)v : -1;
  }
  const int v = __ldg(reinterpret_cast<const int*>(ids) + i);
  return v >= 0 && v < experts ? v : -1;
}

__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// exclusive prefix sums of count[0, n) in shared memory into first[0, n]; every thread of the block takes part
template <int THREADS>
__device__ __forceinline__ void block_exclusive_scan(const int* count, int n, int* first, int* warp_total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (n + THREADS - 1) / THREADS;
  const int lo = threadIdx.x * per, hi = lo + per < n ? lo + per : n;
  int sum = 0;
  for (int i = lo; i < hi; ++i) sum += count[i];
  int incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_sync(0xffffffffu, incl, lane >= o ? lane - o : lane);
    if (lane >= o) incl += other;
  }
  if (lane == 31) warp_total[warp] = incl;
  __syncthreads();
  int at = incl - sum;
  for (int w = 0; w < warp; ++w) at += warp_total[w];
  for (int i = lo; i < hi; ++i) {
    first[i] = at;
    at += count[i];
  }
  if (hi == n && lo < n) first[n] = at;
  __syncthreads();
}

struct Sort {
  const void* ids;
  int wide;                    // 1: int64, 0: int32
  int64_t n;                   // assignments
  int experts;
  int64_t chunk;               // assignments per block, a multiple of kSubChunk
  int* counts;                 // [chunks, experts]
  int* row_map;                // [n]
  int* offsets;                // [experts + 1]
};

__global__ void __launch_bounds__(kSortThreads) moe_count_kernel(Sort p) {
  __shared__ int hist[kMaxExperts];
  for (int e = threadIdx.x; e < p.experts; e += kSortThreads) hist[e] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * p.chunk, hi = lo + p.chunk < p.n ? lo + p.chunk : p.n;
  for (int64_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
    const int e = expert_at(p.ids, p.wide, i, p.experts);
    if (e >= 0) atomicAdd(&hist[e], 1);          // integer counts: their order does not show
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kSortThreads) p.counts[(int64_t)blockIdx.x * p.experts + e] = hist[e];
}

__global__ void __launch_bounds__(kSortThreads) moe_rank_kernel(Sort p, int chunks) {
  __shared__ int count[kMaxExperts], ahead_of_me[kMaxExperts], base[kMaxExperts + 1], warp_total[kSortWarps];
  AMCT_DYNAMIC_SMEM(int, whist);                 // [kSortWarps][experts]: running counts of every warp
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < p.experts; e += kSortThreads) {
    int total = 0, before = 0;
#pragma unroll 8
    for (int c = 0; c < chunks; ++c) {
      const int v = p.counts[(int64_t)c * p.experts + e];
      total += v;
      before += c < (int)blockIdx.x ? v : 0;
    }
    count[e] = total;
    ahead_of_me[e] = before;
  }
  __syncthreads();
  block_exclusive_scan<kSortThreads>(count, p.experts, base, warp_total);
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e <= p.experts; e += kSortThreads) p.offsets[e] = base[e];
    __syncthreads();
  }
  for (int e = threadIdx.x; e < p.experts; e += kSortThreads) base[e] += ahead_of_me[e];
  const int64_t lo = (int64_t)blockIdx.x * p.chunk, hi = lo + p.chunk < p.n ? lo + p.chunk : p.n;
  int* mine = whist + warp * p.experts;
  for (int64_t sub = lo; sub < hi; sub += kSubChunk) {
    for (int i = threadIdx.x; i < kSortWarps * p.experts; i += kSortThreads) whist[i] = 0;
    __syncthreads();
    const int64_t first = sub + (int64_t)warp * (32 * kRounds);
    int expert[kRounds], rank[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int64_t i = first + r * 32 + lane;
      expert[r] = i < hi ? expert_at(p.ids, p.wide, i, p.experts) : -1;
    }
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const unsigned same = __match_any_sync(0xffffffffu, expert[r]);
      const int ahead = __popc(same & ((1u << lane) - 1u));
      const int seen = expert[r] >= 0 ? mine[expert[r]] : 0;
      rank[r] = seen + ahead;
      __syncwarp();
      if (expert[r] >= 0 && ahead == 0) mine[expert[r]] = seen + __popc(same);
      __syncwarp();
    }
    __syncthreads();
    // running counts -> first row of every warp's share of every expert
    for (int e = threadIdx.x; e < p.experts; e += kSortThreads) {
      int at = base[e];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = whist[w * p.experts + e];
        whist[w * p.experts + e] = at;
        at += c;
      }
      base[e] = at;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int64_t i = first + r * 32 + lane;
      if (i < hi) p.row_map[i] = expert[r] >= 0 ? mine[expert[r]] + rank[r] : -1;
    }
    __syncthreads();
  }
}

struct Copy {
  const uint8_t* x;            // [tokens] rows of row_units units of sizeof(U) bytes
  int64_t ld_x_bytes, row_units;
  uint8_t* rows;
  int64_t ld_rows_bytes;
  const float* scales;         // [tokens, scale_cols] or null
  int64_t scale_cols, s_row, s_col;
  float* row_scales;
  int64_t o_row, o_col;
  int64_t tokens;
  int topk;
};

template <typename U> __device__ __forceinline__ U zero_unit();
template <> __device__ __forceinline__ uint4 zero_unit<uint4>() { return make_uint4(0, 0, 0, 0); }
template <> __device__ __forceinline__ uint2 zero_unit<uint2>() { return make_uint2(0, 0); }
template <> __device__ __forceinline__ unsigned zero_unit<unsigned>() { return 0; }
template <> __device__ __forceinline__ unsigned short zero_unit<unsigned short>() { return 0; }
template <> __device__ __forceinline__ unsigned char zero_unit<unsigned char>() { return 0; }

// x[token] into its rows; blockIdx.y takes a slice of the columns.  pos[j] < 0: row ~pos[j] is cleared instead, where
// CLEAR says that such entries are rows, else there is nothing to do.
template <typename U, bool CLEAR>
__device__ __forceinline__ void copy_token(const Copy& c, int64_t token, const int* pos, int64_t n) {
  const U* src = reinterpret_cast<const U*>(c.x + token * c.ld_x_bytes);
  for (int64_t i = (int64_t)blockIdx.y * kThreads + threadIdx.x; i < c.row_units; i += (int64_t)gridDim.y * kThreads) {
    const U v = __ldcs(src + i);
    for (int j = 0; j < c.topk; ++j) {
      const int p = pos[j], r = CLEAR && p < 0 ? ~p : p;
      if (r >= 0 && r < n) __stcs(reinterpret_cast<U*>(c.rows + (int64_t)r * c.ld_rows_bytes) + i, CLEAR && p < 0 ? zero_unit<U>() : v);
    }
  }
  if (c.scales && blockIdx.y == gridDim.y - 1) {
    for (int64_t i = threadIdx.x; i < c.scale_cols; i += kThreads) {
      const float v = __ldg(c.scales + token * c.s_row + i * c.s_col);
      for (int j = 0; j < c.topk; ++j) {
        const int p = pos[j], r = CLEAR && p < 0 ? ~p : p;
        if (r >= 0 && r < n) c.row_scales[(int64_t)r * c.o_row + i * c.o_col] = CLEAR && p < 0 ? 0.f : v;
      }
    }
  }
}

// rows [used, n) cleared, spread over blockIdx.x
template <typename U>
__device__ __forceinline__ void clear_rows(const Copy& c, int64_t used, int64_t n) {
  for (int64_t r = used + blockIdx.x; r < n; r += gridDim.x) {
    U* dst = reinterpret_cast<U*>(c.rows + r * c.ld_rows_bytes);
    for (int64_t i = (int64_t)blockIdx.y * kThreads + threadIdx.x; i < c.row_units; i += (int64_t)gridDim.y * kThreads) dst[i] = zero_unit<U>();
    if (c.scales && blockIdx.y == gridDim.y - 1)
      for (int64_t i = threadIdx.x; i < c.scale_cols; i += kThreads) c.row_scales[r * c.o_row + i * c.o_col] = 0.f;
  }
}

// Few assignments: ranking and copy in one launch.  Block t < tokens owns a token; block `tokens` writes the offsets.  An
// assignment without an expert is ranked behind all others: its place is one of the rows to clear.
template <typename U>
__global__ void __launch_bounds__(kThreads) moe_few_kernel(Sort p, Copy c) {
  __shared__ int pos[kFewAssignments];
  __shared__ int hist[kMaxExperts], first[kMaxExperts + 1], warp_total[kThreads / 32];
  const int n = (int)p.n;
  if ((int64_t)blockIdx.x < c.tokens) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int j = warp; j < c.topk; j += kThreads / 32) {
      const int me = (int)blockIdx.x * c.topk + j;
      const int e = expert_at(p.ids, p.wide, me, p.experts);
      int ahead = 0;
      for (int i = lane; i < n; i += 32) {
        const int o = expert_at(p.ids, p.wide, i, p.experts);
        // as unsigned numbers -1 is the largest expert
        ahead += (unsigned)o < (unsigned)e || (o == e && i < me) ? 1 : 0;
      }
      ahead = warp_sum(ahead);
      if (lane == 0) {
        pos[j] = e >= 0 ? ahead : ~ahead;
        if (blockIdx.y == 0) p.row_map[me] = e >= 0 ? ahead : -1;
      }
    }
    __syncthreads();
    copy_token<U, true>(c, blockIdx.x, pos, n);
  } else {
    for (int e = threadIdx.x; e < p.experts; e += kThreads) hist[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int e = expert_at(p.ids, p.wide, i, p.experts);
      if (e >= 0) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    block_exclusive_scan<kThreads>(hist, p.experts, first, warp_total);
    if (blockIdx.y == 0)
      for (int e = threadIdx.x; e <= p.experts; e += kThreads) p.offsets[e] = first[e];
  }
}

template <typename U>
__global__ void __launch_bounds__(kThreads) moe_copy_kernel(Copy c, const int* row_map, const int* used, int64_t n) {
  copy_token<U, false>(c, blockIdx.x, row_map + (int64_t)blockIdx.x * c.topk, n);
  const int have = __ldg(used);
  clear_rows<U>(c, have < 0 ? 0 : have, n);
}

// ---------------------------------------------------------------------------------------------- back to tokens
__device__ __forceinline__ float weight_at(const void* w, int dtype, int64_t i) {
  switch (dtype) {
    case AMCT_DTYPE_F16: return __half2float(reinterpret_cast<const __half*>(w)[i]);
    case AMCT_DTYPE_BF16: return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
    default: return reinterpret_cast<const float*>(w)[i];
  }
}

struct Combine {
  const void* rows;
  int64_t n_rows, hidden, ld_rows;
  int topk;
  const int* row_map;
  const void* weights;         // [tokens, topk] or null: ones
  int weight_dtype;
  void* out;
  int64_t ld_out;
};

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// rows pass through once: streaming loads and stores
template <typename P> __device__ __forceinline__ P ld_pack(const void* p) {
  P r;
  if constexpr (sizeof(P) == 16) *reinterpret_cast<uint4*>(&r) = __ldcs(reinterpret_cast<const uint4*>(p));
  else r = *reinterpret_cast<const P*>(p);
  return r;
}
template <typename P> __device__ __forceinline__ void st_pack(void* p, const P& v) {
  if constexpr (sizeof(P) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
  else *reinterpret_cast<P*>(p) = v;
}

// acc += sum over u < U of wt[u] * rows[pos[u]], columns [V i, V i + V).  All U loads are issued before the first is used,
// without a branch between them: an assignment without a row reads row 0 and is left out by a select.
template <typename T, int V, int U>
__device__ __forceinline__ void combine_some(const T* rows, int64_t ld, int64_t i, const int* pos, const float* wt, float (&acc)[V]) {
  Pack<T, V> y[U];
  int r[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    r[u] = pos[u];
    y[u] = ld_pack<Pack<T, V>>(rows + (int64_t)max(r[u], 0) * ld + i * V);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float w = wt[u];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float sum = __fmaf_rn(w, ElemTraits<T>::to_f(y[u].v[e]), acc[e]);
      acc[e] = r[u] >= 0 ? sum : acc[e];
    }
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) moe_combine_kernel(Combine p) {
  __shared__ int pos[kMaxTopk];
  __shared__ float wt[kMaxTopk];
  const int64_t token = blockIdx.x;
  for (int j = threadIdx.x; j < p.topk; j += kThreads) {
    const int64_t i = token * p.topk + j;
    const int r = p.row_map[i];
    pos[j] = r >= 0 && r < p.n_rows ? r : -1;
    wt[j] = p.weights ? weight_at(p.weights, p.weight_dtype, i) : 1.f;
  }
  __syncthreads();
  const T* rows = reinterpret_cast<const T*>(p.rows);
  T* out = reinterpret_cast<T*>(p.out) + token * p.ld_out;
  const int64_t vecs = p.hidden / V;             // V == 1 unless it divides the row
  for (int64_t i = (int64_t)blockIdx.y * kThreads + threadIdx.x; i < vecs; i += (int64_t)gridDim.y * kThreads) {
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    if (p.n_rows > 0) {
      int j = 0;
      for (; j + 8 <= p.topk; j += 8) combine_some<T, V, 8>(rows, p.ld_rows, i, pos + j, wt + j, acc);
      switch (p.topk - j) {                      // what is left in one go too: 4 + 2 rows are 10 % slower than 6
        case 7: combine_some<T, V, 7>(rows, p.ld_rows, i, pos + j, wt + j, acc); break;
        case 6: combine_some<T, V, 6>(rows, p.ld_rows, i, pos + j, wt + j, acc); break;
        case 5: combine_some<T, V, 5>(rows, p.ld_rows, i, pos + j, wt + j, acc); break;
        case 4: combine_some<T, V, 4>(rows, p.ld_rows, i, pos + j, wt + j, acc); break;
        case 3: combine_some<T, V, 3>(rows, p.ld_rows, i, pos + j, wt + j, acc); break;
        case 2: combine_some<T, V, 2>(rows, p.ld_rows, i, pos + j, wt + j, acc); break;
        case 1: combine_some<T, V, 1>(rows, p.ld_rows, i, pos + j, wt + j, acc); break;
      }
    }
    Pack<T, V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.v[e] = ElemTraits<T>::from_f(acc[e]);
    st_pack(out + i * V, o);
  }
}

struct CombineBackward {
  const void* grad_out;        // [tokens, hidden]
  const void* rows;            // [n_rows, hidden]; needed for grad_weights
  int64_t n_rows, hidden, ld_grad, ld_rows;
  int topk;
  const int* row_map;
  const int* used;             // rows in use: the rest of grad_rows is cleared
  const void* weights;         // or null: ones
  int weight_dtype;
  void* grad_rows;             // or null
  int64_t ld_grad_rows;
  void* grad_weights;          // [tokens, topk] in weight_dtype, or null
};

// U assignments of a token, from pos / wt on: their rows' gradients and the dot products for their weights' gradients
// (part: [kThreads / 32][8] in shared memory).  The whole block takes part.
template <typename T, int V, int U>
__device__ __forceinline__ void backward_some(const CombineBackward& p, const T* g_row, int64_t first, const int* pos, const float* wt,
                                              float (*part)[8]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* rows = reinterpret_cast<const T*>(p.rows);
  T* grad_rows = reinterpret_cast<T*>(p.grad_rows);
  const int64_t vecs = p.hidden / V;
  int r[U];
  float w[U], dot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    r[u] = pos[u];
    w[u] = wt[u];
    dot[u] = 0.f;
  }
  for (int64_t i = threadIdx.x; i < vecs; i += kThreads) {
    const Pack<T, V> g = *reinterpret_cast<const Pack<T, V>*>(g_row + i * V);
    if (p.grad_weights && p.n_rows > 0) {
      Pack<T, V> y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) y[u] = ld_pack<Pack<T, V>>(rows + (int64_t)max(r[u], 0) * p.ld_rows + i * V);
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int e = 0; e < V; ++e) dot[u] = __fmaf_rn(ElemTraits<T>::to_f(g.v[e]), ElemTraits<T>::to_f(y[u].v[e]), dot[u]);
      }
    }
    if (grad_rows) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        Pack<T, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) o.v[e] = ElemTraits<T>::from_f(__fmul_rn(w[u], ElemTraits<T>::to_f(g.v[e])));
        if (r[u] >= 0) st_pack(grad_rows + (int64_t)r[u] * p.ld_grad_rows + i * V, o);
      }
    }
  }
  if (p.grad_weights) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], o);
      if (lane == 0) part[warp][u] = r[u] >= 0 ? dot[u] : 0.f;      // what was read for an absent row is left out here
    }
    __syncthreads();
    if (threadIdx.x < U) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k) sum += part[k][threadIdx.x];
      const int64_t i = first + threadIdx.x;
      switch (p.weight_dtype) {
        case AMCT_DTYPE_F16: reinterpret_cast<__half*>(p.grad_weights)[i] = __float2half_rn(sum); break;
        case AMCT_DTYPE_BF16: reinterpret_cast<__nv_bfloat16*>(p.grad_weights)[i] = __float2bfloat16_rn(sum); break;
        default: reinterpret_cast<float*>(p.grad_weights)[i] = sum;
      }
    }
    __syncthreads();
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 4) moe_combine_backward_kernel(CombineBackward p) {
  __shared__ int pos[kMaxTopk];
  __shared__ float wt[kMaxTopk];
  __shared__ float part[kThreads / 32][8];
  const int64_t token = blockIdx.x, first = token * p.topk;
  for (int j = threadIdx.x; j < p.topk; j += kThreads) {
    const int r = p.row_map[first + j];
    pos[j] = r >= 0 && r < p.n_rows ? r : -1;
    wt[j] = p.weights ? weight_at(p.weights, p.weight_dtype, first + j) : 1.f;
  }
  __syncthreads();
  const T* g_row = reinterpret_cast<const T*>(p.grad_out) + token * p.ld_grad;
  T* grad_rows = reinterpret_cast<T*>(p.grad_rows);
  const int64_t vecs = p.hidden / V;
  int j = 0;
  for (; j + 8 <= p.topk; j += 8) backward_some<T, V, 8>(p, g_row, first + j, pos + j, wt + j, part);
  switch (p.topk - j) {
    case 7: backward_some<T, V, 7>(p, g_row, first + j, pos + j, wt + j, part); break;
    case 6: backward_some<T, V, 6>(p, g_row, first + j, pos + j, wt + j, part); break;
    case 5: backward_some<T, V, 5>(p, g_row, first + j, pos + j, wt + j, part); break;
    case 4: backward_some<T, V, 4>(p, g_row, first + j, pos + j, wt + j, part); break;
    case 3: backward_some<T, V, 3>(p, g_row, first + j, pos + j, wt + j, part); break;
    case 2: backward_some<T, V, 2>(p, g_row, first + j, pos + j, wt + j, part); break;
    case 1: backward_some<T, V, 1>(p, g_row, first + j, pos + j, wt + j, part); break;
  }
  if (grad_rows) {
    const int used = __ldg(p.used);
    for (int64_t r = (used < 0 ? 0 : used) + (int64_t)blockIdx.x; r < p.n_rows; r += gridDim.x) {
      Pack<T, V> z;
#pragma unroll
      for (int e = 0; e < V; ++e) z.v[e] = ElemTraits<T>::from_f(0.f);
      for (int64_t i = threadIdx.x; i < vecs; i += kThreads) *reinterpret_cast<Pack<T, V>*>(grad_rows + r * p.ld_grad_rows + i * V) = z;
    }
  }
}

// ---------------------------------------------------------------------------------------------- host side
static int64_t sort_chunk(int64_t n) {
  const int64_t subs = (n + kSubChunk - 1) / kSubChunk;
  return ((subs + kMaxChunks - 1) / kMaxChunks) * kSubChunk;
}
static int64_t sort_chunks(int64_t n) { return n > 0 ? (n + sort_chunk(n) - 1) / sort_chunk(n) : 0; }

template <typename U>
static int run_permute(const Sort& s, const Copy& c, cudaStream_t st) {
  const int64_t slices = (c.row_units + kThreads - 1) / kThreads;
  int64_t gy = (148 * 4 + c.tokens - 1) / c.tokens;        // a few tokens: their columns spread over the SMs
  gy = gy < 1 ? 1 : gy;
  gy = gy > slices ? slices : gy;
  gy = gy < 1 ? 1 : gy > 65535 ? 65535 : gy;
  if (s.n <= kFewAssignments) {
    AMCT_LAUNCH(dim3((unsigned)c.tokens + 1, (unsigned)gy), kThreads, st, (s, c), moe_few_kernel<U>);
    AMCT_CHECK_LAUNCH();
    return AMCT_OK;
  }
  const int chunks = (int)sort_chunks(s.n);
  const size_t smem = (size_t)kSortWarps * s.experts * sizeof(int);
  static OncePerDevice attr_set;
  if (!attr_set.run([&] { return cudaFuncSetAttribute(moe_rank_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortWarps * kMaxExperts * (int)sizeof(int)); }))
    return AMCT_ERR_CUDA;
  AMCT_LAUNCH((unsigned)chunks, kSortThreads, st, (s), moe_count_kernel);
  AMCT_LAUNCH_SMEM((unsigned)chunks, kSortThreads, smem, st, (s, chunks), moe_rank_kernel);
  AMCT_LAUNCH(dim3((unsigned)c.tokens, (unsigned)gy), kThreads, st, (c, (const int*)s.row_map, (const int*)(s.offsets + s.experts), s.n), moe_copy_kernel<U>);
  AMCT_CHECK_LAUNCH();
  return AMCT_OK;
}

template <typename T>
static int run_combine(const Combine& p, int64_t tokens, bool vec, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t vecs = vec ? p.hidden / V : p.hidden;
  const int64_t slices = (vecs + kThreads - 1) / kThreads;
  int64_t gy = (148 * 4 + tokens - 1) / tokens;
  gy = gy < 1 ? 1 : gy > slices ? slices : gy;
  gy = gy > 65535 ? 65535 : gy;
  const dim3 grid((unsigned)tokens, (unsigned)gy);
  if (vec) AMCT_LAUNCH(grid, kThreads, st, (p), moe_combine_kernel<T, V>);
  else AMCT_LAUNCH(grid, kThreads, st, (p), moe_combine_kernel<T, 1>);
  AMCT_CHECK_LAUNCH();
  return AMCT_OK;
}

template <typename T>
static int run_backward(const CombineBackward& p, int64_t tokens, bool vec, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  if (vec) AMCT_LAUNCH((unsigned)tokens, kThreads, st, (p), moe_combine_backward_kernel<T, V>);
  else AMCT_LAUNCH((unsigned)tokens, kThreads, st, (p), moe_combine_backward_kernel<T, 1>);
  AMCT_CHECK_LAUNCH();
  return AMCT_OK;
}

static bool float_dtype(int d) { return d == AMCT_DTYPE_F32 || d == AMCT_DTYPE_F16 || d == AMCT_DTYPE_BF16; }

}  // namespace moe
}  // namespace amct

extern "C" int64_t amct_moe_permute_workspace_bytes(int64_t assignments, int experts) {
  if (assignments <= amct::moe::kFewAssignments || experts <= 0) return 0;
  return amct::moe::sort_chunks(assignments) * experts * (int64_t)sizeof(int);
}

extern "C" int amct_moe_permute(const void* x, int elem_bytes, int64_t tokens, int64_t hidden, int64_t ld_x,
                                const void* expert_ids, int ids_are_int64, int topk, int experts, const float* scales,
                                int64_t scale_cols, int64_t scale_stride_row, int64_t scale_stride_col, void* rows,
                                int64_t ld_rows, float* row_scales, int64_t row_scale_stride_row,
                                int64_t row_scale_stride_col, int32_t* row_map, int32_t* offsets, void* workspace,
                                void* stream) {
  using namespace amct::moe;
  if (tokens < 0 || hidden < 0 || topk <= 0 || experts <= 0 || !offsets) return AMCT_ERR_ARG;
  if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) return AMCT_ERR_ARG;
  if (topk > kMaxTopk || experts > kMaxExperts || tokens > 0x7ffffffeLL / topk) return AMCT_ERR_UNSUPPORTED;
  if (scale_cols < 0 || (scale_cols > 0 && tokens > 0 && (!scales || !row_scales))) return AMCT_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t n = tokens * topk;
  if (tokens > 0 && (!expert_ids || !row_map || ld_x < hidden || ld_rows < hidden || (hidden > 0 && (!x || !rows)))) return AMCT_ERR_ARG;
  if (n > kFewAssignments && !workspace) return AMCT_ERR_ARG;
  Sort s{expert_ids, ids_are_int64 != 0, n, experts, sort_chunk(n > 0 ? n : 1), reinterpret_cast<int*>(workspace), row_map, offsets};
  Copy c{};
  c.x = reinterpret_cast<const uint8_t*>(x);
  c.ld_x_bytes = ld_x * elem_bytes;
  c.rows = reinterpret_cast<uint8_t*>(rows);
  c.ld_rows_bytes = ld_rows * elem_bytes;
  c.scales = scale_cols > 0 ? scales : nullptr;
  c.scale_cols = scale_cols; c.s_row = scale_stride_row; c.s_col = scale_stride_col;
  c.row_scales = row_scales; c.o_row = row_scale_stride_row; c.o_col = row_scale_stride_col;
  c.tokens = tokens; c.topk = topk;
  // the widest unit that divides a row, both strides and both addresses
  const uint64_t bytes = (uint64_t)hidden * elem_bytes;
  const uint64_t all = bytes | (uint64_t)c.ld_x_bytes | (uint64_t)c.ld_rows_bytes | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows);
  if (n == 0) {                       // nothing to copy: the offsets alone
    c.tokens = 0;
    AMCT_LAUNCH(dim3(1, 1), kThreads, st, (s, c), moe_few_kernel<unsigned char>);
    AMCT_CHECK_LAUNCH();
    return AMCT_OK;
  }
  if (all % 16 == 0) { c.row_units = bytes / 16; return run_permute<uint4>(s, c, st); }
  if (all % 8 == 0) { c.row_units = bytes / 8; return run_permute<uint2>(s, c, st); }
  if (all % 4 == 0) { c.row_units = bytes / 4; return run_permute<unsigned>(s, c, st); }
  if (all % 2 == 0) { c.row_units = bytes / 2; return run_permute<unsigned short>(s, c, st); }
  c.row_units = bytes;
  return run_permute<unsigned char>(s, c, st);
}

extern "C" int amct_moe_unpermute(const void* rows, int dtype, int64_t n_rows, int64_t tokens, int topk, int64_t hidden,
                                  int64_t ld_rows, const int32_t* row_map, const void* weights, int weight_dtype, void* out,
                                  int64_t ld_out, void* stream) {
  using namespace amct::moe;
  if (n_rows < 0 || tokens < 0 || topk <= 0 || hidden < 0 || !float_dtype(dtype)) return AMCT_ERR_ARG;
  if (weights && !float_dtype(weight_dtype)) return AMCT_ERR_ARG;
  if (tokens == 0 || hidden == 0) return AMCT_OK;
  if (ld_rows < hidden || ld_out < hidden || !row_map || !out || (n_rows > 0 && !rows)) return AMCT_ERR_ARG;
  if (topk > kMaxTopk || tokens > 0x7ffffffeLL / topk || n_rows > 0x7fffffffLL) return AMCT_ERR_UNSUPPORTED;
  Combine p{rows, n_rows, hidden, ld_rows, topk, row_map, weights, weight_dtype, out, ld_out};
  const int esize = dtype == AMCT_DTYPE_F32 ? 4 : 2;
  const bool vec = (hidden * esize) % 16 == 0 && (ld_rows * esize) % 16 == 0 && (ld_out * esize) % 16 == 0 && amct::aligned16(rows) && amct::aligned16(out);
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case AMCT_DTYPE_F32: return run_combine<float>(p, tokens, vec, st);
    case AMCT_DTYPE_F16: return run_combine<__half>(p, tokens, vec, st);
    default: return run_combine<__nv_bfloat16>(p, tokens, vec, st);
  }
}

extern "C" int amct_moe_unpermute_backward(const void* grad_out, const void* rows, int dtype, int64_t n_rows, int64_t tokens,
                                           int topk, int64_t hidden, int64_t ld_grad, int64_t ld_rows, const int32_t* row_map,
                                           const int32_t* used_rows, const void* weights, int weight_dtype, void* grad_rows,
                                           int64_t ld_grad_rows, void* grad_weights, void* stream) {
  using namespace amct::moe;
  if (n_rows < 0 || tokens < 0 || topk <= 0 || hidden < 0 || !float_dtype(dtype)) return AMCT_ERR_ARG;
  if ((weights || grad_weights) && !float_dtype(weight_dtype)) return AMCT_ERR_ARG;
  if (tokens == 0 || (!grad_rows && !grad_weights)) return AMCT_OK;
  if (!row_map || (hidden > 0 && !grad_out) || ld_grad < hidden) return AMCT_ERR_ARG;
  if (grad_rows && (!used_rows || ld_grad_rows < hidden)) return AMCT_ERR_ARG;
  if (grad_weights && n_rows > 0 && hidden > 0 && (!rows || ld_rows < hidden)) return AMCT_ERR_ARG;
  if (topk > kMaxTopk || tokens > 0x7ffffffeLL / topk || n_rows > 0x7fffffffLL) return AMCT_ERR_UNSUPPORTED;
  CombineBackward p{grad_out, rows, n_rows, hidden, ld_grad, ld_rows, topk, row_map, used_rows, weights, weight_dtype,
                    grad_rows, ld_grad_rows, grad_weights};
  const int esize = dtype == AMCT_DTYPE_F32 ? 4 : 2;
  bool vec = (hidden * esize) % 16 == 0 && (ld_grad * esize) % 16 == 0 && amct::aligned16(grad_out);
  if (grad_rows) vec = vec && (ld_grad_rows * esize) % 16 == 0 && amct::aligned16(grad_rows);
  if (grad_weights) vec = vec && (ld_rows * esize) % 16 == 0 && amct::aligned16(rows);
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case AMCT_DTYPE_F32: return run_backward<float>(p, tokens, vec, st);
    case AMCT_DTYPE_F16: return run_backward<__half>(p, tokens, vec, st);
    default: return run_backward<__nv_bfloat16>(p, tokens, vec, st);
  }
}
