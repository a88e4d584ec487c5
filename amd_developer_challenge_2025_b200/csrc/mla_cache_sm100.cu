// Operators around a paged latent cache for B200 (sm_100a): append, attend, evict (include/b200_mla_cache.h).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "b200_fp8_mm.h"
#include "b200_mla_cache.h"

namespace {

// Programmatic dependent launch: a kernel may begin while the one before it on the stream drains; it waits here before
// it touches memory, and lets the next one begin once all of its own CTAs have been scheduled. Every thread of every CTA
// waits, so that the end of a kernel is the end of all that ran before it.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16* out) { *out = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_float(float v, __half* out) { *out = __float2half_rn(v); }

// The cache as the kernels take it.
struct CacheView {
  void* data;
  const int* block_table;
  const int* lens;
  int pages, page_size, pages_per_seq, capacity;
  int dv, d;
  long long page_stride, slot_stride, table_stride;
};

// Element offset of slot j (0 <= j < capacity) of sequence b, or -1 where its page is not one of the cache's.
__device__ __forceinline__ long long slot_offset(const CacheView& c, int b, int j) {
  const int at = j / c.page_size;
  const int page = c.block_table[b * c.table_stride + at];
  if (page < 0 || page >= c.pages) return -1;
  return page * c.page_stride + static_cast<long long>(j - at * c.page_size) * c.slot_stride;
}

__device__ __forceinline__ int rows_of(const CacheView& c, int b, int most) { return max(0, min(c.lens[b], most)); }

// ---------------------------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------------------------

constexpr int kAppendThreads = 128;
constexpr int kAppendHeads = 4;  // query heads per CTA
constexpr int kMaxPairs = 224;   // dr / 2

struct AppendParams {
  CacheView cache;
  const void* row;
  const int* position;
  const void* q;
  void* q_out;
  float* score;
  int* slot_position;
  long long row_stride, q_sb, q_sh, qo_sb, qo_sh, score_stride, slot_position_stride;
  int heads, half;
  int copy;      // the elements before the rotated ones go to q_out too (0: q_out is q)
  int vec;       // every row of q, q_out and `row` starts on a 16-byte boundary
  double turns[kMaxPairs];  // theta^(-2t/dr) / (2 pi): turns per position
};

// dst[0..dv + 2 half) = src with its last 2 half elements rotated; all threads of the CTA. src may be dst (copy = 0).
template <typename T, bool VEC>
__device__ __forceinline__ void rotate_rows(const T* src, long long src_step, T* dst, long long dst_step, int rows, int dv, int half,
                                            bool copy, const float2* cs) {
  constexpr int E = VEC ? 8 : 1;
  struct alignas(sizeof(T) * E) Piece {
    T v[E];
  };
  const int nope = copy ? dv / E : 0, pairs = half / E, each = nope + pairs;
  for (int i = static_cast<int>(threadIdx.x); i < rows * each; i += kAppendThreads) {
    const int r = i / each, k = i - r * each;
    const T* s = src + r * src_step;
    T* o = dst + r * dst_step;
    if (k < nope) {
      *reinterpret_cast<Piece*>(o + k * E) = *reinterpret_cast<const Piece*>(s + k * E);
      continue;
    }
    const int t = (k - nope) * E;
    Piece a = *reinterpret_cast<const Piece*>(s + dv + t), b = *reinterpret_cast<const Piece*>(s + dv + half + t);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float x1 = to_float(a.v[e]), x2 = to_float(b.v[e]);
      const float2 w = cs[t + e];
      from_float(x1 * w.x - x2 * w.y, &a.v[e]);
      from_float(x2 * w.x + x1 * w.y, &b.v[e]);
    }
    *reinterpret_cast<Piece*>(o + dv + t) = a;
    *reinterpret_cast<Piece*>(o + dv + half + t) = b;
  }
}

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ float2 cs[kMaxPairs];
  pdl_wait();
  pdl_launch_dependents();
  const CacheView& c = p.cache;
  const int b = static_cast<int>(blockIdx.y);
  const int position = p.position[b];
  for (int t = static_cast<int>(threadIdx.x); t < p.half; t += kAppendThreads) {
    // In 64 bits up to the whole turns, which no function of the angle sees: position 10^6 leaves 32 bits with two digits.
    const double turns = position * p.turns[t];
    float s, co;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &co);
    cs[t] = make_float2(co, s);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    const int j = c.lens[b];
    if (j < 0 || j >= c.capacity) return;
    const long long at = slot_offset(c, b, j);
    if (at < 0) return;
    const T* src = static_cast<const T*>(p.row) + b * p.row_stride;
    T* dst = static_cast<T*>(c.data) + at;
    if (p.vec)
      rotate_rows<T, true>(src, 0, dst, 0, 1, c.dv, p.half, true, cs);
    else
      rotate_rows<T, false>(src, 0, dst, 0, 1, c.dv, p.half, true, cs);
    if (threadIdx.x == 0) {
      if (p.score != nullptr) p.score[b * p.score_stride + j] = 0.f;
      if (p.slot_position != nullptr) p.slot_position[b * p.slot_position_stride + j] = position;
    }
    return;
  }
  const int h0 = (static_cast<int>(blockIdx.x) - 1) * kAppendHeads, rows = min(kAppendHeads, p.heads - h0);
  const T* src = static_cast<const T*>(p.q) + b * p.q_sb + h0 * p.q_sh;
  T* dst = static_cast<T*>(p.q_out) + b * p.qo_sb + h0 * p.qo_sh;
  if (p.vec)
    rotate_rows<T, true>(src, p.q_sh, dst, p.qo_sh, rows, c.dv, p.half, p.copy != 0, cs);
  else
    rotate_rows<T, false>(src, p.q_sh, dst, p.qo_sh, rows, c.dv, p.half, p.copy != 0, cs);
}

// ---------------------------------------------------------------------------------------------
// Attend
// ---------------------------------------------------------------------------------------------

constexpr float kLn2 = 0.69314718055994531f, kLog2E = 1.4426950408889634f;
constexpr int kMaxD = 576;
constexpr int kAttendThreads = 256;
constexpr int kAttendWarps = kAttendThreads / 32;
constexpr int kLaneD = kMaxD / 32;
constexpr int kLaneV = 512 / 32;

struct AttendParams {
  CacheView cache;
  const void* q;
  void* out;
  float* lse;  // [batch][heads]
  const float* score;
  float* score_out;
  long long q_sb, q_sh, out_sb, out_sh, score_stride, score_out_stride;
  int heads, max_len;
  float scale_log2;  // scale * log2(e)
};

// scale * log2(e) * (q . row of slot j), the same value in every lane
template <typename T>
__device__ __forceinline__ float logit(const CacheView& c, const float (&q)[kLaneD], int b, int j, int lane, float scale_log2,
                                       float (&x)[kLaneD]) {
  const long long at = slot_offset(c, b, j);
  const T* row = static_cast<const T*>(c.data) + at;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kLaneD; ++i) {
    const int e = lane + 32 * i;
    x[i] = (at >= 0 && e < c.d) ? to_float(row[e]) : 0.f;
    s += q[i] * x[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s * scale_log2;
}

// One CTA per (head, sequence): the warps share the rows, each with its own running maximum, sum and weighted sum.
template <typename T>
__global__ void __launch_bounds__(kAttendThreads) attend_kernel(const __grid_constant__ AttendParams p) {
  __shared__ float part[kAttendWarps][512];
  __shared__ float2 stat[kAttendWarps];
  pdl_wait();
  pdl_launch_dependents();
  const CacheView& c = p.cache;
  const int h = static_cast<int>(blockIdx.x), b = static_cast<int>(blockIdx.y);
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  const int n = rows_of(c, b, p.max_len);
  const T* qrow = static_cast<const T*>(p.q) + b * p.q_sb + h * p.q_sh;
  float q[kLaneD], x[kLaneD], acc[kLaneV] = {};
#pragma unroll
  for (int i = 0; i < kLaneD; ++i) q[i] = lane + 32 * i < c.d ? to_float(qrow[lane + 32 * i]) : 0.f;
  float m = -INFINITY, l = 0.f;
  for (int j = warp; j < n; j += kAttendWarps) {
    const float s = logit<T>(c, q, b, j, lane, p.scale_log2, x);
    const float top = fmaxf(m, s);
    const float base = top == -INFINITY ? 0.f : top;
    const float keep = exp2f(m - base), w = exp2f(s - base);
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < kLaneV; ++i) acc[i] = acc[i] * keep + w * x[i];
    m = top;
  }
#pragma unroll
  for (int i = 0; i < kLaneV; ++i) part[warp][lane + 32 * i] = acc[i];
  if (lane == 0) stat[warp] = make_float2(m, l);
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < kAttendWarps; ++w) top = fmaxf(top, stat[w].x);
  const float base = top == -INFINITY ? 0.f : top;
  for (int w = 0; w < kAttendWarps; ++w) sum += stat[w].y * exp2f(stat[w].x - base);
  T* out = static_cast<T*>(p.out) + b * p.out_sb + h * p.out_sh;
  for (int e = static_cast<int>(threadIdx.x); e < c.dv; e += kAttendThreads) {
    float v = 0.f;
    for (int w = 0; w < kAttendWarps; ++w) v += part[w][e] * exp2f(stat[w].x - base);
    from_float(n == 0 ? 0.f : v / sum, &out[e]);
  }
  if (threadIdx.x == 0) p.lse[static_cast<long long>(b) * p.heads + h] = n == 0 ? -INFINITY : (base + log2f(sum)) * kLn2;
}

// score_out = score + the weights of all heads: one warp per slot.
template <typename T>
__global__ void __launch_bounds__(kAttendThreads) attend_score_kernel(const __grid_constant__ AttendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const CacheView& c = p.cache;
  const int b = static_cast<int>(blockIdx.y), lane = static_cast<int>(threadIdx.x) & 31;
  const int j = static_cast<int>(blockIdx.x) * kAttendWarps + (static_cast<int>(threadIdx.x) >> 5);
  if (j >= rows_of(c, b, p.max_len)) return;
  float sum = 0.f, q[kLaneD], x[kLaneD];
  for (int h = 0; h < p.heads; ++h) {
    const T* qrow = static_cast<const T*>(p.q) + b * p.q_sb + h * p.q_sh;
#pragma unroll
    for (int i = 0; i < kLaneD; ++i) q[i] = lane + 32 * i < c.d ? to_float(qrow[lane + 32 * i]) : 0.f;
    const float s = logit<T>(c, q, b, j, lane, p.scale_log2, x);
    sum += exp2f(s - p.lse[static_cast<long long>(b) * p.heads + h] * kLog2E);
  }
  if (lane == 0) p.score_out[b * p.score_out_stride + j] = p.score[b * p.score_stride + j] + sum;
}

// ---------------------------------------------------------------------------------------------
// Evict
// ---------------------------------------------------------------------------------------------

constexpr int kSelectThreads = 1024;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kMoveThreads = 256;

struct EvictParams {
  CacheView cache;
  const float* score;
  const int* position;
  int* lens_out;
  float* score_out;
  int* position_out;
  long long score_stride, position_stride, score_out_stride, position_out_stride;
  int budget, recent;
  int* moves;    // [batch]: how many rows of each sequence move
  int* holes;    // [batch][most]: slots given up below the budget, ascending
  int* late;     // [batch][most]: slots kept behind it, ascending
  int most;
  int vecs;      // 16-byte pieces of a row
};

// Order of the scores as unsigned integers: protected rows above all, NaN above every number, -0 as 0.
__device__ __forceinline__ uint32_t rank_of(float score, int position, long long safe_above) {
  if (position > safe_above) return 0xffffffffu;
  if (score != score) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(score + 0.f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Exclusive sum over the warps' values v (one per warp, given by lane 0 through `scratch`), and the total.
__device__ __forceinline__ int warps_before(int v, int* scratch, int* total) {
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kSelectWarps; ++w) {
    if (w < warp) before += scratch[w];
    all += scratch[w];
  }
  *total = all;
  return before;
}

// One CTA per sequence: the budget-th largest rank, eight bits at a time, then the slots to fill and the slots to move.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int hist[256];
  __shared__ int scratch[kSelectWarps];
  __shared__ int found[2];
  pdl_wait();
  pdl_launch_dependents();
  const CacheView& c = p.cache;
  const int b = static_cast<int>(blockIdx.x), tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int len = c.lens[b], n = rows_of(c, b, c.capacity), budget = p.budget;
  const float* score = p.score + b * p.score_stride;
  const int* position = p.position + b * p.position_stride;
  float* score_out = p.score_out + b * p.score_out_stride;
  int* position_out = p.position_out + b * p.position_out_stride;
  __syncthreads();  // lens_out may be lens
  if (tid == 0) p.lens_out[b] = min(len, budget);
  if (n <= budget) {
    if (tid == 0) p.moves[b] = 0;
    for (int i = tid; i < n; i += kSelectThreads) {
      score_out[i] = score[i];
      position_out[i] = position[i];
    }
    return;
  }
  int newest = INT_MIN;
  for (int i = tid; i < n; i += kSelectThreads) newest = max(newest, position[i]);
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) scratch[warp] = newest;
  __syncthreads();
  for (int w = 0; w < kSelectWarps; ++w) newest = max(newest, scratch[w]);
  const long long safe_above = static_cast<long long>(newest) - p.recent;
  uint32_t bits = 0, mask = 0;
  int left = budget;  // of the rows that share `bits` under `mask`, how many are kept
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSelectThreads) {
      const uint32_t r = rank_of(score[i], position[i], safe_above);
      if ((r & mask) == bits) atomicAdd(&hist[(r >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, v = 255;
      while (above + hist[v] < left) above += hist[v--];
      found[0] = v;
      found[1] = above;
    }
    __syncthreads();
    bits |= static_cast<uint32_t>(found[0]) << shift;
    mask |= 255u << shift;
    left -= found[1];
  }
  // A warp takes a run of slots, so that what it finds is in order. Of the rows at the threshold the first `left` stay.
  const int run = (n + kSelectThreads - 1) / kSelectThreads * 32;
  const int begin = min(n, warp * run), end = min(n, begin + run);
  int total, ties = 0;
  for (int i0 = begin; i0 < end; i0 += 32) {
    const int i = i0 + lane;
    ties += __popc(__ballot_sync(0xffffffffu, i < end && rank_of(score[i], position[i], safe_above) == bits));
  }
  const int ties_before = warps_before(ties, scratch, &total);
  int holes_at = 0, late_at = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int seen = ties_before, holes = 0, late = 0;
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t r = i < end ? rank_of(score[i], position[i], safe_above) : 0u;
      const uint32_t tie = __ballot_sync(0xffffffffu, i < end && r == bits);
      const uint32_t below = (1u << lane) - 1u;
      const bool kept = i < end && (r > bits || (r == bits && seen + __popc(tie & below) < left));
      seen += __popc(tie);
      const bool hole = i < end && !kept && i < budget, moved = kept && i >= budget;
      const uint32_t hm = __ballot_sync(0xffffffffu, hole), lm = __ballot_sync(0xffffffffu, moved);
      if (pass == 1) {
        if (hole) p.holes[static_cast<long long>(b) * p.most + holes_at + holes + __popc(hm & below)] = i;
        if (moved) p.late[static_cast<long long>(b) * p.most + late_at + late + __popc(lm & below)] = i;
        if (kept && i < budget) {
          score_out[i] = score[i];
          position_out[i] = position[i];
        }
      }
      holes += __popc(hm);
      late += __popc(lm);
    }
    if (pass == 0) {
      late_at = warps_before(late, scratch, &total);
      holes_at = warps_before(holes, scratch, &total);
      if (tid == 0) p.moves[b] = total;
    }
  }
}

// A warp per moved row: the row, its score and its position.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const CacheView& c = p.cache;
  const int b = static_cast<int>(blockIdx.y), lane = static_cast<int>(threadIdx.x) & 31;
  const int warps = static_cast<int>(gridDim.x) * (kMoveThreads / 32);
  const int moves = p.moves[b];
  for (int i = static_cast<int>(blockIdx.x) * (kMoveThreads / 32) + (static_cast<int>(threadIdx.x) >> 5); i < moves; i += warps) {
    const int to = p.holes[static_cast<long long>(b) * p.most + i], of = p.late[static_cast<long long>(b) * p.most + i];
    const long long dst = slot_offset(c, b, to), src = slot_offset(c, b, of);
    if (dst >= 0) {
      uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(c.data) + dst);
      const uint4* s = reinterpret_cast<const uint4*>(static_cast<uint16_t*>(c.data) + src);
      for (int v = lane; v < p.vecs; v += 32) o[v] = src >= 0 ? s[v] : make_uint4(0u, 0u, 0u, 0u);
    }
    if (lane == 0) {
      p.score_out[b * p.score_out_stride + to] = p.score[b * p.score_stride + of];
      p.position_out[b * p.position_out_stride + to] = p.position[b * p.position_stride + of];
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------

// <<<grid, threads>>> on `stream`, allowed to begin under the kernel before it (see pdl_wait).
template <typename Params>
int launch_pdl(void (*kernel)(Params), dim3 grid, int threads, size_t smem, void* stream, const Params& params) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, params) != cudaSuccess) {
    (void)cudaGetLastError();
    return B200_FP8_MM_ERR_LAUNCH;
  }
  return B200_FP8_MM_OK;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

constexpr int kMaxBatch = 65535;  // a grid dimension

// Checks the description of a cache and turns it into what the kernels take.
int view_of(const b200_mla_cache* c, CacheView* v) {
  if (c == nullptr || c->data == nullptr || c->block_table == nullptr || c->lens == nullptr) return B200_FP8_MM_ERR_NULL;
  if (c->dtype != B200_MLA_CACHE_BF16 && c->dtype != B200_MLA_CACHE_FP16) return B200_FP8_MM_ERR_SHAPE;
  if (c->batch <= 0 || c->batch > kMaxBatch || c->pages <= 0 || c->page_size <= 0 || c->pages_per_seq <= 0) return B200_FP8_MM_ERR_SHAPE;
  if (c->dv <= 0 || c->dv % 128 != 0 || c->dv > 512 || c->dr < 0 || c->dr % 64 != 0 || c->dr > 2 * kMaxPairs || c->dv + c->dr > kMaxD)
    return B200_FP8_MM_ERR_SHAPE;
  const long long capacity = static_cast<long long>(c->pages_per_seq) * c->page_size;
  if (capacity > (1ll << 30)) return B200_FP8_MM_ERR_SHAPE;
  const int d = c->dv + c->dr;
  if (c->page_stride < d || c->slot_stride < d || c->page_stride % 8 != 0 || c->slot_stride % 8 != 0 || c->table_stride < 0)
    return B200_FP8_MM_ERR_STRIDE;
  if (!aligned16(c->data)) return B200_FP8_MM_ERR_ALIGN;
  *v = CacheView{c->data, c->block_table, c->lens, c->pages, c->page_size, c->pages_per_seq, static_cast<int>(capacity),
                 c->dv, d, c->page_stride, c->slot_stride, c->table_stride};
  return B200_FP8_MM_OK;
}

int evict_most(long long capacity, int budget) {
  const long long behind = capacity - budget;
  return static_cast<int>(behind < budget ? (behind > 0 ? behind : 0) : budget);
}

}  // namespace

extern "C" {

int b200_mla_cache_append(const b200_mla_cache* cache, const void* row, long long row_stride, const int* position,
                          double theta, const void* q, long long q_sb, long long q_sh, void* q_out, long long qo_sb,
                          long long qo_sh, int heads, float* score, long long score_stride, int* slot_position,
                          long long slot_position_stride, void* stream) {
  AppendParams p;
  const int rc = view_of(cache, &p.cache);
  if (rc != B200_FP8_MM_OK) return rc;
  if (row == nullptr || position == nullptr || (q == nullptr) != (q_out == nullptr)) return B200_FP8_MM_ERR_NULL;
  if (!(theta > 0.0) || !isfinite(theta) || (q != nullptr && (heads <= 0 || heads > (1 << 20)))) return B200_FP8_MM_ERR_SHAPE;
  p.row = row;
  p.position = position;
  p.q = q;
  p.q_out = q_out;
  p.score = score;
  p.slot_position = slot_position;
  p.row_stride = row_stride;
  p.q_sb = q_sb;
  p.q_sh = q_sh;
  p.qo_sb = qo_sb;
  p.qo_sh = qo_sh;
  p.score_stride = score_stride;
  p.slot_position_stride = slot_position_stride;
  p.heads = q != nullptr ? heads : 0;
  p.half = cache->dr / 2;
  p.copy = q != q_out || q_sb != qo_sb || q_sh != qo_sh;
  p.vec = aligned16(row) && row_stride % 8 == 0 &&
          (q == nullptr || (aligned16(q) && aligned16(q_out) && q_sb % 8 == 0 && q_sh % 8 == 0 && qo_sb % 8 == 0 && qo_sh % 8 == 0));
  for (int t = 0; t < p.half; ++t) p.turns[t] = pow(theta, -static_cast<double>(t) / p.half) / 6.283185307179586476925;
  const dim3 grid(static_cast<unsigned>(1 + (p.heads + kAppendHeads - 1) / kAppendHeads), static_cast<unsigned>(cache->batch));
  return cache->dtype == B200_MLA_CACHE_BF16 ? launch_pdl(append_kernel<__nv_bfloat16>, grid, kAppendThreads, 0, stream, p)
                                             : launch_pdl(append_kernel<__half>, grid, kAppendThreads, 0, stream, p);
}

size_t b200_mla_cache_attend_workspace_bytes(int batch, int heads, int dv, int dr, int max_len, int with_score) {
  (void)dv, (void)dr, (void)max_len, (void)with_score;
  if (batch <= 0 || heads <= 0) return 0;
  return (static_cast<size_t>(batch) * heads * sizeof(float) + 255) / 256 * 256;
}

int b200_mla_cache_attend(const b200_mla_cache* cache, const void* q, long long q_sb, long long q_sh, int heads, float scale,
                          void* out, long long out_sb, long long out_sh, float* lse, const float* score,
                          long long score_stride, float* score_out, long long score_out_stride, int max_len, void* workspace,
                          size_t workspace_bytes, int* device_status, void* stream) {
  AttendParams p;
  int rc = view_of(cache, &p.cache);
  if (rc != B200_FP8_MM_OK) return rc;
  if (q == nullptr || out == nullptr || (score_out != nullptr && score == nullptr)) return B200_FP8_MM_ERR_NULL;
  if (heads <= 0 || heads > (1 << 16) || max_len < 0 || !isfinite(scale)) return B200_FP8_MM_ERR_SHAPE;
  if (q_sb % 8 != 0 || q_sh % 8 != 0 || q_sb < 0 || q_sh < 0) return B200_FP8_MM_ERR_STRIDE;
  if (!aligned16(q)) return B200_FP8_MM_ERR_ALIGN;
  (void)device_status;
  if (max_len == 0 || max_len > p.cache.capacity) max_len = p.cache.capacity;
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 ||
      workspace_bytes < b200_mla_cache_attend_workspace_bytes(cache->batch, heads, cache->dv, cache->dr, max_len, score_out != nullptr))
    return B200_FP8_MM_ERR_WORKSPACE;
  p.q = q;
  p.out = out;
  p.lse = lse != nullptr ? lse : static_cast<float*>(workspace);
  p.score = score;
  p.score_out = score_out;
  p.q_sb = q_sb;
  p.q_sh = q_sh;
  p.out_sb = out_sb;
  p.out_sh = out_sh;
  p.score_stride = score_stride;
  p.score_out_stride = score_out_stride;
  p.heads = heads;
  p.max_len = max_len;
  p.scale_log2 = scale * kLog2E;
  const bool bf16 = cache->dtype == B200_MLA_CACHE_BF16;
  const dim3 grid(static_cast<unsigned>(heads), static_cast<unsigned>(cache->batch));
  rc = launch_pdl(bf16 ? attend_kernel<__nv_bfloat16> : attend_kernel<__half>, grid, kAttendThreads, 0, stream, p);
  if (rc != B200_FP8_MM_OK || score_out == nullptr) return rc;
  const dim3 slots(static_cast<unsigned>((max_len + kAttendWarps - 1) / kAttendWarps), static_cast<unsigned>(cache->batch));
  return launch_pdl(bf16 ? attend_score_kernel<__nv_bfloat16> : attend_score_kernel<__half>, slots, kAttendThreads, 0, stream, p);
}

size_t b200_mla_cache_evict_workspace_bytes(int batch, int capacity, int budget) {
  if (batch <= 0 || capacity <= 0 || budget <= 0) return 0;
  return (static_cast<size_t>(batch) * (1 + 2 * static_cast<size_t>(evict_most(capacity, budget))) * sizeof(int) + 255) / 256 * 256;
}

int b200_mla_cache_evict(const b200_mla_cache* cache, const float* score, long long score_stride, const int* slot_position,
                         long long slot_position_stride, int budget, int recent, int* lens_out, float* score_out,
                         long long score_out_stride, int* position_out, long long position_out_stride, void* workspace,
                         size_t workspace_bytes, void* stream) {
  EvictParams p;
  int rc = view_of(cache, &p.cache);
  if (rc != B200_FP8_MM_OK) return rc;
  if (score == nullptr || slot_position == nullptr || lens_out == nullptr || score_out == nullptr || position_out == nullptr)
    return B200_FP8_MM_ERR_NULL;
  if (budget <= 0 || recent < 0 || recent > budget) return B200_FP8_MM_ERR_SHAPE;
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 ||
      workspace_bytes < b200_mla_cache_evict_workspace_bytes(cache->batch, p.cache.capacity, budget))
    return B200_FP8_MM_ERR_WORKSPACE;
  p.score = score;
  p.position = slot_position;
  p.lens_out = lens_out;
  p.score_out = score_out;
  p.position_out = position_out;
  p.score_stride = score_stride;
  p.position_stride = slot_position_stride;
  p.score_out_stride = score_out_stride;
  p.position_out_stride = position_out_stride;
  p.budget = budget;
  p.recent = recent;
  p.most = evict_most(p.cache.capacity, budget);
  p.moves = static_cast<int*>(workspace);
  p.holes = p.moves + cache->batch;
  p.late = p.holes + static_cast<size_t>(cache->batch) * p.most;
  p.vecs = p.cache.d / 8;
  rc = launch_pdl(evict_select_kernel, dim3(static_cast<unsigned>(cache->batch)), kSelectThreads, 0, stream, p);
  if (rc != B200_FP8_MM_OK || p.most == 0) return rc;
  const int want = (p.most + kMoveThreads / 32 - 1) / (kMoveThreads / 32);
  const int fill = (148 * 8 + cache->batch - 1) / cache->batch;
  const dim3 grid(static_cast<unsigned>(want < fill ? want : fill), static_cast<unsigned>(cache->batch));
  return launch_pdl(evict_move_kernel, grid, kMoveThreads, 0, stream, p);
}

}  // extern "C"
