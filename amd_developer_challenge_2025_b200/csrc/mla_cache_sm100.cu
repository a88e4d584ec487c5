// Operators around a paged latent cache for B200 (sm_100a): append, attend, evict (include/b200_mla_cache.h).

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "b200_fp8_mm.h"
#include "b200_mla_cache.h"
#include "cache_walk.h"

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

constexpr int kAppendThreads = 256;
constexpr int kAppendHeads = 8;  // query heads per CTA
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
  double turns[kMaxPairs];  // theta^(-2t/dr) / (2 pi): turns per position
};

template <typename T, bool VEC>
struct Piece;
template <typename T>
struct alignas(16) Piece<T, true> {
  static constexpr int E = 8;
  T v[8];
};
template <typename T>
struct Piece<T, false> {
  static constexpr int E = 1;
  T v[1];
};

// `rows` rows of dv + 2 half elements from src to dst (which may be src, then copy = false), the last 2 half rotated for `position`.
// The unrotated elements, most of the bytes, are on their way while the angles are worked out.
template <typename T, bool VEC>
__device__ __forceinline__ void rotate_rows(const AppendParams& p, const T* src, long long src_step, T* dst, long long dst_step, int rows, int dv,
                                            bool copy, int position, float2* cs) {
  using P = Piece<T, VEC>;
  constexpr int E = P::E, kAhead = 2;
  const int tid = static_cast<int>(threadIdx.x), half = p.half, each = dv / E, nope = copy ? rows * each : 0;
  auto at = [&](int i, const T** s, T** o) {
    const int r = i / each, k = i - r * each;
    *s = src + r * src_step + k * E;
    *o = dst + r * dst_step + k * E;
  };
  P ahead[kAhead];
#pragma unroll
  for (int n = 0; n < kAhead; ++n) {
    const T* s;
    T* o;
    at(tid + n * kAppendThreads, &s, &o);
    if (tid + n * kAppendThreads < nope) ahead[n] = *reinterpret_cast<const P*>(s);
  }
  for (int t = tid; t < half; t += kAppendThreads) {
    // In 64 bits up to the whole turns, which no function of the angle sees: position 10^6 leaves 32 bits with two digits.
    const double turns = position * p.turns[t];
    float sn, co;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sn, &co);
    cs[t] = make_float2(co, sn);
  }
#pragma unroll
  for (int n = 0; n < kAhead; ++n) {
    const T* s;
    T* o;
    at(tid + n * kAppendThreads, &s, &o);
    if (tid + n * kAppendThreads < nope) *reinterpret_cast<P*>(o) = ahead[n];
  }
  for (int i = tid + kAhead * kAppendThreads; i < nope; i += kAppendThreads) {
    const T* s;
    T* o;
    at(i, &s, &o);
    *reinterpret_cast<P*>(o) = *reinterpret_cast<const P*>(s);
  }
  __syncthreads();
  const int pairs = half / E;
  for (int i = tid; i < rows * pairs; i += kAppendThreads) {
    const int r = i / pairs, t = (i - r * pairs) * E;
    const T* s = src + r * src_step + dv + t;
    T* o = dst + r * dst_step + dv + t;
    P a = *reinterpret_cast<const P*>(s), b = *reinterpret_cast<const P*>(s + half);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float x1 = to_float(a.v[e]), x2 = to_float(b.v[e]);
      const float2 w = cs[t + e];
      from_float(x1 * w.x - x2 * w.y, &a.v[e]);
      from_float(x2 * w.x + x1 * w.y, &b.v[e]);
    }
    *reinterpret_cast<P*>(o) = a;
    *reinterpret_cast<P*>(o + half) = b;
  }
}

// Writes the new rows (the first CTA of a sequence) and rotates the queries (the others, kAppendHeads heads each): every element of q
// once in and once out. 128 sequences x 128 heads: 10.0 us, 38 MB at 3.8 TB/s; a CTA is a chain of waits (position, angles in 64 bits,
// loads), so the unrotated elements' loads go first (11.7 us with all after the angles). One sequence of 16 heads: 3.9 us, the launch.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ float2 cs[kMaxPairs];
  pdl_wait();
  pdl_launch_dependents();
  const CacheView& c = p.cache;
  const int b = static_cast<int>(blockIdx.y), position = p.position[b];
  if (blockIdx.x == 0) {
    const int j = c.lens[b];
    if (j < 0 || j >= c.capacity) return;
    const long long to = slot_offset(c, b, j);
    if (to < 0) return;
    rotate_rows<T, VEC>(p, static_cast<const T*>(p.row) + b * p.row_stride, 0, static_cast<T*>(c.data) + to, 0, 1, c.dv, true, position, cs);
    if (threadIdx.x == 0) {
      if (p.score != nullptr) p.score[b * p.score_stride + j] = 0.f;
      if (p.slot_position != nullptr) p.slot_position[b * p.slot_position_stride + j] = position;
    }
    return;
  }
  const int h0 = (static_cast<int>(blockIdx.x) - 1) * kAppendHeads;
  rotate_rows<T, VEC>(p, static_cast<const T*>(p.q) + b * p.q_sb + h0 * p.q_sh, p.q_sh, static_cast<T*>(p.q_out) + b * p.qo_sb + h0 * p.qo_sh,
                      p.qo_sh, min(kAppendHeads, p.heads - h0), c.dv, p.copy != 0, position, cs);
}

// ---------------------------------------------------------------------------------------------
// Attend
// ---------------------------------------------------------------------------------------------

constexpr float kLn2 = 0.69314718055994531f, kLog2E = 1.4426950408889634f;
constexpr int kMaxD = 576;
// Rows of the cache per tile. 64 heads leave room for two tiles of 64 rows, fewer heads for three of 48 (more in flight: 128 sequences of
// 4096 rows with 16 heads 132 -> 125 us).
__host__ __device__ constexpr int tile_rows_for(int tile_heads) { return tile_heads < 64 ? 48 : 64; }
constexpr int kRowBytes = 128;                 // of a row that lie together under the 128-byte swizzle: a chunk of 64 elements
constexpr int kGroupBytes = 8 * kRowBytes;     // 8 rows of a chunk, the swizzle's period
constexpr int kMaxStages = 12;
constexpr int kSoftmaxThreads = 128;
constexpr int kAttendThreads = kSoftmaxThreads + 128;
constexpr int kRowWarps = 3;                   // that copy where pages are not whole groups of 8 rows
constexpr int kHeaderBytes = 2048;             // barriers and small arrays, behind the rings
constexpr int kMaxSmem = 232448;               // 227 KiB opt-in limit per CTA on sm_100
constexpr int kTmemCols = 512;
constexpr int kTmemLogits = 256;               // two buffers of a tile's columns behind the accumulators
constexpr unsigned long long kWaitLimitNs = 2000000000ull;
constexpr float kRescaleAbove = 8.f;  // log2: a running maximum is replaced when it is exceeded by this much
// log2 of the weight that a running maximum has. fp16 ends at 2^16 and loses bits below 2^-14: at 2^7 (with 2^8 above it to go), rows
// keep all bits down to 2^-21 of the largest weight, and a long tail's error is 2^-32 of the largest weight a row. bf16 needs none.
template <typename T>
constexpr float kTopWeight = std::is_same<T, __half>::value ? 7.f : 0.f;

struct AttendParams {
  CacheView cache;
  void* out;
  float* lse;              // [batch][heads] or null
  const float* score;
  float* score_out;
  long long out_sb, out_sh, score_stride, score_out_stride;
  int heads, head_tiles, max_len, batch;
  int workers, least;      // workers per head tile, and the least places worth one
  int tile, extra;         // rows per tile; see cache_walk.h
  int joined;              // a join follows; else no sequence can be split
  int copy_rows;           // rows of a TMA copy, 0: copies row by row
  int stages;              // tiles of the ring
  int v_units, chunks;     // 128-element units of the value; 64-element chunks of a row
  float scale_log2;        // scale * log2(e)
  // Workspace
  long long* begins;       // [batch + 1]: places before each sequence, and all
  float* lse2;             // [batch][heads]: log2 of the sum of 2^x; 0 where that sum is 0 (every logit is -inf, and so no weight)
  float2* part_stat;       // [worker][head tile][2][heads of a tile]: maximum and sum
  float* part_out;         // [worker][head tile][2][128-element unit of the value][heads of a tile][128]
  float* logits;           // [batch][tile][heads][rows of a tile] in log2, or null
  int logit_tiles;
  int* status;             // may be null
  unsigned long long selftest_wait_limit_ns;  // the self-test's kernels give up a wait after this long,
  int selftest_skip_tile;                     // and do not copy this tile of the first sequence
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// One probe; the hint (nanoseconds) lets the hardware park the thread until the phase completes.
__device__ __forceinline__ uint32_t mbar_try_wait(uint32_t bar, uint32_t parity, uint32_t hint) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(hint)
      : "memory");
  return ok;
}
__device__ __forceinline__ uint32_t mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
__device__ __forceinline__ unsigned long long global_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Every wait is bounded: the first that expires raises the CTA's flag and reports itself, all others see the flag.
struct Waits {
  volatile int* expired;  // shared memory
  int* status;            // global, may be null
  unsigned long long limit_ns;

  __device__ bool give_up(unsigned long long t0, uint32_t parity, int where) const {
    if (*expired) return true;
    if (global_ns() - t0 <= limit_ns) return false;
    *expired = 1;
    if (status != nullptr && atomicCAS(status, 0, B200_FP8_MM_DEV_WAIT_EXPIRED) == 0) {
      status[1] = where;
      status[2] = static_cast<int>(blockIdx.x);
      status[3] = static_cast<int>(parity);
    }
    return true;
  }
  __device__ __noinline__ bool slow(uint32_t bar, uint32_t parity, int where) const {
    const unsigned long long t0 = global_ns();
    while (!mbar_try_wait(bar, parity, 200000)) {
      if (give_up(t0, parity, where)) return false;
    }
    return true;
  }
  __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int where) const {
    return mbar_try_wait(bar, parity, 200000) || slow(bar, parity, where);
  }
  // For a whole warp, which leaves together.
  __device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, int where) const {
    return __all_sync(0xffffffffu, wait(bar, parity, where)) != 0;
  }
};

enum Where { kAtFree = 0x201, kAtQEmpty, kAtOperands, kAtSFull, kAtPvDone };

// Copies for a whole warp, which comes here together: one lane issues.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred leader;\n\t"
      "elect.sync _|leader, 0xffffffff;\n\t"
      "@leader cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n\t}" ::"r"(dst),
      "l"(map), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int c1, int c2, int c3, int c4, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred leader;\n\t"
      "elect.sync _|leader, 0xffffffff;\n\t"
      "@leader cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];\n\t}" ::"r"(dst),
      "l"(map), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
      : "memory");
}
// The same rows on their way to L2 only.
__device__ __forceinline__ void tma_prefetch_5d(const CUtensorMap* map, int c3, int c4) {
  asm volatile(
      "{\n\t.reg .pred leader;\n\t"
      "elect.sync _|leader, 0xffffffff;\n\t"
      "@leader cp.async.bulk.prefetch.tensor.5d.L2.global.tile [%0, {%1, %1, %1, %2, %3}];\n\t}" ::"l"(map), "r"(0), "r"(c3), "r"(c4)
      : "memory");
}
__device__ __forceinline__ void tcgen05_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Three or four products along K into one accumulator, a_step (of 16 bytes) of A and 32 bytes of B from one to the next. Matrix
// descriptors as 32-bit halves, as in the GEMM: low word address and leading offset, high word stride offset, version and the 128-byte
// swizzle. The whole warp comes here and one lane of it, always the same, issues. One statement for all, and rolled loops around it: a
// warp that issues from unrolled code is held up by its instruction fetch (56 clocks a product against 30).
template <int N>
__device__ __forceinline__ void umma_f16(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t a_step, uint32_t b_lo, uint32_t b_hi,
                                         uint32_t idesc, uint32_t accumulate) {
  static_assert(N == 3 || N == 4, "products of a statement");
  asm volatile(
      "{\n\t.reg .pred p, leader, yes, last;\n\t.reg .b64 da, db;\n\t.reg .b32 la, lb;\n\t"
      "elect.sync _|leader, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.eq.b32 yes, 0, 0;\n\t"
      "setp.eq.and.b32 last, %8, 4, leader;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "@leader tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t"
      "add.u32 la, %1, %7;\n\tadd.u32 lb, %3, 2;\n\tmov.b64 da, {la, %2};\n\tmov.b64 db, {lb, %4};\n\t"
      "@leader tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, yes;\n\t"
      "add.u32 la, la, %7;\n\tadd.u32 lb, %3, 4;\n\tmov.b64 da, {la, %2};\n\tmov.b64 db, {lb, %4};\n\t"
      "@leader tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, yes;\n\t"
      "add.u32 la, la, %7;\n\tadd.u32 lb, %3, 6;\n\tmov.b64 da, {la, %2};\n\tmov.b64 db, {lb, %4};\n\t"
      "@last tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, yes;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(a_step), "n"(N)
      : "memory");
}

__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred leader;\n\t"
      "elect.sync _|leader, 0xffffffff;\n\t"
      "@leader tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}

// 16 lanes x 64 columns: thread t gets columns 8 i + 2 (t % 4) + {0, 1} of lane t / 4 in v[4 i + {0, 1}], of lane t / 4 + 8 in
// v[4 i + {2, 3}].
__device__ __forceinline__ void tmem_ld_16x64(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
// 32 lanes x 16 columns: thread t gets lane t.
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, uint32_t (&v)[16]) { tmem_ld_32x16(taddr, v); }
// 32 lanes x 32 columns.
__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// 2^x, the hardware's (relative error about 2^-22; 0 below 2^-126).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a sum of weights is divided by. It is 0 only where every logit is -inf: such a head gets zeros, as one of a sequence without rows.
__device__ __forceinline__ float inverse_of(float total) { return total == 0.f ? 0.f : 1.f / total; }

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory"); }
__device__ __forceinline__ bool softmax_any(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(mine)), "n"(kSoftmaxThreads)
      : "memory");
  return any != 0;
}

// What the roles of a CTA share, at the end of its shared memory.
struct alignas(8) AttendShared {
  uint64_t full[kMaxStages], pv_done[kMaxStages];  // a tile is there; the second product is done with it
  uint64_t s_full[2], s_free[2], p_full, q_full, q_empty, o_free, drained;
  float factor[64];     // by which a head's accumulators are multiplied when its maximum is replaced
  float2 stat[64];      // maximum and sum of weights of a head
  float inverse[64];    // 1 / sum
  long long sums[kAttendThreads / 32];
  long long share, share_end;  // this worker's places
  long long first_begin;       // where those of the sequence that the share begins in begin
  uint32_t tmem_base;
  int expired, first_seq;
};
static_assert(sizeof(AttendShared) <= kHeaderBytes, "the header is too small");

// A worker's walk over its share: segment after segment, each a run of tiles of one sequence.
struct Walk {
  int b, t, rows, count;   // sequence and first tile of the segment, rows of the sequence, tiles of the segment
  int slot;                // where a part of it is left
  long long begin, from, to;

  __device__ __forceinline__ Walk(const AttendShared& sh)
      : b(sh.first_seq - 1), t(0), rows(0), count(0), slot(0), begin(sh.first_begin), from(sh.share), to(sh.share_end) {}
  __device__ __forceinline__ bool next(const AttendParams& p) {
    while (begin < to) {
      ++b;
      rows = rows_of(p.cache, b, p.max_len);
      count = cache_walk::tiles_in(begin, cache_walk::tiles_of(rows, p.tile), p.extra, from, to, &t);
      slot = cache_walk::part_slot(from, begin);
      begin += cache_walk::places_of(rows, p.tile, p.extra);
      if (rows > 0 && count > 0) return true;
    }
    return false;
  }
  __device__ __forceinline__ bool whole(int tile) const { return count == cache_walk::tiles_of(rows, tile); }
};

// Flash attention of one token per sequence over a latent cache: heads x rows x (d + dv) products per row of d elements read.
//
//   S = Q K^T        [64 heads x rows]      M = heads (64), K = d:     Q and the rows as they lie (K-major)
//   O^T += V^T P^T   [128 x heads] x dv/128 M = value elements, K = rows: the same rows read as an MN-major operand, so that
//                                            a tile is fetched once for both products and never transposed
// With the value's elements in the lanes, the accumulators of 64 heads take 256 of the 512 TMEM columns; with the heads in the
// lanes, 128 heads would take them all and leave none for S. Fewer heads shrink N (16 or 32) and what Q takes of shared memory.
//
// A tile lies in shared memory as [groups of 8 rows][chunk of 64 elements][8 rows x 128 bytes]: one stride from group to group and one
// from chunk to chunk for both operands, and one copy brings all chunks of as many rows as lie together in a page, up to the tile.
//
// What bounds it: up to 32 heads, memory (5.4 TB/s over a whole launch of 128 sequences of 4096 rows, beginning and end included, where a
// copy reaches 6.5); 64 heads, how long a tile stays. From its copy's way through memory
// (1900 clocks, 39 bytes a clock: what L2 gives when all SMs ask) over the first product (1200), the softmax (1450, with its hand-overs)
// and the second product (740) to the next copy it takes 5900, and two tiles of 64 rows are all that fits next to Q: 2950 clocks a tile,
// where the tensor core needs 1900 and, for 128 heads, memory 1600. That is with the next tile fetched to L2 while the ring is full (3400
// a tile without; one sequence of 65536 rows with 128 heads 45.8 -> 43.5 us). The softmax waits for the warp that shares a scheduler with
// the issuing one, 270 clocks behind the others. Beginning costs 3300 clocks of setup and 7000 to 10000 up to the first product, as all
// SMs fetch at once; a segment's end 9000.
// Slower were: tiles of 32 rows, four of them in flight (162 against 142 us, 64 sequences of 4096 rows with 128 heads: an MMA takes 27
// clocks to issue however small it is); units of 128 elements as the ring's grain; halves of a tile freed one by one; the second product
// issued between chunks of the next tile's first (153 against 142 us: the issuing loop loses its pace).
//
// One CTA per SM and worker: warp 4 copies (with warps 6 and 7, 16 bytes a lane, where pages are not whole groups of 8 rows: TMA would
// have to bring them in copies of 128 to 512 bytes, 579 against 99 us for pages of one row), warp 5 issues the products, warps 0 to 3 do
// the softmax (S comes as 16 x 256-bit fragments, 4 threads to a head) and the epilogue. S is double buffered; the next tile's first
// product runs under this tile's softmax. The running maximum is replaced only when a logit exceeds it by 8 (in base 2): the weights
// stay below 2^8 in bf16 and 2^15 in fp16, and rescaling the accumulators is rare. Sums are kept in fp32, weights are rounded to the
// cache's type for the second product, as matrix operands have to be: half a step each, as the result's own rounding, so that bf16 outputs
// are off by 0.0021 of their size instead of 0.0017 (77 rows, in the mean square; 0.0017 both for 65536 rows with 128 heads). A second
// matrix instruction for what the rounding leaves would double the second product.
template <typename T, int HT, bool SELFTEST = false>
__global__ void __launch_bounds__(kAttendThreads, 1)
attend_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap row_map, const __grid_constant__ AttendParams p) {
  constexpr int kTile = tile_rows_for(HT);
  extern __shared__ __align__(1024) uint8_t smem[];
  // The loops below are full of statements that touch memory, behind each of which a parameter would be read anew.
  const CacheView c = p.cache;
  const int v_units = p.v_units, chunks = p.chunks, stages = p.stages, copy_rows = p.copy_rows, heads_all = p.heads;
  const float scale_log2 = p.scale_log2;
  const long long out_sb = p.out_sb, out_sh = p.out_sh;
  float *const logits = p.logits, *const part_out = p.part_out;
  T* const out_at = static_cast<T*>(p.out);
  const int group_bytes = chunks * kGroupBytes, tile_bytes = kTile / 8 * group_bytes;
  uint8_t* const q_smem = smem;  // [chunk][HT rows x 128 bytes]; the first product reads 64 rows, those behind HT are never looked at
  uint8_t* const ring = q_smem + chunks * HT * kRowBytes;
  uint8_t* const p_smem = ring + stages * tile_bytes;
  AttendShared& sh = *reinterpret_cast<AttendShared*>(p_smem + HT * kRowBytes);
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int head_tile = static_cast<int>(blockIdx.x) % p.head_tiles, worker = static_cast<int>(blockIdx.x) / p.head_tiles;
  const int head0 = head_tile * HT;
  const Waits waits{&sh.expired, p.status, SELFTEST ? p.selftest_wait_limit_ns : kWaitLimitNs};
  if (tid == 0) {
    for (int i = 0; i < kMaxStages; ++i) {
      mbar_init(smem_u32(&sh.full[i]), p.copy_rows > 0 ? 1 : kRowWarps);
      mbar_init(smem_u32(&sh.pv_done[i]), 1);
    }
    mbar_init(smem_u32(&sh.q_full), 1);
    mbar_init(smem_u32(&sh.q_empty), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh.s_full[i]), 1);
      mbar_init(smem_u32(&sh.s_free[i]), 4);
    }
    mbar_init(smem_u32(&sh.p_full), 4);
    mbar_init(smem_u32(&sh.o_free), 4);
    mbar_init(smem_u32(&sh.drained), 1);
    sh.expired = (smem_u32(smem) & 1023u) != 0;  // the swizzle needs it; never so with no static shared memory before it
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&q_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&row_map) : "memory");
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  // Places before each thread's run of sequences, and where this worker's share begins.
  const int run = (p.batch + kAttendThreads - 1) / kAttendThreads;
  const int b0 = min(p.batch, tid * run), b1 = min(p.batch, b0 + run);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += cache_walk::places_of(rows_of(c, b, p.max_len), kTile, p.extra);
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sh.sums[warp] = upto;
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  // Not before this CTA has its TMEM: a CTA of the next kernel that took some of it first would wait for this one's end, and this one
  // for its columns.
  pdl_launch_dependents();
  constexpr uint32_t tmem = 0;  // all columns are this CTA's, so they begin at the first (checked here)
  if (tid == 0 && sh.tmem_base != tmem) sh.expired = 1;
  {
    long long before = upto - mine, places = 0;
    for (int w = 0; w < kAttendThreads / 32; ++w) {
      if (w < warp) before += sh.sums[w];
      places += sh.sums[w];
    }
    const int workers = cache_walk::workers_of(places, p.workers, p.least);
    const long long begin = worker < workers ? cache_walk::share_begin(places, workers, worker) : 0;
    const long long end = worker < workers ? cache_walk::share_begin(places, workers, worker + 1) : 0;
    if (tid == 0) {
      sh.share = begin;
      sh.share_end = end;
      if (begin == end) sh.first_begin = end;
    }
    if (begin < end && before <= begin && begin < before + mine) {
      long long at = before;
      int b = b0;
      for (; b + 1 < b1; ++b) {  // (the last of the thread's sequences if none before it)
        const int n = cache_walk::places_of(rows_of(c, b, p.max_len), kTile, p.extra);
        if (begin < at + n) break;
        at += n;
      }
      sh.first_seq = b;
      sh.first_begin = at;
    }
    if (blockIdx.x == 0) {
      for (int b = b0; b < b1; ++b) {
        p.begins[b] = before;
        if (b + 1 < b1) before += cache_walk::places_of(rows_of(c, b, p.max_len), kTile, p.extra);
      }
      if (tid == 0) p.begins[p.batch] = places;
    }
  }
  __syncthreads();

  // The queries of a segment, once the first products of the segment before are over.
  auto copy_queries = [&](int segment, int b) {
    if (segment > 0 && !waits.wait_all(smem_u32(&sh.q_empty), (segment - 1) & 1, kAtQEmpty)) return false;
    if (lane == 0) mbar_expect_tx(smem_u32(&sh.q_full), chunks * HT * kRowBytes);
    __syncwarp();
    tma_load_4d(smem_u32(q_smem), &q_map, head0, 0, b, smem_u32(&sh.q_full));
    return true;
  };
  // Warps 6 and 7: where no join follows, what sequences without rows get.
  auto write_empty = [&]() {
    if (p.joined) return;
    const int heads = min(HT, heads_all - head0);
    for (int b = worker; b < p.batch; b += p.workers) {
      if (rows_of(c, b, p.max_len) > 0) continue;
      for (int h = warp - 6; h < heads; h += 2) {
        T* const out = out_at + b * out_sb + (head0 + h) * out_sh;
        for (int e = lane; e < c.dv; e += 32) from_float(0.f, out + e);
        const long long at = static_cast<long long>(b) * heads_all + head0 + h;
        if (lane == 0) p.lse2[at] = -INFINITY;
        if (lane == 0 && p.lse != nullptr) p.lse[at] = -INFINITY;
      }
    }
  };

  if (warp == 4 && copy_rows > 0) {
    // Copies by TMA. Lane l knows where piece l (copy_rows rows) of a tile comes from.
    const int pieces = kTile / copy_rows;
    int stage = 0, segment = 0;
    uint32_t lap = 0;  // parity of the ring's current use
    bool first_lap = true, ok = __all_sync(0xffffffffu, sh.expired == 0);
    Walk walk(sh);
    while (ok && __all_sync(0xffffffffu, walk.next(p))) {
      const int* table = c.block_table + walk.b * c.table_stride;
      int page, slot;
      // rows behind the sequence come from a page behind the last, as zeros
      auto place = [&](int tile) {
        const int row = tile * kTile + lane * copy_rows;
        page = c.pages;
        slot = 0;
        if (lane < pieces && tile < walk.t + walk.count && row < walk.rows) {
          const int at = row / c.page_size;
          slot = row - at * c.page_size;
          const int id = table[at];
          page = id < 0 || id > c.pages ? c.pages : id;
        }
      };
      place(walk.t);
      const int count = __shfl_sync(0xffffffffu, walk.count, 0), left_out = SELFTEST && walk.b == 0 ? p.selftest_skip_tile - walk.t : -1;
      for (int tile = 0; tile < count; ++tile) {
        const uint32_t full = smem_u32(&sh.full[stage]), to = smem_u32(ring) + stage * tile_bytes;
        if (!first_lap && !(ok = waits.wait_all(smem_u32(&sh.pv_done[stage]), lap ^ 1, kAtFree))) break;
        const int copies = SELFTEST && tile == left_out ? 0 : pieces;
        if (lane == 0 && (!SELFTEST || copies > 0)) mbar_expect_tx(full, tile_bytes);
        __syncwarp();
        for (int k = 0; k < copies; ++k)
          tma_load_5d(to + k * (copy_rows >> 3) * group_bytes, &row_map, 0, 0, __shfl_sync(0xffffffffu, slot, k) >> 3,
                      __shfl_sync(0xffffffffu, page, k), full);
        if (++stage == stages) stage = 0, lap ^= 1, first_lap = false;
        if (tile == 0 && !(ok = copy_queries(segment, walk.b))) break;
        place(walk.t + tile + 1);  // on its way during the waits
        if (HT == 64 && !first_lap && tile + 1 < count)
          for (int k = 0; k < pieces; ++k) {
            const int of = __shfl_sync(0xffffffffu, page, k), at = __shfl_sync(0xffffffffu, slot, k) >> 3;
            if (of < c.pages) tma_prefetch_5d(&row_map, at, of);
          }
      }
      ++segment;
    }
  } else if ((warp == 4 || warp > 5) && copy_rows == 0) {
    // Copies row by row, every third row of a tile, 16 bytes a lane. Lane l knows where rows l and l + 32 of a tile come from. A tile
    // is announced once its copies have landed: when the next one's are on their way, or when nothing else can be done.
    const int first_row = warp == 4 ? 0 : warp - 5;
    const uint16_t* const data = static_cast<const uint16_t*>(c.data);
    int stage = 0, segment = 0, landing = -1;
    uint32_t lap = 0;
    bool first_lap = true, ok = __all_sync(0xffffffffu, sh.expired == 0);
    auto announce = [&](bool all) {
      if (landing < 0) return;
      if (all)
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      else
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.full[landing]));
      landing = -1;
    };
    Walk walk(sh);
    while (ok && __all_sync(0xffffffffu, walk.next(p))) {
      const int* table = c.block_table + walk.b * c.table_stride;
      long long from[2];  // element offset, -1 where there is no row: zeros
      auto place = [&](int tile) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int in_tile = lane + 32 * k, row = tile * kTile + in_tile;
          from[k] = -1;
          if (in_tile < kTile && tile < walk.t + walk.count && row < walk.rows) {
            const int at = row / c.page_size, id = table[at];
            if (id >= 0 && id < c.pages) from[k] = id * c.page_stride + static_cast<long long>(row - at * c.page_size) * c.slot_stride;
          }
        }
      };
      place(walk.t);
      const int count = __shfl_sync(0xffffffffu, walk.count, 0), left_out = SELFTEST && walk.b == 0 ? p.selftest_skip_tile - walk.t : -1;
      for (int tile = 0; tile < count; ++tile) {
        if (!first_lap && !__all_sync(0xffffffffu, mbar_test(smem_u32(&sh.pv_done[stage]), lap ^ 1))) {
          announce(true);
          if (!(ok = waits.wait_all(smem_u32(&sh.pv_done[stage]), lap ^ 1, kAtFree))) break;
        }
        const uint32_t to = smem_u32(ring) + stage * tile_bytes;
        for (int row = first_row; row < kTile; row += kRowWarps) {
          const long long at = __shfl_sync(0xffffffffu, row < 32 ? from[0] : from[1], row & 31);
          const uint16_t* const src = data + (at < 0 ? 0 : at) + 8 * lane;
          const uint32_t bytes = at < 0 ? 0u : 16u;
          // 16-byte piece n of a chunk's 128 bytes lies at piece n ^ (row % 8)
          const uint32_t dst = to + (row >> 3) * group_bytes + (row & 7) * kRowBytes + (((lane & 7) ^ (row & 7)) << 4) + (lane >> 3) * kGroupBytes;
#pragma unroll
          for (int k = 0; k < 3; ++k)
            if (lane + 32 * k < 8 * chunks)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 4 * k * kGroupBytes), "l"(src + 256 * k), "r"(bytes) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        announce(false);
        landing = SELFTEST && tile == left_out ? -1 : stage;
        if (++stage == stages) stage = 0, lap ^= 1, first_lap = false;
        if (tile == 0 && warp == 4) {
          announce(true);
          if (!(ok = copy_queries(segment, walk.b))) break;
        }
        place(walk.t + tile + 1);  // on its way during the waits
      }
      ++segment;
    }
    announce(true);
    asm volatile("cp.async.wait_all;" ::: "memory");  // (those of a tile that was begun when a wait expired)
    if (warp > 5) write_empty();
  } else if (warp > 5) {
    write_empty();
  } else if (warp == 5) {
    // Products. All lanes walk along, and votes make the branches uniform: the operands of the instructions are then formed in
    // uniform registers. With one lane walking alone, each instruction took 97 clocks to issue. (Two issuing warps, one for each
    // product, were three times slower: the tensor core does not like the shapes to alternate.)
    constexpr uint32_t kAll = 0xffffffffu;
    constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t kIdesc = (1u << 4) | (kType << 7) | (kType << 10);
    constexpr uint32_t kIdescS = kIdesc | (static_cast<uint32_t>(kTile >> 3) << 17) | (64u >> 4 << 24);
    constexpr uint32_t kIdescO = kIdesc | (1u << 15) | (static_cast<uint32_t>(HT >> 3) << 17) | (128u >> 4 << 24);  // A is MN-major
    constexpr uint32_t kHi = (1u << 14) | (2u << 29);
    constexpr uint32_t kHiDense = kHi | (kGroupBytes >> 4);      // queries and weights: groups of 8 rows one behind the other
    constexpr uint32_t kLoK = 1u << 16;                                       // K-major: no leading offset
    constexpr uint32_t kLoV = static_cast<uint32_t>(kGroupBytes >> 4) << 16;  // MN-major: to the next 64 elements
    const uint32_t hi_rows = kHi | (group_bytes >> 4);
    const uint32_t q_lo = kLoK | (smem_u32(q_smem) >> 4), p_lo = kLoK | (smem_u32(p_smem) >> 4), ring_at = smem_u32(ring) >> 4;
    // One value for the warp, in a uniform register.
    auto uniform = [](uint32_t v) { return __reduce_max_sync(kAll, v); };
    int stage = 0, i = 0, segment = 0;
    uint32_t lap = 0;
    // The second product that is still to be issued, of the tile before.
    bool pending = false, pending_first = false;
    int pv_stage = 0, pv_segment = 0, pv_tile = 0;
    uint32_t pv_values = 0;
    auto second = [&]() {
      tcgen05_fence_after();
      uint32_t values = uniform(pv_values), o = tmem;
#pragma unroll 1
      for (int u = 0; u < v_units; ++u, values += 2 * kGroupBytes >> 4, o += HT)
        umma_f16<kTile / 16>(o, values, hi_rows, 2 * group_bytes >> 4, p_lo, kHiDense, kIdescO, pending_first ? 0u : 1u);
      umma_commit(smem_u32(&sh.pv_done[pv_stage]));
      pending = false;
    };
    // Whether the first product of tile i can go: its rows, a buffer of S and, where a segment begins, the queries. The second one of the
    // tile before: the weights and, where its segment begins, the accumulators of the one before read out. All lanes look at the same
    // barriers: 17 clocks each; a barrier per lane, all at once, took 200.
    auto first_ready = [&](bool begins) {
      uint32_t there = mbar_test(smem_u32(&sh.full[stage]), lap) & mbar_test(smem_u32(&sh.s_free[i & 1]), (static_cast<uint32_t>(i) >> 1 & 1u) ^ 1u);
      if (begins) there &= mbar_test(smem_u32(&sh.q_full), static_cast<uint32_t>(segment) & 1u);
      return __all_sync(kAll, there != 0) != 0;
    };
    auto second_ready = [&]() {
      uint32_t there = mbar_test(smem_u32(&sh.p_full), static_cast<uint32_t>(pv_tile) & 1u);
      if (pending_first && pv_segment > 0) there &= mbar_test(smem_u32(&sh.o_free), static_cast<uint32_t>(pv_segment - 1) & 1u);
      return __all_sync(kAll, there != 0) != 0;
    };
    // Waits for the first product to become possible, or for the pending second one (`first` false); the second one goes meanwhile as
    // soon as it can, because it frees the ring.
    auto until = [&](bool first, bool begins) {
      unsigned long long t0 = 0;  // (read late: reading the timer takes several hundred clocks)
      for (uint32_t spins = 1;; ++spins) {
        if (first && first_ready(begins)) return true;
        if (pending && second_ready()) {
          if (!first) return true;
          second();
        }
        if ((spins & 1023u) == 0) {
          if (t0 == 0) t0 = global_ns();
          if (__any_sync(kAll, waits.give_up(t0, static_cast<uint32_t>(i), kAtOperands))) return false;
        }
      }
    };
    bool ok = __all_sync(kAll, sh.expired == 0);
    Walk walk(sh);
    while (ok && __all_sync(kAll, walk.next(p))) {
      const int count = __shfl_sync(kAll, walk.count, 0);
      for (int tile = 0; tile < count; ++tile) {
        if (!until(true, tile == 0)) {
          ok = false;
          break;
        }
        tcgen05_fence_after();
        const uint32_t values = kLoV | (ring_at + stage * (tile_bytes >> 4));
        const int here = stage;
        uint32_t rows = uniform(kLoK | (ring_at + stage * (tile_bytes >> 4))), q_at = q_lo;
        const uint32_t s = tmem + kTmemLogits + (i & 1) * 64;
#pragma unroll 1
        for (int n = 0; n < chunks; ++n, q_at += HT * kRowBytes >> 4, rows += kGroupBytes >> 4)
          umma_f16<4>(s, q_at, kHiDense, 2, rows, hi_rows, kIdescS, n > 0);
        umma_commit(smem_u32(&sh.s_full[i & 1]));
        if (tile == count - 1) umma_commit(smem_u32(&sh.q_empty));
        if (++stage == stages) stage = 0, lap ^= 1;
        ++i;
        if (pending) {
          if (!until(false, false)) {
            ok = false;
            break;
          }
          second();
        }
        pending = true;
        pending_first = tile == 0;
        pv_tile = i - 1;
        pv_stage = here;
        pv_values = values;
        pv_segment = segment;
      }
      ++segment;
    }
    if (ok && pending && until(false, false)) second();
    __syncwarp();
  } else if (warp < 4) {
    // Softmax: warp w has heads 16 w .. 16 w + 15 of the tile, thread t rows (heads) t / 4 and t / 4 + 8 of these.
    const bool active = 16 * warp < HT;
    const int row0 = 16 * warp + lane / 4, row1 = row0 + 8;
    const uint32_t lanes = static_cast<uint32_t>(32 * warp) << 16;
    // The tile's place in the ring, and that of the tile before it, whose second product is waited for.
    struct Place {
      int stage;
      uint32_t lap;
    } here = {0, 0}, before = {0, 0};
    int i = 0;
    bool ok = sh.expired == 0;
    // A wait that has expired does not end this role, because the other warps meet it at the barriers below: the rest of the walk
    // goes by without waiting, over whatever is there.
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
      if (ok && !mbar_test(smem_u32(bar), parity)) ok = waits.wait(smem_u32(bar), parity, where);
    };
    Walk walk(sh);
    while (walk.next(p)) {
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
      for (int tile = 0; tile < walk.count; ++tile, ++i) {
        wait(&sh.s_full[i & 1], (i >> 1) & 1, kAtSFull);
        tcgen05_fence_after();
        uint32_t x[32];
        if (active) tmem_ld_16x64(tmem + lanes + kTmemLogits + (i & 1) * 64, x);
        tcgen05_fence_before();
        const int left = walk.rows - (walk.t + tile) * kTile;  // rows that exist from this tile on
        float t0 = -INFINITY, t1 = -INFINITY, sum0 = 0.f, sum1 = 0.f;
        uint32_t w[16];
        bool up = false;
        auto head_max = [&]() {  // over the four threads of a head
#pragma unroll
          for (int o = 1; o < 4; o <<= 1) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
          }
        };
        auto weigh = [&]() {
          const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
          sum0 = sum1 = 0.f;
#pragma unroll
          for (int n = 0; n < kTile / 8; ++n) {
            const float a = exp2_fast(__uint_as_float(x[4 * n]) - z0), b = exp2_fast(__uint_as_float(x[4 * n + 1]) - z0);
            const float e = exp2_fast(__uint_as_float(x[4 * n + 2]) - z1), f = exp2_fast(__uint_as_float(x[4 * n + 3]) - z1);
            sum0 += a + b;
            sum1 += e + f;
            w[2 * n] = pack2(a, b, T());
            w[2 * n + 1] = pack2(e, f, T());
          }
        };
        if (active) {
          if (left >= kTile) {
#pragma unroll
            for (int n = 0; n < kTile / 2; ++n) x[n] = __float_as_uint(__uint_as_float(x[n]) * scale_log2);
          } else {
#pragma unroll
            for (int n = 0; n < kTile / 2; ++n) {
              const int col = 8 * (n / 4) + 2 * (lane % 4) + (n & 1);
              x[n] = __float_as_uint(col < left ? __uint_as_float(x[n]) * scale_log2 : -INFINITY);
            }
          }
#pragma unroll
          for (int n = 0; n < kTile / 2; ++n) {
            if (n & 2) t1 = fmaxf(t1, __uint_as_float(x[n])); else t0 = fmaxf(t0, __uint_as_float(x[n]));
          }
          if (logits != nullptr) {
            float* to = logits + ((static_cast<long long>(walk.b) * p.logit_tiles + walk.t + tile) * heads_all + head0) * kTile + 2 * (lane % 4);
#pragma unroll
            for (int n = 0; n < kTile / 8; ++n) {
              if (row0 < HT && head0 + row0 < heads_all)
                *reinterpret_cast<uint2*>(to + row0 * kTile + 8 * n) = make_uint2(x[4 * n], x[4 * n + 1]);
              if (row1 < HT && head0 + row1 < heads_all)
                *reinterpret_cast<uint2*>(to + row1 * kTile + 8 * n) = make_uint2(x[4 * n + 2], x[4 * n + 3]);
            }
          }
          // Against the maximum that is; the tile's own matters only where it is far above.
          if (tile == 0) {
            head_max();
            m0 = t0 - kTopWeight<T>;
            m1 = t1 - kTopWeight<T>;
          }
          weigh();
          up = t0 > m0 + kRescaleAbove + kTopWeight<T> || t1 > m1 + kRescaleAbove + kTopWeight<T>;
        }
        // The weights before are read, and the accumulators at rest, once the second product of the tile before is over. (Looked at
        // before the vote, which takes as long.)
        const bool over = i == 0 || mbar_test(smem_u32(&sh.pv_done[before.stage]), before.lap);
        const bool rescale = tile > 0 && softmax_any(up);
        if (rescale && active) {
          const float from0 = m0, from1 = m1;
          head_max();
          float f0 = 1.f, f1 = 1.f;
          if (t0 - kTopWeight<T> > m0 + kRescaleAbove) m0 = t0 - kTopWeight<T>, f0 = exp2_fast(from0 - m0);
          if (t1 - kTopWeight<T> > m1 + kRescaleAbove) m1 = t1 - kTopWeight<T>, f1 = exp2_fast(from1 - m1);
          l0 *= f0;
          l1 *= f1;
          if (lane % 4 == 0) {
            sh.factor[row0] = f0;
            sh.factor[row1] = f1;
          }
          weigh();
        }
        l0 += sum0;
        l1 += sum1;
        if (!over) wait(&sh.pv_done[before.stage], before.lap, kAtPvDone);
        if (rescale) {
          softmax_sync();  // (the factors)
          tcgen05_fence_after();
          for (int col = 0; col < v_units * HT; col += 16) {
            uint32_t o[16];
            tmem_ld_32x16(tmem + lanes + col, o);
#pragma unroll
            for (int n = 0; n < 16; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * sh.factor[col % HT + n]);
            tmem_st_32x16(tmem + lanes + col, o);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tcgen05_fence_before();
        }
        if (active) {
          // 16-byte piece n of row r lies at piece n ^ (r % 8) of its 128 bytes (the swizzle of K-major operands)
          uint8_t* to = p_smem + 4 * (lane % 4);
#pragma unroll
          for (int n = 0; n < kTile / 8; ++n) {
            const int piece = 16 * (n ^ (lane / 4));
            *reinterpret_cast<uint32_t*>(to + row0 * kRowBytes + piece) = w[2 * n];
            *reinterpret_cast<uint32_t*>(to + row1 * kRowBytes + piece) = w[2 * n + 1];
          }
        }
        if (left < kTile) {
          // What lies behind the sequence in its last page may be anything: as values it has to be 0, because 0 weights times
          // infinity or NaN would be NaN. (Pieces that begin behind the sequence have come as zeros.)
          const int end = copy_rows > 0 ? (left + copy_rows - 1) / copy_rows * copy_rows : left;
          for (int row = left + warp; row < end; row += kSoftmaxThreads / 32) {
            uint8_t* const at = ring + here.stage * tile_bytes + (row >> 3) * group_bytes + (row & 7) * kRowBytes;
            for (int piece = lane; piece < 16 * v_units; piece += 32)  // 16 bytes each
              *reinterpret_cast<uint4*>(at + (piece >> 3) * kGroupBytes + (piece & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        before = here;
        if (++here.stage == stages) here.stage = 0, here.lap ^= 1;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&sh.p_full));
          mbar_arrive(smem_u32(&sh.s_free[i & 1]));
        }
      }
      // End of the segment: sums over the four threads of a head, then the accumulators, a value element per thread.
      if (active) {
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          l0 += __shfl_xor_sync(0xffffffffu, l0, o);
          l1 += __shfl_xor_sync(0xffffffffu, l1, o);
        }
      }
      // (The last second product has needed all four warps' weights: none of them still reads what the segment before left here.)
      wait(&sh.pv_done[before.stage], before.lap, kAtPvDone);
      if (active && lane % 4 == 0) {
        sh.stat[row0] = make_float2(m0, l0);
        sh.stat[row1] = make_float2(m1, l1);
        sh.inverse[row0] = inverse_of(l0);
        sh.inverse[row1] = inverse_of(l1);
      }
      softmax_sync();
      tcgen05_fence_after();
      const int heads = min(HT, heads_all - head0);
      const bool whole = walk.whole(kTile);
      const long long part = (static_cast<long long>(worker) * p.head_tiles + head_tile) * 2 + walk.slot;
      // kCols heads of 128 value elements at a time: a warp writes 32 elements of a head at once
      constexpr int kCols = HT < 32 ? HT : 32;
      for (int u = 0; u < v_units; ++u) {
#pragma unroll
        for (int h0 = 0; h0 < HT; h0 += kCols) {
          uint32_t o[kCols];
          tmem_ld_32(tmem + lanes + u * HT + h0, o);
          if (whole) {
            T* out = out_at + walk.b * out_sb + (head0 + h0) * out_sh + u * 128 + tid;
#pragma unroll
            for (int n = 0; n < kCols; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * sh.inverse[h0 + n]);
#pragma unroll
            for (int n = 0; n < kCols; ++n, out += out_sh)
              if (h0 + n < heads) from_float(__uint_as_float(o[n]), out);
          } else {
            float* const out = part_out + ((part * v_units + u) * HT + h0) * 128 + tid;
#pragma unroll
            for (int n = 0; n < kCols; ++n) out[n * 128] = __uint_as_float(o[n]);
          }
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.o_free));
      if (whole) {
        if (tid < heads) {
          const float2 st = sh.stat[tid];
          const float lse2 = (st.x == -INFINITY ? 0.f : st.x) + log2f(st.y);
          const long long at = static_cast<long long>(walk.b) * heads_all + head0 + tid;
          p.lse2[at] = st.y == 0.f ? 0.f : lse2;
          if (p.lse != nullptr) p.lse[at] = lse2 * kLn2;
        }
      } else if (tid < heads) {
        p.part_stat[part * HT + tid] = sh.stat[tid];
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  // Where a wait has expired, copies and products may still be in flight, whichever role it was: no shared memory and no TMEM is given
  // back before they have come to rest. (Looked at when all roles are over: one that ended early has not seen a later one's wait expire.)
  // Each of these waits is bounded too; a phase that will not complete, because its use was not begun, runs out of its 10 ms.
  if (sh.expired != 0) {
    auto at_rest = [&](uint64_t* bar, uint32_t parity) {
      for (int n = 0; n < 1000 && !mbar_try_wait(smem_u32(bar), parity, 10000); ++n) {
      }
    };
    if (warp == 4 && lane == 0) {
      for (uint32_t parity = 0; parity < 2; ++parity) {
        for (int n = 0; copy_rows > 0 && n < stages; ++n) at_rest(&sh.full[n], parity);
        at_rest(&sh.q_full, parity);
      }
    }
    if (warp == 5) {
      umma_commit(smem_u32(&sh.drained));
      at_rest(&sh.drained, 0);
    }
    __syncwarp();
  }
  if (warp == 5) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// Heads of a CTA of the join: two where sequences have few parts, whose statistics and values are all on their way together. (64 ragged
// sequences, 128 heads, in a row: 126.9 us with one, 122.4 with two, 127.6 with four.)
__host__ __device__ constexpr int join_heads(int groups) { return groups == 1 ? 2 : 1; }

// Joins the parts of split sequences, in the order of their rows, and writes what sequences without rows get: a CTA per head (or
// two) and sequence, GROUPS groups of a thread for every 4 value elements that share the parts. It reads what the attention left in L2;
// what it costs is a chain of loads (where the sequence's parts are, their statistics, the parts), so every thread looks up all of it
// for itself and only the groups' sums go through shared memory. Without it, where no sequence can be split, 128 sequences of 60 rows
// with 32 heads take 11.2 us instead of 16.2. The parts of one sequence of 65536 rows with 128 heads are 19 MB: 11.7 us by itself from
// cold caches.
template <typename T, int GROUPS>
__global__ void __launch_bounds__(128 * GROUPS) attend_join_kernel(const __grid_constant__ AttendParams p, int tile_heads) {
  constexpr int kHeads = join_heads(GROUPS), kAhead = 3;  // parts whose values are on their way along with the statistics
  __shared__ float4 sums[GROUPS][128];
  pdl_wait();
  pdl_launch_dependents();
  const int h0 = static_cast<int>(blockIdx.x) * kHeads, heads = min(kHeads, p.heads - h0), b = static_cast<int>(blockIdx.y);
  const long long places = p.begins[p.batch], begin = p.begins[b], end = p.begins[b + 1];
  const int tid = static_cast<int>(threadIdx.x), dv = p.cache.dv, group = tid >> 7, e = tid & 127, lane = tid & 31;
  T* const out = static_cast<T*>(p.out) + b * p.out_sb + h0 * p.out_sh;
  const long long at = static_cast<long long>(b) * p.heads + h0;
  if (begin == end) {
    for (int n = 0; n < heads; ++n)
      for (int i = tid; i < dv; i += 128 * GROUPS) from_float(0.f, out + n * p.out_sh + i);
    if (tid < heads) {
      p.lse2[at + tid] = -INFINITY;
      if (p.lse != nullptr) p.lse[at + tid] = -INFINITY;
    }
    return;
  }
  const int workers = cache_walk::workers_of(places, p.workers, p.least);
  const int tiles = static_cast<int>(end - begin) - p.extra;
  const int g0 = cache_walk::worker_of(places, workers, cache_walk::first_place(begin, tiles, p.extra));
  const int parts = cache_walk::worker_of(places, workers, cache_walk::last_place(begin, tiles, p.extra)) - g0 + 1;
  if (parts == 1) return;  // written by its worker
  const int head_tile = h0 / tile_heads, in_tile = h0 - head_tile * tile_heads;
  // Only the first part can lie behind another sequence's in its worker's share.
  const int slot0 = cache_walk::part_slot(cache_walk::share_begin(places, workers, g0), begin);
  auto part_of = [&](int i) { return (static_cast<long long>(g0 + i) * p.head_tiles + head_tile) * 2 + (i == 0 ? slot0 : 0); };
  auto stat_of = [&](int n, int i) { return p.part_stat[part_of(i) * tile_heads + in_tile + n]; };
  auto value_of = [&](int n, int i) {
    return *reinterpret_cast<const float4*>(p.part_out + ((part_of(i) * (dv / 128) + e / 32) * tile_heads + in_tile + n) * 128 + 4 * (e % 32));
  };
  // (A head tile has room for heads that do not exist; what is read there is not used.)
  float2 stat[kHeads];
  float4 ahead[kHeads][kAhead];
#pragma unroll
  for (int n = 0; n < kHeads; ++n) stat[n] = lane < parts ? stat_of(n, lane) : make_float2(-INFINITY, 0.f);
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
#pragma unroll
    for (int n = 0; n < kHeads; ++n)
      if (group + k * GROUPS < parts && 4 * e < dv) ahead[n][k] = value_of(n, group + k * GROUPS);
#pragma unroll
  for (int n = 0; n < kHeads; ++n) {
    float top = stat[n].x;
    for (int i = lane + 32; i < parts; i += 32) top = fmaxf(top, stat_of(n, i).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top, mine = exp2_fast(stat[n].x - base);
    float total = lane < parts ? stat[n].y * mine : 0.f;
    for (int i = lane + 32; i < parts; i += 32) {
      const float2 s = stat_of(n, i);
      total += s.y * exp2_fast(s.x - base);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int i, const float4& v) {  // (i is the same for the warp)
      const float w = i < 32 ? __shfl_sync(0xffffffffu, mine, i) : exp2_fast(stat_of(n, i).x - base);
      sum.x += w * v.x;
      sum.y += w * v.y;
      sum.z += w * v.z;
      sum.w += w * v.w;
    };
    if (4 * e < dv) {  // (whole warps: dv is a multiple of 128)
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (group + k * GROUPS < parts) add(group + k * GROUPS, ahead[n][k]);
#pragma unroll 4
      for (int i = group + kAhead * GROUPS; i < parts; i += GROUPS) add(i, value_of(n, i));
    }
    if constexpr (GROUPS > 1) {
      sums[group][e] = sum;
      __syncthreads();
      if (group > 0) return;
#pragma unroll
      for (int k = 1; k < GROUPS; ++k) {
        const float4 v = sums[k][e];
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
    }
    if (n >= heads) return;
    if (4 * e < dv) {
      const float inverse = inverse_of(total);
      T* const to = out + n * p.out_sh + 4 * e;
      from_float(sum.x * inverse, to);
      from_float(sum.y * inverse, to + 1);
      from_float(sum.z * inverse, to + 2);
      from_float(sum.w * inverse, to + 3);
    }
    if (tid == 0) {
      const float lse2 = base + log2f(total);
      p.lse2[at + n] = total == 0.f ? 0.f : lse2;
      if (p.lse != nullptr) p.lse[at + n] = lse2 * kLn2;
    }
  }
}

// score_out = score + the weights of all heads, from the logits that the attention left: a CTA per tile, a group of threads for every
// fourth head. It needs every head's sum over the whole sequence, so it follows the join. (One kernel for both, in which each tile's CTA
// takes the sums from the parts itself, was slower: 28 against 18 us for 8 sequences of 2049 rows, 69 against 63 for 32 with 128 heads.)
constexpr int kScoreGroups = 4;

template <int kTile>
__global__ void __launch_bounds__(kScoreGroups * kTile) attend_score_kernel(const __grid_constant__ AttendParams p) {
  __shared__ float sums[kScoreGroups][kTile];
  pdl_wait();
  pdl_launch_dependents();
  const int b = static_cast<int>(blockIdx.y), tile = static_cast<int>(blockIdx.x);
  const int rows = rows_of(p.cache, b, p.max_len);
  if (tile * kTile >= rows) return;
  const int col = static_cast<int>(threadIdx.x) % kTile, group = static_cast<int>(threadIdx.x) / kTile;
  const float* x = p.logits + (static_cast<long long>(b) * p.logit_tiles + tile) * p.heads * kTile + col;
  const float* lse2 = p.lse2 + static_cast<long long>(b) * p.heads;
  float sum = 0.f;
#pragma unroll 4
  for (int h = group; h < p.heads; h += kScoreGroups) sum += exp2_fast(x[static_cast<long long>(h) * kTile] - lse2[h]);
  sums[group][col] = sum;
  __syncthreads();
  const int j = tile * kTile + col;
  if (group == 0 && j < rows) {
#pragma unroll
    for (int k = 1; k < kScoreGroups; ++k) sum += sums[k][col];
    p.score_out[b * p.score_out_stride + j] = p.score[b * p.score_stride + j] + sum;
  }
}

// ---------------------------------------------------------------------------------------------
// Evict
// ---------------------------------------------------------------------------------------------

constexpr int kMaxCluster = 8;
constexpr int kMaxStaged = 20480;               // slots of a CTA whose ranks and positions are kept in shared memory (160 KB)
constexpr int kFewMoves = 64;                   // a sequence's rows that the selecting CTAs move themselves
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
  int cluster;   // CTAs per sequence
  int staged;    // ranks that fit the CTA's shared memory
  int few;       // the selecting CTAs move the rows
};

// Order of the scores as unsigned integers: NaN above every number, -0 as 0. Protected rows are above all.
constexpr uint32_t kProtected = 0xffffffffu;
__device__ __forceinline__ uint32_t rank_of(float score) {
  if (score != score) return kProtected - 1;
  const uint32_t u = __float_as_uint(score + 0.f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Exclusive sum of v over the CTA's threads, and the total.
template <int THREADS>
__device__ __forceinline__ int threads_before(int v, int* scratch, int* total) {
  constexpr int kWarps = THREADS / 32;
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  uint32_t upto = static_cast<uint32_t>(v);  // (two counts of 16 bits may come as one)
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  __syncthreads();  // (scratch may still be read from the last time)
  if (lane == 31) scratch[warp] = static_cast<int>(upto);
  __syncthreads();
  uint32_t w = lane < kWarps ? static_cast<uint32_t>(scratch[lane]) : 0u;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  *total = static_cast<int>(__shfl_sync(0xffffffffu, w, kWarps - 1));
  const uint32_t before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  return static_cast<int>((warp > 0 ? before : 0u) + upto - static_cast<uint32_t>(v));
}

__device__ __forceinline__ void move_row(const EvictParams& p, int b, int to, int of, int lane) {
  const CacheView& c = p.cache;
  if (to < 0 || to >= c.capacity || of < 0 || of >= c.capacity) return;
  const long long dst = slot_offset(c, b, to), src = slot_offset(c, b, of);
  if (dst >= 0) {
    uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(c.data) + dst);
    const uint4* s = reinterpret_cast<const uint4*>(static_cast<uint16_t*>(c.data) + src);
    uint4 v[3];  // 72 pieces at most
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] = src >= 0 && lane + 32 * k < p.vecs ? s[lane + 32 * k] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (lane + 32 * k < p.vecs) o[lane + 32 * k] = v[k];
  }
  if (lane == 0) {
    p.score_out[b * p.score_out_stride + to] = p.score[b * p.score_stride + of];
    p.position_out[b * p.position_out_stride + to] = p.position[b * p.position_stride + of];
  }
}
static_assert(kMaxD / 8 <= 96, "move_row holds a row in three pieces a lane");

// A cluster of CTAs per sequence, each with a run of its slots. Finds the budget-th largest rank: the range of the ranks is cut into 512
// bins, the bin that holds it again, until the bin is one rank or holds so few that they can be compared with each other. Then the slots
// to fill and the slots to move, in order. Scores and positions are read from memory once; from then on ranks and positions lie in
// shared memory, and the CTAs of a cluster read each other's counts there.
//
// What it costs is neither bytes nor operations but a chain: some fifteen barriers (dearer between CTAs, and the more threads wait), the
// loads behind them, and code that is gone through once and waits for its instructions longer than for anything else. 64 sequences of
// 2049 slots 7.9 us, 8 of 16384 17.5, one of 131072 26.4 (14.4, 24.5 and 36 with fixed digits of the rank and both arrays read twice).
// 512 threads up to 8192 slots of a CTA, 1024 above: 7.9, 17.5 and 29.1 us with 512, 8.4, 18.6 and 26.4 with 1024 (with 256, one sequence
// of 131072 took 45). Up to 128 ranks are compared with each other: with 32, 64 sequences of 2049 slots took 8.7 us, with 256 16 of 5000
// 18.9 instead of 16.8. Loops rolled to save instructions waited for shared memory instead: 9.2, 19.7 and 30.5.
template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1) evict_select_kernel(const __grid_constant__ EvictParams p) {
  constexpr int kWarps = THREADS / 32, kBins = 512, kDigitBits = 9, kScan = kBins / 2, kAtOnce = 8, kFew = 128;
  constexpr int kDigits = 4;  // the first cut leaves one bin for the protected rows: 32 bits to 24, then 15, 6, none
  extern __shared__ uint32_t ranks[];
  __shared__ alignas(8) int bins[kDigits][kBins];
  __shared__ int holes_of[kMaxCluster], late_of[kMaxCluster];
  __shared__ uint32_t newest_of[kMaxCluster], lowest_of[kMaxCluster], highest_of[kMaxCluster], few[kFew];
  __shared__ int scratch[kWarps], found[4], equal[3], few_count, few_to[kFewMoves], few_of[kFewMoves];
  // Which of 32 slots lie above the threshold, and on it; then which are to fill, which to move, and how many of both lie before.
  __shared__ uint32_t above_words[THREADS], tie_words[THREADS], before_words[THREADS];
  const CacheView& c = p.cache;
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int cluster = p.cluster, b = static_cast<int>(blockIdx.x) / cluster, me = static_cast<int>(blockIdx.x) % cluster, budget = p.budget;
  auto arrive = [&]() {
    if (cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  };
  auto wait = [&]() {
    if (cluster > 1)
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    else
      __syncthreads();
  };
  // Two neighbouring values in sum, of all of the cluster's CTAs (x, y) and of those before this one (z, w). (All loads of a thread are
  // on their way together.)
  auto sum_over = [&](const int* mine) {
    if (cluster == 1) {
      const int2 v = *reinterpret_cast<const int2*>(mine);
      return make_int4(v.x, v.y, 0, 0);
    }
    int2 v[kMaxCluster];
    int4 s = make_int4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k) {
      v[k] = make_int2(0, 0);
      if (k >= cluster) continue;
      uint32_t at;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(mine)), "r"(k));
      asm volatile("ld.shared::cluster.v2.b32 {%0, %1}, [%2];" : "=r"(v[k].x), "=r"(v[k].y) : "r"(at) : "memory");
    }
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k) {
      s.x += v[k].x, s.y += v[k].y;
      if (k < me) s.z += v[k].x, s.w += v[k].y;
    }
    return s;
  };
  auto put = [&](const void* mine, int cta, uint32_t value) {  // into that CTA's shared memory
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(mine)), "r"(cta));
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(value) : "memory");
  };
  arrive();  // all CTAs are there once this is waited for
  for (int i = tid; i < kDigits * kBins; i += THREADS) (&bins[0][0])[i] = 0;
  if (tid == 0) few_count = 0;
  pdl_wait();
  pdl_launch_dependents();
  const int len = c.lens[b], n = max(0, min(len, c.capacity));
  const float* score = p.score + b * p.score_stride;
  const int* position = p.position + b * p.position_stride;
  float* score_out = p.score_out + b * p.score_out_stride;
  int* position_out = p.position_out + b * p.position_out_stride;
  if (n <= budget) {
    wait();
    arrive();  // lens_out may be lens: all have read it
    wait();
    if (me == 0 && tid == 0) {
      p.lens_out[b] = min(len, budget);
      if (!p.few) p.moves[b] = 0;
    }
    for (int i = me * THREADS + tid; i < n; i += cluster * THREADS) {
      score_out[i] = score[i];
      position_out[i] = position[i];
    }
    return;
  }
  const int run = ((n + cluster - 1) / cluster + 31) / 32 * 32, begin = min(n, me * run), count = min(n, begin + run) - begin;
  const int staged = p.staged;
  int* const positions = reinterpret_cast<int*>(ranks + staged);
  // Slots below the budget keep what they have for now; those given up are written again by the rows that move there.
  const bool copy_scores = score_out != score, copy_positions = position_out != position;
  int newest = INT_MIN;
  uint32_t lowest = 0xffffffffu, highest = 0u;
  for (int i0 = tid; i0 < count; i0 += kAtOnce * THREADS) {  // (stores between them would keep the compiler from loading ahead)
    float s[kAtOnce];
    int at[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (i0 + k * THREADS >= count) break;
      s[k] = score[begin + i0 + k * THREADS];
      at[k] = position[begin + i0 + k * THREADS];
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int i = i0 + k * THREADS;
      if (i >= count) break;
      const uint32_t r = rank_of(s[k]);
      newest = max(newest, at[k]);
      lowest = min(lowest, r);
      highest = max(highest, r);
      if (i < staged) {
        ranks[i] = r;
        positions[i] = at[k];
      }
      if (begin + i < budget) {
        if (copy_scores) score_out[begin + i] = s[k];
        if (copy_positions) position_out[begin + i] = at[k];
      }
    }
  }
  if (tid < 32 && count + tid < min(staged, (count + 31) / 32 * 32)) ranks[count + tid] = 0u;
  newest = __reduce_max_sync(0xffffffffu, newest);
  lowest = __reduce_min_sync(0xffffffffu, lowest);
  highest = __reduce_max_sync(0xffffffffu, highest);
  if (lane == 0) {  // (above_words and tie_words have their own use later)
    scratch[warp] = newest;
    above_words[warp] = lowest;
    tie_words[warp] = highest;
  }
  __syncthreads();
  newest = __reduce_max_sync(0xffffffffu, scratch[lane % kWarps]);
  lowest = __reduce_min_sync(0xffffffffu, above_words[lane % kWarps]);
  highest = __reduce_max_sync(0xffffffffu, tie_words[lane % kWarps]);
  if (cluster > 1) {  // every CTA's goes to all
    wait();
    if (tid < cluster) {
      put(&newest_of[me], tid, static_cast<uint32_t>(newest));
      put(&lowest_of[me], tid, lowest);
      put(&highest_of[me], tid, highest);
    }
    arrive();
    wait();
    for (int k = 0; k < cluster; ++k) {
      newest = max(newest, static_cast<int>(newest_of[k]));
      lowest = min(lowest, lowest_of[k]);
      highest = max(highest, highest_of[k]);
    }
  }
  if (me == 0 && tid == 0) p.lens_out[b] = budget;  // (all have read lens, which it may be)
  const long long safe_above = static_cast<long long>(newest) - p.recent;
  auto rank_at = [&](int i) {
    if (i < staged) return ranks[i];
    return position[begin + i] > safe_above ? kProtected : rank_of(score[begin + i]);
  };
  // f(slot, rank) for the thread's slots, four at a time. (The instructions that 1024 threads issue are what these loops cost.)
  auto each = [&](auto&& f) {
    const int near = min(count, staged);
    int i = tid;
    for (; i + 3 * THREADS < near; i += 4 * THREADS) {
      uint32_t r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) r[k] = ranks[i + k * THREADS];
#pragma unroll
      for (int k = 0; k < 4; ++k) f(i + k * THREADS, r[k]);
    }
    for (; i < near; i += THREADS) f(i, ranks[i]);
    for (; i < count; i += THREADS) f(i, rank_at(i));
  };
  int shift = max(0, 32 - __clz(static_cast<int>(highest - lowest)) - kDigitBits);
  if ((highest - lowest) >> shift > kBins - 2) ++shift;
  each([&](int i, uint32_t r) {
    if (i < staged && positions[i] > safe_above) ranks[i] = r = kProtected;
    atomicAdd(&bins[0][r == kProtected ? kBins - 1 : (r - lowest) >> shift], 1);
  });
  // Of the rows with the rank `lowest`, `left` are kept, of `ties`, of which `ties_before` belong to the CTAs before this one.
  int left = budget, ties = 0, ties_before = 0;
  for (int digit = 0;; ++digit) {
    arrive();
    wait();
    if (tid < kScan) {  // thread t has bins kBins - 1 - 2 t and the one below: counted from the top
      const int high = kBins - 1 - 2 * tid;
      const int4 pair = sum_over(&bins[digit][high - 1]);
      const int n0 = pair.y, n1 = pair.x;
      int upto = n0 + n1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      if (lane == 31) scratch[warp] = upto;
      asm volatile("bar.sync 1, %0;" ::"n"(kScan) : "memory");
      const int above = __reduce_add_sync(0xffffffffu, lane < warp ? scratch[lane] : 0) + upto - n0 - n1;
      if (above < left && left <= above + n0 + n1) {
        const bool second = left > above + n0;
        found[0] = high - (second ? 1 : 0);
        found[1] = above + (second ? n0 : 0);
        found[2] = second ? n1 : n0;
        found[3] = second ? pair.z : pair.w;
      }
    }
    __syncthreads();
    const int bin = found[0];
    left -= found[1];
    ties = found[2];
    ties_before = found[3];
    const bool safe = digit == 0 && bin == kBins - 1;  // more are protected than stay
    lowest = safe ? kProtected : lowest + (static_cast<uint32_t>(bin) << shift);
    if (safe || shift == 0) break;
    const uint32_t span = min(1u << shift, kProtected - lowest);  // (ranks below `lowest` are far above it in the difference)
    if (ties <= kFew) {
      uint32_t hits = 0;  // of up to 32 slots, looked for first: a warp would go through the rest for every slot
      int at = tid;
      auto hand_out = [&]() {
        for (; hits != 0; hits &= hits - 1) {
          const int to = ties_before + atomicAdd(&few_count, 1);
          const uint32_t r = rank_at(at + (__ffs(hits) - 1) * THREADS);
          for (int k = 0; k < cluster && to < kFew; ++k) put(&few[to], k, r);
        }
      };
      int seen = 0;
      each([&](int i, uint32_t r) {
        hits |= static_cast<uint32_t>(r - lowest < span) << seen;
        if (++seen == 32) {
          hand_out();
          at = i + THREADS;
          seen = 0;
        }
      });
      hand_out();
      arrive();
      wait();
      if (tid < ties) {
        const uint32_t mine = few[tid];
        int larger = 0, at_least = 0;
#pragma unroll 8
        for (int k = 0; k < ties; ++k) {
          larger += few[k] > mine;
          at_least += few[k] >= mine;
        }
        if (larger < left && left <= at_least) {  // (threads with the same rank write the same)
          equal[0] = static_cast<int>(mine);
          equal[1] = larger;
          equal[2] = at_least;
        }
      }
      __syncthreads();
      lowest = static_cast<uint32_t>(equal[0]);
      left -= equal[1];
      ties = equal[2] - equal[1];
      int same_before = 0;
      for (int k = lane; k < ties_before; k += 32) same_before += few[k] == lowest;
      ties_before = __reduce_add_sync(0xffffffffu, same_before);
      break;
    }
    shift = max(0, shift - kDigitBits);
    each([&](int, uint32_t r) {
      if (r - lowest < span) atomicAdd(&bins[digit + 1][(r - lowest) >> shift], 1);
    });
  }
  // The first `left` ties stay. A thread takes a word of 32 slots; slots of more words than threads are gone through in blocks, and
  // then twice.
  int* const holes_list = p.holes + static_cast<long long>(b) * p.most;
  int* const late_list = p.late + static_cast<long long>(b) * p.most;
  const int words = (count + 31) / 32, blocks = (words + THREADS - 1) / THREADS;
  int holes_at = 0, late_at = 0, moves = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int seen = ties_before, holes = 0, late = 0;
    for (int block = 0; block < blocks; ++block) {
      const int w0 = block * THREADS, here = min(THREADS, words - w0), holes_before = holes_at + holes, late_before = late_at + late;
      if (pass == 0 || blocks > 1) {
        __syncthreads();
#pragma unroll 4
        for (int w = warp; w < here; w += kWarps) {
          const int i = 32 * (w0 + w) + lane;
          const uint32_t r = i < staged || i < count ? rank_at(i) : 0u;  // (0, below all ranks, behind the last slot)
          const uint32_t above = __ballot_sync(0xffffffffu, r > lowest), tie = __ballot_sync(0xffffffffu, r == lowest);
          if (lane == 0) {
            above_words[w] = above;
            tie_words[w] = tie;
          }
        }
        __syncthreads();
        uint32_t stays = tid < here ? tie_words[tid] : 0u;
        if (left < ties) {  // the first of the word that stay: those below its (left - rank)-th
          int all;
          const int in_word = __popc(stays), rank = seen + threads_before<THREADS>(in_word, scratch, &all), stay = max(0, min(in_word, left - rank));
          if (stay < in_word) stays = stay == 0 ? 0u : stays & ((2u << __fns(stays, 0, stay)) - 1u);
          seen += all;
        }
        const uint32_t kept = stays | (tid < here ? above_words[tid] : 0u);
        const int slot = begin + 32 * (w0 + tid), in_run = count - 32 * (w0 + tid);
        const uint32_t valid = in_run >= 32 ? 0xffffffffu : in_run > 0 ? (1u << in_run) - 1u : 0u;
        const uint32_t low = budget - slot >= 32 ? 0xffffffffu : budget > slot ? (1u << (budget - slot)) - 1u : 0u;  // below the budget
        const uint32_t hole = ~kept & valid & low, moved = kept & ~low;
        int both;  // 16 bits each: at most 32768 slots in a block
        before_words[tid] = static_cast<uint32_t>(threads_before<THREADS>(__popc(moved) << 16 | __popc(hole), scratch, &both));
        above_words[tid] = hole;
        tie_words[tid] = moved;
        holes += both & 0xffff;
        late += static_cast<int>(static_cast<uint32_t>(both) >> 16);
      }
      if (pass == 1) {  // a warp per word, a lane per slot: stores lie together
        if (blocks > 1) __syncthreads();
        const uint32_t lower = (1u << lane) - 1u;
        for (int w = warp; w < here; w += kWarps) {
          const uint32_t hole = above_words[w], moved = tie_words[w], before = before_words[w];
          if ((hole | moved) == 0) continue;
          const int slot = begin + 32 * (w0 + w) + lane;
          const int to = holes_before + static_cast<int>(before & 0xffffu) + __popc(hole & lower);
          const int of = late_before + static_cast<int>(before >> 16) + __popc(moved & lower);
          // (The lists hold p.most slots, more than there are unless something else writes to the scores meanwhile.)
          const bool fill = (hole >> lane & 1u) && to < p.most, move = (moved >> lane & 1u) && of < p.most;
          if (!p.few) {
            if (fill) holes_list[to] = slot;
            if (move) late_list[of] = slot;
          } else if (fill || move) {  // every CTA moves some
            for (int k = 0; k < cluster; ++k) put(fill ? &few_to[to] : &few_of[of], k, static_cast<uint32_t>(slot));
          }
        }
      }
    }
    if (pass == 0) {
      if (tid < cluster) {
        put(&holes_of[me], tid, static_cast<uint32_t>(holes));
        put(&late_of[me], tid, static_cast<uint32_t>(late));
      }
      arrive();
      wait();
      for (int k = 0; k < cluster; ++k) {
        moves += holes_of[k];
        if (k < me) holes_at += holes_of[k], late_at += late_of[k];
      }
      moves = min(moves, p.most);
      if (me == 0 && tid == 0 && !p.few) p.moves[b] = moves;
    }
  }
  arrive();
  wait();  // the lists are complete, and no CTA leaves while another reads its counts
  if (p.few)
    for (int i = me * kWarps + warp; i < moves; i += cluster * kWarps) move_row(p, b, few_to[i], few_of[i], lane);
}

// A warp per moved row: the row, its score and its position. 8 sequences that move up to 2048 rows of 1152 bytes each: 8.4 us by itself
// from cold caches, some 30 MB.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int b = static_cast<int>(blockIdx.y), warps = static_cast<int>(gridDim.x) * (kMoveThreads / 32), moves = p.moves[b];
  for (int i = static_cast<int>(blockIdx.x) * (kMoveThreads / 32) + (static_cast<int>(threadIdx.x) >> 5); i < moves; i += warps) {
    const long long at = static_cast<long long>(b) * p.most + i;
    move_row(p, b, p.holes[at], p.late[at], static_cast<int>(threadIdx.x) & 31);
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------

// <<<grid, threads>>> on `stream`, allowed to begin under the kernel before it (see pdl_wait).
template <typename... Params>
int launch_clusters(void (*kernel)(Params...), int cluster, dim3 grid, int threads, size_t smem, void* stream, const std::decay_t<Params>&... params) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, params...) != cudaSuccess) {
    (void)cudaGetLastError();
    return B200_FP8_MM_ERR_LAUNCH;
  }
  return B200_FP8_MM_OK;
}

template <typename... Params>
int launch_pdl(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, void* stream, const std::decay_t<Params>&... params) {
  return launch_clusters(kernel, 1, grid, threads, smem, stream, params...);
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

constexpr int kMaxHeads = 1 << 16;
constexpr int kMaxDevices = 64;
constexpr int kLeastPlaces = 1;

// What beginning and ending a sequence costs a worker, in tiles: its accumulators are read out and written while the tensor core has
// little to do, with 64 heads 128 KB at the 32 bytes that an SM stores per clock. A segment's end takes 9000 clocks there and a tile 2950,
// but a place more also moves borders in short sequences, and neither is better throughout. With 64 heads to a tile, us with 1, 2 and 3:
// 64 ragged sequences up to 8192 rows, 128 heads 125.0, 121.0, 118.5; 128 up to 2048 88.8, 87.4, 85.8; 128 up to 400 49.3, 46.3, 47.5; 32
// up to 4096 50.3, 48.4, 48.1; 7 up to 3001 with 40 heads and dv 256 17.1, 18.1, 18.6.
int extra_for(int ht) { return ht < 64 ? 1 : 2; }

int current_device() {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    (void)cudaGetLastError();
    return -1;
  }
  return dev;
}

constexpr int kSmsOfB200 = 148;

// SM count of the current device, looked up once; B200's where there is none (sizes are asked for on hosts without a GPU too).
int sm_count_for_sizing() {
  static std::atomic<int> known[kMaxDevices];
  const int dev = current_device();
  if (dev < 0) return kSmsOfB200;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      return kSmsOfB200;
    }
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Heads per tile. N of the second product, and what the queries take of shared memory.
int tile_heads_for(int heads) { return heads <= 16 ? 16 : heads <= 32 ? 32 : 64; }

// Workers per head tile: one CTA per SM.
int attend_workers(int heads, int sms) {
  const int ht = tile_heads_for(heads), tiles = (heads + ht - 1) / ht;
  const int n = sms / tiles;
  return n < 1 ? 1 : n;
}

struct AttendWorkspace {
  size_t lse2, part_stat, part_out, logits, bytes;
};

AttendWorkspace attend_workspace(int batch, int heads, int dv, int max_len, bool with_score, int sms) {
  const int ht = tile_heads_for(heads);
  const size_t head_tiles = (heads + ht - 1) / ht;
  const size_t parts = 2 * head_tiles * attend_workers(heads, sms) * ht;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  AttendWorkspace w;
  w.lse2 = up((static_cast<size_t>(batch) + 1) * sizeof(long long));
  w.part_stat = w.lse2 + up(static_cast<size_t>(batch) * heads * sizeof(float));
  w.part_out = w.part_stat + up(parts * sizeof(float2));
  w.logits = w.part_out + up(parts * dv * sizeof(float));
  w.bytes = w.logits + (with_score ? up(static_cast<size_t>(batch) * cache_walk::tiles_of(max_len, tile_rows_for(ht)) * heads * tile_rows_for(ht) * sizeof(float)) : 0);
  return w;
}

// Tiles in the ring: as many as fit, two of the largest next to 64 heads. Returns the shared memory of the CTA.
size_t plan_ring(int ht, AttendParams* p) {
  const int fixed = kHeaderBytes + (p->chunks + 1) * ht * kRowBytes, tile = p->chunks * tile_rows_for(ht) * kRowBytes;
  const int fit = (kMaxSmem - fixed) / tile;
  p->stages = fit < kMaxStages ? fit : kMaxStages;
  return static_cast<size_t>(fixed) + p->stages * tile;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A map of 16-bit elements, 128-byte swizzle, first dimension and box 64 elements. What lies outside reads as 0. Encoded for every
// call: a map holds an address, and is not kept beyond the call that it was made for.
struct MapDims {
  int rank = 1;
  cuuint64_t dims[5] = {64}, strides[4] = {};
  cuuint32_t box[5] = {64};
  void add(long long extent, long long stride, int box_extent) {
    dims[rank] = static_cast<cuuint64_t>(extent);
    strides[rank - 1] = static_cast<cuuint64_t>(stride) * 2;
    box[rank++] = static_cast<cuuint32_t>(box_extent);
  }
  bool encode(CUtensorMap* map, const void* base, bool bf16) const {
    static const EncodeTiledFn fn = []() -> EncodeTiledFn {
      void* ptr = nullptr;
      cudaDriverEntryPointQueryResult found;
      if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
        (void)cudaGetLastError();
        return nullptr;
      }
      return reinterpret_cast<EncodeTiledFn>(ptr);
    }();
    const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
    return fn != nullptr &&
           fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, static_cast<cuuint32_t>(rank),
              const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  }
};

typedef void (*AttendFn)(const CUtensorMap, const CUtensorMap, const AttendParams);

AttendFn attend_fn(bool bf16, int ht) {
  if (bf16) return ht == 16 ? attend_kernel<__nv_bfloat16, 16> : ht == 32 ? attend_kernel<__nv_bfloat16, 32> : attend_kernel<__nv_bfloat16, 64>;
  return ht == 16 ? attend_kernel<__half, 16> : ht == 32 ? attend_kernel<__half, 32> : attend_kernel<__half, 64>;
}

// Their own kernels: looking for the tile to leave out in every launch cost 0.4 % (128 x 4096 rows, 16 heads: 113.0 against 112.6 us).
AttendFn attend_selftest_fn(int ht) {
  return ht == 16 ? attend_kernel<__nv_bfloat16, 16, true> : ht == 32 ? attend_kernel<__nv_bfloat16, 32, true> : attend_kernel<__nv_bfloat16, 64, true>;
}

// Lets a kernel take that much shared memory, once per device.
template <typename Fn>
bool opt_in(Fn fn, int bytes, std::atomic<bool>* done) {
  if (done->load(std::memory_order_relaxed)) return true;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    (void)cudaGetLastError();
    return false;
  }
  done->store(true, std::memory_order_relaxed);
  return true;
}

// b200_mla_cache_attend, and its self-test with a shorter limit for the waits and a tile that is left out.
int run_attend(const b200_mla_cache* cache, const void* q, long long q_sb, long long q_sh, int heads, float scale, void* out,
               long long out_sb, long long out_sh, float* lse, const float* score, long long score_stride, float* score_out,
               long long score_out_stride, int max_len, void* workspace, size_t workspace_bytes, int* device_status, void* stream,
               unsigned long long wait_limit_ns, int selftest_skip_tile) {
  AttendParams p = {};
  int rc = view_of(cache, &p.cache);
  if (rc != B200_FP8_MM_OK) return rc;
  if (q == nullptr || out == nullptr || (score_out != nullptr && score == nullptr)) return B200_FP8_MM_ERR_NULL;
  if (heads <= 0 || heads > kMaxHeads || max_len < 0 || !(fabsf(scale) < 0x1p127f)) return B200_FP8_MM_ERR_SHAPE;
  if (cache->batch == 1) q_sb = p.cache.d;  // (no second one)
  if (heads == 1) q_sh = p.cache.d;
  if (q_sb % 8 != 0 || q_sh % 8 != 0 || q_sb < p.cache.d || q_sh < p.cache.d) return B200_FP8_MM_ERR_STRIDE;
  if (!aligned16(q)) return B200_FP8_MM_ERR_ALIGN;
  if (max_len == 0 || max_len > p.cache.capacity) max_len = p.cache.capacity;
  const int sms = sm_count_for_sizing();
  const AttendWorkspace w = attend_workspace(cache->batch, heads, cache->dv, max_len, score_out != nullptr, sms);
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 || workspace_bytes < w.bytes) return B200_FP8_MM_ERR_WORKSPACE;
  const int ht = tile_heads_for(heads), device = current_device();
  if (device < 0) return B200_FP8_MM_ERR_DRIVER;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.out = out;
  p.lse = lse;
  p.score = score;
  p.score_out = score_out;
  p.out_sb = out_sb;
  p.out_sh = out_sh;
  p.score_stride = score_stride;
  p.score_out_stride = score_out_stride;
  p.heads = heads;
  p.head_tiles = (heads + ht - 1) / ht;
  p.max_len = max_len;
  p.batch = cache->batch;
  p.workers = attend_workers(heads, sms);
  p.least = kLeastPlaces + extra_for(ht);
  p.tile = tile_rows_for(ht);
  p.extra = extra_for(ht);
  p.copy_rows = cache_walk::copy_rows(cache->page_size, p.tile);
  if (p.copy_rows < 8) p.copy_rows = 0;
  p.v_units = cache->dv / 128;
  p.chunks = p.cache.d / 64;
  p.scale_log2 = scale * kLog2E;
  p.joined = cache_walk::tiles_of(max_len, p.tile) > cache_walk::kWholeTiles;
  p.begins = reinterpret_cast<long long*>(ws);
  p.lse2 = reinterpret_cast<float*>(ws + w.lse2);
  p.part_stat = reinterpret_cast<float2*>(ws + w.part_stat);
  p.part_out = reinterpret_cast<float*>(ws + w.part_out);
  p.logits = score_out != nullptr ? reinterpret_cast<float*>(ws + w.logits) : nullptr;
  p.logit_tiles = cache_walk::tiles_of(max_len, p.tile);
  p.status = device_status;
  p.selftest_wait_limit_ns = wait_limit_ns;
  p.selftest_skip_tile = selftest_skip_tile;
  const size_t smem = plan_ring(ht, &p);
  const bool bf16 = cache->dtype == B200_MLA_CACHE_BF16;
  CUtensorMap q_map, row_map;
  MapDims q_dims, row_dims;
  q_dims.add(heads, q_sh, ht);
  q_dims.add(p.chunks, 64, p.chunks);
  q_dims.add(cache->batch, q_sb, 1);
  if (p.copy_rows > 0) {
    row_dims.add(8, cache->slot_stride, 8);
    row_dims.add(p.chunks, 64, p.chunks);
    row_dims.add(cache->page_size / 8, 8 * cache->slot_stride, p.copy_rows / 8);
    row_dims.add(cache->pages, cache->page_stride, 1);
  }
  if (!q_dims.encode(&q_map, q, bf16)) return B200_FP8_MM_ERR_DRIVER;
  if (p.copy_rows == 0)
    row_map = q_map;  // (not used)
  else if (!row_dims.encode(&row_map, cache->data, bf16))
    return B200_FP8_MM_ERR_DRIVER;
  const bool selftest = selftest_skip_tile >= 0;
  if (selftest && !bf16) return B200_FP8_MM_ERR_SHAPE;
  const AttendFn fn = selftest ? attend_selftest_fn(ht) : attend_fn(bf16, ht);
  static std::atomic<bool> opted[kMaxDevices][9];
  if (!opt_in(fn, kMaxSmem, &opted[device][(selftest ? 6 : bf16 ? 0 : 3) + (ht == 16 ? 0 : ht == 32 ? 1 : 2)])) return B200_FP8_MM_ERR_DRIVER;
  rc = launch_pdl(fn, dim3(static_cast<unsigned>(p.workers) * p.head_tiles), kAttendThreads, smem, stream, q_map, row_map, p);
  if (rc != B200_FP8_MM_OK) return rc;
  // Eight groups where a sequence has eight parts and more on average, one where most have one or two.
  auto joins = [&](int groups) {
    return dim3(static_cast<unsigned>((heads + join_heads(groups) - 1) / join_heads(groups)), static_cast<unsigned>(cache->batch));
  };
  if (!p.joined)
    rc = B200_FP8_MM_OK;
  else if (p.workers / cache->batch >= 8)
    rc = launch_pdl(bf16 ? attend_join_kernel<__nv_bfloat16, 8> : attend_join_kernel<__half, 8>, joins(8), 1024, 0, stream, p, ht);
  else
    rc = launch_pdl(bf16 ? attend_join_kernel<__nv_bfloat16, 1> : attend_join_kernel<__half, 1>, joins(1), 128, 0, stream, p, ht);
  if (rc != B200_FP8_MM_OK || score_out == nullptr) return rc;
  const dim3 tiles(static_cast<unsigned>(p.logit_tiles), static_cast<unsigned>(cache->batch));
  return launch_pdl(p.tile == 64 ? attend_score_kernel<64> : attend_score_kernel<48>, tiles, kScoreGroups * p.tile, 0, stream, p);
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
  const bool vec = aligned16(row) && row_stride % 8 == 0 &&
          (q == nullptr || (aligned16(q) && aligned16(q_out) && q_sb % 8 == 0 && q_sh % 8 == 0 && qo_sb % 8 == 0 && qo_sh % 8 == 0));
  for (int t = 0; t < p.half; ++t) p.turns[t] = pow(theta, -static_cast<double>(t) / p.half) / 6.283185307179586476925;
  const dim3 grid(static_cast<unsigned>(1 + (p.heads + kAppendHeads - 1) / kAppendHeads), static_cast<unsigned>(cache->batch));
  if (cache->dtype == B200_MLA_CACHE_BF16)
    return launch_pdl(vec ? append_kernel<__nv_bfloat16, true> : append_kernel<__nv_bfloat16, false>, grid, kAppendThreads, 0, stream, p);
  return launch_pdl(vec ? append_kernel<__half, true> : append_kernel<__half, false>, grid, kAppendThreads, 0, stream, p);
}

size_t b200_mla_cache_attend_workspace_bytes(int batch, int heads, int dv, int dr, int max_len, int with_score) {
  (void)dr;
  if (batch <= 0 || heads <= 0 || dv <= 0 || max_len <= 0) return 0;
  return attend_workspace(batch, heads, dv, max_len, with_score != 0, sm_count_for_sizing()).bytes;
}

int b200_mla_cache_attend(const b200_mla_cache* cache, const void* q, long long q_sb, long long q_sh, int heads, float scale,
                          void* out, long long out_sb, long long out_sh, float* lse, const float* score,
                          long long score_stride, float* score_out, long long score_out_stride, int max_len, void* workspace,
                          size_t workspace_bytes, int* device_status, void* stream) {
  return run_attend(cache, q, q_sb, q_sh, heads, scale, out, out_sb, out_sh, lse, score, score_stride, score_out, score_out_stride,
                    max_len, workspace, workspace_bytes, device_status, stream, kWaitLimitNs, -1);
}

int b200_mla_cache_attend_selftest_wait_expiry(const b200_mla_cache* cache, const void* q, long long q_sb, long long q_sh, int heads,
                                               float scale, void* out, long long out_sb, long long out_sh, void* workspace,
                                               size_t workspace_bytes, unsigned long long wait_limit_ns, int skip_tile,
                                               int* device_status, void* stream) {
  if (device_status == nullptr) return B200_FP8_MM_ERR_NULL;
  if (skip_tile < 0) return B200_FP8_MM_ERR_SHAPE;
  // Soon, because the GPU is busy until then, but later than any wait that is only slow.
  if (wait_limit_ns < 1000000ull || wait_limit_ns > 100000000ull) return B200_FP8_MM_ERR_PLAN;
  return run_attend(cache, q, q_sb, q_sh, heads, scale, out, out_sb, out_sh, nullptr, nullptr, 0, nullptr, 0, 0, workspace,
                    workspace_bytes, device_status, stream, wait_limit_ns, skip_tile);
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
  // CTAs per sequence: 4096 slots each where the batch leaves SMs for it. (64 sequences of 2049 slots with 1024 threads: 8.4 us with one
  // CTA each, 10.7 with two. One of 16000: 15.6 us with four, 15.3 with eight, 18.3 with two.)
  p.cluster = 1;
  const int sms = sm_count_for_sizing();
  while (p.cluster < kMaxCluster && 2 * p.cluster * cache->batch <= sms && p.cache.capacity > 4096 * p.cluster) p.cluster *= 2;
  const int slots = ((p.cache.capacity + p.cluster - 1) / p.cluster + 31) / 32 * 32;
  p.staged = slots < kMaxStaged ? slots : kMaxStaged;
  p.few = p.most <= kFewMoves;
  const int device = current_device();
  static std::atomic<bool> opted[kMaxDevices][2];
  const bool few_slots = slots <= 8192;
  const auto select = few_slots ? evict_select_kernel<512> : evict_select_kernel<1024>;
  if (device < 0 || !opt_in(select, kMaxStaged * 8, &opted[device][few_slots])) return B200_FP8_MM_ERR_DRIVER;
  rc = launch_clusters(select, p.cluster, dim3(static_cast<unsigned>(cache->batch * p.cluster)), few_slots ? 512 : 1024,
                       static_cast<size_t>(p.staged) * 8, stream, p);
  if (rc != B200_FP8_MM_OK || p.most == 0 || p.few) return rc;
  const int want = (p.most + kMoveThreads / 32 - 1) / (kMoveThreads / 32);
  const int fill = (sms * 8 + cache->batch - 1) / cache->batch;
  const dim3 grid(static_cast<unsigned>(want < fill ? want : fill), static_cast<unsigned>(cache->batch));
  return launch_pdl(evict_move_kernel, grid, kMoveThreads, 0, stream, p);
}

}  // extern "C"
