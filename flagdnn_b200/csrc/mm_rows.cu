// A product of few rows with its epilogue: y = act(a b + bias + residual).
//
// With one to some dozens of rows a product is a reading of b.  A block takes 64 columns of b (or 128) and, with the others of its cluster, a
// share of the reduction; b's tiles come through a ring of asynchronous copies, all of a block's first ones on their way at once.  On the tensor
// cores columns are the M side (16 a warp) and rows the N side (8 at a time), so that a single row fills an eighth of an
// instruction and not a 128th.  The blocks of a cluster add up their sums through each other's shared memory, in their order, and finish
// a share of the columns each: no workspace, no atomics.
//
// Sums are fp32; fp32 operands go in as 3 x TF32 (a high part, and what it leaves: 2^-22); one rounding at the end.  The tensor cores cut
// what they add to an accumulator, always towards zero: a sum of 4096 fp32 products that stays in one is 3e-5 too small.  Each step of the
// ring (32 or 64 products) therefore has accumulators of its own, which are added to the sums in fp32 (at most 4e-7, 2e-7 in the mean).  That
// is why fp32 products of any size come here: many rows in blocks of 64 x 128, whose operands are split once for eight or four products each.
#include "group_norm.cuh"
#include "mma_sync.cuh"
#include "mm_rows.h"

namespace fdnn {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kTileBytes = 128;           // of the reduction, a step of the ring
constexpr int kPitch = kTileBytes + 16;   // eight rows of 16 bytes lie in different banks
// Steps of the ring: some 90 KB, two blocks to an SM; four of 64 fp32 rows (300 x 1000 x 777 28.3 us with three steps, 21.0 with four;
// 64 x 2048 x 4096 33.0 and 34.9).
template <typename T>
constexpr int stages_of(int rows, int cols) {
  return cols == 128 ? 4 : rows <= 16 ? 8 : rows <= 32 ? 6 : sizeof(T) == 4 ? 4 : 5;
}
constexpr int kShortRing = 4;   // .. four blocks to an SM

template <int BYTES>
__device__ __forceinline__ void copy_few(uint32_t to, const void* from, bool there) {   // 4 or 8, or as many zeros
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(there ? BYTES : 0) : "memory");
}
__device__ __forceinline__ float cluster_f32(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

enum class Order { kReduction, kColumns, kAny };   // what lies together in b, in 16-byte pieces; kAny: in fewer bytes, or value by value

// ACROSS x LINES values to shared memory in pieces of UNIT, neighbouring threads across: a thread keeps its place across, and walks lines.
// `across_step` and `line_step` are the strides of the source, the bytes those of shared memory; zeros from the bounds on.
template <typename T, int ACROSS, int LINES, int UNIT>
__device__ __forceinline__ void few_bytes(uint8_t* smem, int at, int line_bytes, int across_bytes, const T* src, const T* safe, long long line_step,
                                          long long across_step, int lines, int across) {
  constexpr int kAcross = ACROSS / UNIT, kBy = kThreads / kAcross;
  const uint32_t base = smem_u32(smem);
  const int place = threadIdx.x % kAcross * UNIT, first = threadIdx.x / kAcross, most = place < across ? lines : 0;
  src += place * across_step + first * line_step;
  at += place * across_bytes + first * line_bytes;
  constexpr int kCount = LINES / kBy;
  if constexpr (sizeof(T) * UNIT >= 4) {
#pragma unroll
    for (int n = 0; n < kCount; ++n, src += kBy * line_step, at += kBy * line_bytes) {
      const bool there = first + n * kBy < most;
      copy_few<int(sizeof(T)) * UNIT>(base + at, there ? src : safe, there);
    }
  } else {   // (two bytes cannot be copied asynchronously: all on their way before the first is stored)
    T v[kCount];
#pragma unroll
    for (int n = 0; n < kCount; ++n, src += kBy * line_step) v[n] = first + n * kBy < most ? *src : from_f32<T>(0.0f);
#pragma unroll
    for (int n = 0; n < kCount; ++n, at += kBy * line_bytes) *reinterpret_cast<T*>(smem + at) = v[n];
  }
}

// ROWS: of a, 16, 32 or 64 to a block.  WIDE: 16 columns to a warp, times this.  A_WHOLE: 16 bytes of a row of a are copied at once.
template <typename T, int ROWS, int WIDE, Order ORDER, bool A_WHOLE, int STAGES>
__global__ void __launch_bounds__(kThreads)
mm_rows_kernel(const MmRowsParams p, int split) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  chained();
  constexpr int kV = 16 / int(sizeof(T)), kStep = kTileBytes / int(sizeof(T)), kCols = 16 * WIDE * kWarps;
  constexpr int kWord = sizeof(T) == 2 ? 2 : 1;   // values in four bytes
  constexpr int kColTile = kCols * kPitch, kStage = kColTile + ROWS * kPitch;   // (b's tile takes that in either order)
  // columns together: rows of 64 columns, a step of the reduction apart
  constexpr int kColPitch = ORDER == Order::kColumns ? kCols * int(sizeof(T)) + (sizeof(T) == 2 ? 16 : 32) : kPitch;
  static_assert(ORDER != Order::kColumns || kStep * kColPitch <= kColTile, "fits the tile's place");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, m = lane >> 3, r = lane & 7;
  const int rank = int(blockIdx.x % split), col0 = int(blockIdx.x / split) * kCols;
  const int row0 = int(blockIdx.z * gridDim.y + blockIdx.y) * ROWS;   // (as many layers of blocks as 65535 to a layer ask for)
  if (row0 >= p.M) return;
  const int steps = (p.K + kStep - 1) / kStep;
  const int from = int((long long)steps * rank / split), to = int((long long)steps * (rank + 1) / split);
  const uint32_t smem = smem_u32(smem_raw);
  const T *a0 = static_cast<const T*>(p.a) + row0 * p.a_s[0], *b0 = static_cast<const T*>(p.b) + col0 * p.b_s[1];

  auto ask = [&](int step) {
    if (step < to) {
      const int at = (step - from) % STAGES * kStage, k0 = step * kStep;
      if constexpr (ORDER == Order::kReduction) {
#pragma unroll
        for (int i = tid; i < kCols * 8; i += kThreads) {
          const int c = i / 8, k = k0 + i % 8 * kV;
          const bool there = col0 + c < p.N && k < p.K;
          copy16(smem + at + c * kPitch + i % 8 * 16, there ? b0 + c * p.b_s[1] + k : b0, there ? 16 : 0);
        }
      } else if constexpr (ORDER == Order::kColumns) {
        constexpr int kPieces = kCols / kV;
#pragma unroll
        for (int i = tid; i < kStep * kPieces; i += kThreads) {
          const int k = i / kPieces, c = i % kPieces * kV;
          const bool there = col0 + c < p.N && k0 + k < p.K;
          copy16(smem + at + k * kColPitch + i % kPieces * 16, there ? b0 + (k0 + k) * p.b_s[0] + c : b0, there ? 16 : 0);
        }
      } else {
        // threads side by side along what lies together; along the reduction eight or four bytes at once, where all places allow it
        if (p.b_s[0] != 1) few_bytes<T, kCols, kStep, 1>(smem_raw, at, int(sizeof(T)), kPitch, b0 + k0 * p.b_s[0], b0, p.b_s[0], p.b_s[1], p.K - k0, p.N - col0);
        else if (p.b_bytes == 8) few_bytes<T, kStep, kCols, 2 * kWord>(smem_raw, at, kPitch, int(sizeof(T)), b0 + k0, b0, p.b_s[1], 1, p.N - col0, p.K - k0);
        else if (p.b_bytes == 4) few_bytes<T, kStep, kCols, kWord>(smem_raw, at, kPitch, int(sizeof(T)), b0 + k0, b0, p.b_s[1], 1, p.N - col0, p.K - k0);
        else few_bytes<T, kStep, kCols, 1>(smem_raw, at, kPitch, int(sizeof(T)), b0 + k0, b0, p.b_s[1], 1, p.N - col0, p.K - k0);
      }
      const int a_at = at + kColTile;
      if constexpr (A_WHOLE) {
#pragma unroll
        for (int i = tid; i < ROWS * 8; i += kThreads) {
          const int row = i / 8, k = k0 + i % 8 * kV;
          const bool there = row0 + row < p.M && k < p.K;
          copy16(smem + a_at + row * kPitch + i % 8 * 16, there ? a0 + row * p.a_s[0] + k : static_cast<const T*>(p.a), there ? 16 : 0);
        }
      } else {
        const T* safe = static_cast<const T*>(p.a);
        if (p.a_bytes == 8) few_bytes<T, kStep, ROWS, 2 * kWord>(smem_raw, a_at, kPitch, int(sizeof(T)), a0 + k0, safe, p.a_s[0], 1, p.M - row0, p.K - k0);
        else if (p.a_bytes == 4) few_bytes<T, kStep, ROWS, kWord>(smem_raw, a_at, kPitch, int(sizeof(T)), a0 + k0, safe, p.a_s[0], 1, p.M - row0, p.K - k0);
        else few_bytes<T, kStep, ROWS, 1>(smem_raw, a_at, kPitch, int(sizeof(T)), a0 + k0 * p.a_s[1], safe, p.a_s[0], p.a_s[1], p.M - row0, p.K - k0);
      }
    }
    async_commit();
  };

  float sum[WIDE][ROWS / 8][4] = {};
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) ask(from + i);
  for (int step = from; step < to; ++step) {
    async_wait<STAGES - 2>();
    __syncthreads();
    ask(step + STAGES - 1);
    const int at = (step - from) % STAGES * kStage;
    float d[WIDE][ROWS / 8][4] = {};
    if constexpr (sizeof(T) == 2) {
      static_assert(WIDE == 1, "wide blocks are fp32's");
      const uint32_t cols = smem + at, rows = smem + at + kColTile;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a[4];
        if constexpr (ORDER == Order::kColumns) ldmatrix<true>(a, cols + (k * 16 + (m >> 1) * 8 + r) * kColPitch + (warp * 16 + (m & 1) * 8) * 2);
        else ldmatrix<false>(a, cols + (warp * 16 + (m & 1) * 8 + r) * kPitch + (k * 16 + (m >> 1) * 8) * 2);
#pragma unroll
        for (int j = 0; j < ROWS / 16; ++j) {
          uint32_t b[4];
          ldmatrix<false>(b, rows + (j * 16 + (m >> 1) * 8 + r) * kPitch + (k * 16 + (m & 1) * 8) * 2);
          mma<T>(d[0][2 * j], a, b[0], b[1]);
          mma<T>(d[0][2 * j + 1], a, b[2], b[3]);
        }
      }
    } else {
      const float *cols = reinterpret_cast<const float*>(smem_raw + at), *rows = reinterpret_cast<const float*>(smem_raw + at + kColTile);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a[WIDE][4], al[WIDE][4];
#pragma unroll
        for (int n = 0; n < WIDE; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = (warp * WIDE + n) * 16 + g + (i & 1) * 8, kk = k * 8 + t + (i >> 1) * 4;
            two_parts(ORDER == Order::kColumns ? cols[kk * (kColPitch / 4) + c] : cols[c * (kPitch / 4) + kk], a[n][i], al[n][i]);
          }
        uint32_t b[ROWS / 8][2], bl[ROWS / 8][2];
#pragma unroll
        for (int j = 0; j < ROWS / 8; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) two_parts(rows[(j * 8 + g) * (kPitch / 4) + k * 8 + t + i * 4], b[j][i], bl[j][i]);
        // (a product waits for the one before it on the same accumulator: all of one kind, then all of the next)
#pragma unroll
        for (int n = 0; n < WIDE; ++n)
#pragma unroll
          for (int j = 0; j < ROWS / 8; ++j) mma<T>(d[n][j], a[n], bl[j][0], bl[j][1]);
#pragma unroll
        for (int n = 0; n < WIDE; ++n)
#pragma unroll
          for (int j = 0; j < ROWS / 8; ++j) mma<T>(d[n][j], al[n], b[j][0], b[j][1]);
#pragma unroll
        for (int n = 0; n < WIDE; ++n)
#pragma unroll
          for (int j = 0; j < ROWS / 8; ++j) mma<T>(d[n][j], a[n], b[j][0], b[j][1]);
      }
    }
#pragma unroll
    for (int n = 0; n < WIDE; ++n)
#pragma unroll
      for (int j = 0; j < ROWS / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[n][j][i] += d[n][j][i];
  }
  async_wait<0>();
  __syncthreads();
  // sums to shared memory, [row][column]; then every block of the cluster finishes its share of the columns
  constexpr int kSumPitch = kCols + 4;
  float* sums = reinterpret_cast<float*>(smem_raw);
#pragma unroll
  for (int n = 0; n < WIDE; ++n)
#pragma unroll
    for (int j = 0; j < ROWS / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[(j * 8 + 2 * t + (i & 1)) * kSumPitch + (warp * WIDE + n) * 16 + g + (i >> 1) * 8] = sum[n][j][i];
  if (split > 1) cluster_sync_all();
  else __syncthreads();
  const int share = kCols / split, c0 = rank * share, rows = min(ROWS, p.M - row0);
  with_activation(p.act, [&](auto act) {
    for (int i = tid; i < rows * share; i += kThreads) {
      const int row = i / share, c = c0 + i % share;
      const uint32_t at = smem + uint32_t(row * kSumPitch + c) * 4;
      float v = 0.0f;
      if (split > 1) {
        for (int q = 0; q < split; ++q) v += cluster_f32(map_to_cta(at, uint32_t(q)));
      } else {
        v = sums[row * kSumPitch + c];
      }
      if (col0 + c >= p.N) continue;
      const long long y_row = row0 + row;
      if (p.bias != nullptr) v += to_f32<T>(static_cast<const T*>(p.bias)[col0 + c]);
      if (p.residual != nullptr) v += to_f32<T>(static_cast<const T*>(p.residual)[y_row * p.residual_s[0] + (col0 + c) * p.residual_s[1]]);
      static_cast<T*>(p.y)[y_row * p.y_s[0] + (col0 + c) * p.y_s[1]] = from_f32<T>(activate<decltype(act)::value>(v));
    }
  });
  if (split > 1) cluster_sync_all();   // (the others have read this block's sums)
}

template <typename T, int ROWS, int WIDE, Order ORDER, bool A_WHOLE>
cudaError_t go(const MmRowsParams& p, cudaStream_t stream) {
  constexpr int kCols = 16 * WIDE * kWarps, kStep = kTileBytes / int(sizeof(T));
  const long long tiles = (p.N + kCols - 1) / kCols, row_blocks = (p.M + ROWS - 1) / ROWS;
  const int steps = (p.K + kStep - 1) / kStep;
  const long long layers = (row_blocks + 65534) / 65535;
  if (tiles > 0x7fffffffll / 8 || layers > 65535) return cudaErrorInvalidConfiguration;
  // parts of the reduction: as many blocks as run at once, as long as each has two steps
  auto split_of = [&](int at_once) {
    int split = 1;
    while (split < 8 && 2 * split * tiles * row_blocks <= (long long)at_once * current_sm_count() && steps >= 4 * split) split *= 2;
    return split;
  };
  auto run = [&](auto stages, int split) -> cudaError_t {
    constexpr int kStages = decltype(stages)::value, kSmem = kStages * (kCols + ROWS) * kPitch;
    static_assert(ROWS * (kCols + 4) * 4 <= kSmem, "the sums fit");
    static std::atomic<uint64_t> done;
    auto* kernel = mm_rows_kernel<T, ROWS, WIDE, ORDER, A_WHOLE, kStages>;
    constexpr int kRoom = 227 * 1024, kAlone = 5;   // (five blocks leave no room to spread)
    const cudaError_t e = allow_smem(kernel, kRoom, done);
    if (e != cudaSuccess) return e;
    // No more blocks to an SM than an even spread has, where all of them still run at once: three blocks on some SMs and one on others take
    // 44.9 us, two on each 35.0 (fp32, 64 x 2048 x 4096).  Clusters need their blocks in one group of SMs, so fewer fit than SMs would
    // hold: sixteen clusters of eight with an SM to a block ran in two waves (bf16, 16 x 1024 x 1024: 7.1 us for 4.4).
    // Not where two steps read the same 128 bytes of a row, which shorter rings leave in the L1 cache (2 x 7260 x 2432: 16.5 us, 21.2 with
    // it); values one by one across columns lose there at times (fp32, 7 x 792 x 7905: 15.7 to 18.0) and gain more often (bf16,
    // 33 x 7295 x 726: 36.9 to 32.7).
    const long long blocks = tiles * split * row_blocks, each = (blocks + current_sm_count() - 1) / current_sm_count();
    int smem = kSmem;
    if (!(ORDER == Order::kAny && p.b_s[0] == 1) && each < kAlone && int(kRoom / each) - 2048 > kSmem) {
      const int even = int(kRoom / each) - 2048, of = split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3;
      static ClusterCounts known[kAlone][4];
      if (tiles * row_blocks <= clusters_at_once(kernel, kThreads, even, split, known[each][of])) smem = even;
    }
    return launch_seq(kernel, dim3(unsigned(tiles * split), unsigned((row_blocks + layers - 1) / layers), unsigned(layers)), kThreads, smem, split, stream, p, split);
  };
  // One row, bf16, two blocks to an SM, 2048 x 4096 9.8 / 8.1 / 6.1 / 9.0 us in 1 / 2 / 4 / 8 parts (64 to 512 blocks), 4096 x 8192 20.8 / 16.0 /
  // 18.5 / 23.4 (128 to 1024).  Where two parts too many would not run at once (7264 x 2432: 152 blocks of 4 parts 15.5 us), blocks of half the
  // ring do, four to an SM (304 of 8 parts 12.7, 11.5 evenly spread; 4096 x 2048, 256 blocks either way, 6.3 and 7.9).
  constexpr int kStages = stages_of<T>(ROWS, kCols);
  constexpr int kAtOnce = 227 * 1024 / (kStages * (kCols + ROWS) * kPitch + 1024);
  const int split = split_of(kAtOnce);
  if constexpr (kStages > 2 * kShortRing - 1) {
    const int more = split_of(2 * kAtOnce);
    if (more > split && 4 * split * tiles * row_blocks < 3ll * kAtOnce * current_sm_count()) return run(std::integral_constant<int, kShortRing>{}, more);
  }
  return run(std::integral_constant<int, kStages>{}, split);
}

template <typename T>
cudaError_t by_layout(MmRowsParams p, cudaStream_t stream) {
  constexpr int kV = 16 / int(sizeof(T));
  // a stride over an extent of one says nothing (a vector as b, 16 x 4096 x 1 in bf16: 10.2 us as if it did, 4.7 so)
  if (p.M == 1) p.a_s[0] = 0;
  if (p.N == 1) p.b_s[1] = 0;
  auto whole = [&](const void* q, long long along, long long across, long long extent) {
    return along == 1 && (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && across % kV == 0 && extent % kV == 0;
  };
  const bool a_whole = whole(p.a, p.a_s[1], p.a_s[0], p.K);
  const Order order = whole(p.b, p.b_s[0], p.b_s[1], p.K) ? Order::kReduction : whole(p.b, p.b_s[1], p.b_s[0], p.N) ? Order::kColumns : Order::kAny;
  auto bytes = [&](const void* q, long long along, long long across) {   // that can be copied at once along the reduction
    if (along != 1) return 0;
    for (int n = 8; n >= 4; n /= 2)
      if (reinterpret_cast<uintptr_t>(q) % n == 0 && across * int(sizeof(T)) % n == 0 && (long long)p.K * int(sizeof(T)) % n == 0) return n;
    return 0;
  };
  p.a_bytes = bytes(p.a, p.a_s[1], p.a_s[0]);
  p.b_bytes = bytes(p.b, p.b_s[0], p.b_s[1]);
  auto rows = [&](auto count, auto wide) -> cudaError_t {
    constexpr int R = decltype(count)::value, W = decltype(wide)::value;
    if (order == Order::kReduction) return a_whole ? go<T, R, W, Order::kReduction, true>(p, stream) : go<T, R, W, Order::kReduction, false>(p, stream);
    if (order == Order::kColumns) return a_whole ? go<T, R, W, Order::kColumns, true>(p, stream) : go<T, R, W, Order::kColumns, false>(p, stream);
    return a_whole ? go<T, R, W, Order::kAny, true>(p, stream) : go<T, R, W, Order::kAny, false>(p, stream);
  };
  constexpr std::integral_constant<int, 1> one{};
  if (p.M <= 16) return rows(std::integral_constant<int, 16>{}, one);
  if (p.M <= 32) return rows(std::integral_constant<int, 32>{}, one);
  if constexpr (sizeof(T) == 4) {
    // 128 columns split rows of a half as often, 64 spread short reductions over more blocks: us with 64 and with 128, 100 x 2048 x 4096 65 and
    // 52, 1000 x 4096 x 1024 229 and 181, 8192 x 4096 x 4096 5850 and 4540; 3000 x 500 x 500 51 and 59, 300 x 1000 x 777 21 and 31
    const bool many = (p.M + 63ll) / 64 * ((p.N + 127ll) / 128) >= 2 * current_sm_count();
    if (p.M > 64 && (p.K > 1024 || many)) return rows(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  }
  return rows(std::integral_constant<int, 64>{}, one);
}

}  // namespace

// Its time goes with N K and, slowly, with M; the convolution's, on tiles of 128 rows, with K alone as long as they run at once.  16-bit,
// us here and there: K = 4096, N = 2048 64 rows 12.4 and 15.6, 96 rows 22.3 and 15.6; N = 1024 128 rows 12.1 and 15.5, 192 rows 19.4 and
// 15.5; N = 512 256 rows 12.0 and 15.4, 512 rows 19.4 and 15.5.  K = 8192, N = 1024 128 rows 18.7 and 27.7, 192 rows 32.4 and 27.6; N = 128
// 513 rows 17.5 and 27.4, 1024 rows 17.9 and 27.5, 1200 rows 30.1 and 27.6.  K = 2048, N = 4096 16 rows 7.9 and 14.0, 32 rows 9.5 and 9.6;
// N = 256 256 rows 8.5 and 9.3.  K = 1024, N = 1024 32 rows 5.4 and 6.1, 48 rows 6.6 and 6.1; N = 512 64 rows 6.0 and 5.7.  K = 512, N = 4096
// 16 rows 5.3 and 5.5, 32 rows 6.5 and 5.4.  Fewer than eight terms fill no 16 bytes: the convolution's paths for few channels add a residual
// in a step of its own.  Its fp32 sums stay in one accumulator (see above).
//
// Up to 16 rows, 16-bit, us here and there.  K = 4096: 8 rows N = 8192 18.2 and 30.2, 16 rows N = 6144 14.9 and 17.1, 8192 20.4 and 18.6 (b's
// columns together 20.6 and 17.9; with GELU 20.4 and 20.9, 20.9 and 20.2), 12288 28.6 and 31.3, 14336 31.9 and 32.4 (36.0 and 31.2): from 16 rows
// on the convolution takes a round of 74 tiles of 128 columns, full or not, in about 17 us.  K = 512, N = 18944 8 rows 8.5 and 8.8, N = 24576
// 4 rows 11.0 and 10.8, 8 rows 12.2 and 10.7, 16 rows 14.7 and 10.6 (K = 1024: 8 rows 18.6 and 21.2, 16 rows 20.9 and 20.2): more blocks than run
// at once, of few steps each.  (Left as it is: K = 256, N = 8192 16 rows 6.0 and 5.0.)
bool mm_rows_preferred(int dtype, const MmRowsParams& p) {
  if (p.K < 8 || dtype == FDNN_F32) return true;
  if (p.M > 16) return p.M <= (p.K < 4096 ? 512 : 1024) && (long long)p.M * p.N <= (p.K < 4096 ? 32ll * p.K : 131072);
  // (operands that are not copied 16 bytes at a time are laid out anew for the convolution; rows of y off 16 bytes cost it 1 to 4 us)
  auto whole = [](long long along, long long across, int extent) { return along == 1 && across % 8 == 0 && extent % 8 == 0; };
  if (p.N % 8 != 0 || !whole(p.a_s[1], p.a_s[0], p.K) || !(whole(p.b_s[0], p.b_s[1], p.K) || whole(p.b_s[1], p.b_s[0], p.N))) return true;
  const long long sms = current_sm_count(), tiles = (p.N + 127ll) / 128, at_once = sms / 2, rounds = (tiles + at_once - 1) / at_once;
  if (p.M == 16 && p.K >= 4096 && p.act <= FDNN_ACT_RELU) return 4 * tiles < 3 * rounds * at_once;
  return !(p.M > 4 && p.K < 1024 && p.N > 128 * sms);
}

cudaError_t launch_mm_rows(int dtype, const MmRowsParams& p, cudaStream_t stream) {
  switch (dtype) {
    case FDNN_F16: return by_layout<__half>(p, stream);
    case FDNN_BF16: return by_layout<__nv_bfloat16>(p, stream);
    default: return by_layout<float>(p, stream);
  }
}

}  // namespace fdnn
