// The gated delta rule over prompts, in chunks of 64 tokens.
//
// With G_i = g_1 + .. + g_i within a chunk (g: logarithms of the decays), S the state before it ([V, K]) and D_ij = e^(G_i - G_j):
//   A_ij = b_i D_ij (k_i . k_j) for j < i                 what token j wrote is answered to key i
//   U    = T (v - e^G S k),   T = (1 + A)^-1 diag(b)      what each token writes
//   y_i  = scale (e^(G_i) S q_i + sum over j <= i of D_ij (q_i . k_j) U_j)
//   S    <- e^(G_64) S + sum over j of e^(G_64 - G_j) U_j k_j^T
// delta_prepare_kernel makes, for all chunks side by side, what does not need S: T, P_ij = scale D_ij (q_i . k_j), the keys and queries as
// 16-bit operands and the factors of each token.  delta_chunks_kernel then walks a head's chunks in order.  A state's rows do
// not meet, so two warps keep 16 of them in registers for the whole prompt, half of the keys' channels each, as the accumulators of their own
// products: with rows as the M side, S, v - S k, U and e^.. U are in turn the accumulators of one product and the A operand of the next.
// Through shared memory go only the halves of S k and of U, to each other, and S and U, to the warps that make y beside them.
//
// Precision.  The tensor cores take 16 bits.  Keys and queries that come as f16 or bf16 are f16 operands exactly: each token's is
// scaled by a power of two to a largest value of 2^14 .. 2^15 (a bf16 value below 2^-29 of that loses bits that fp32 sums do not see).
// Everything made in fp32 (S, T, v - S k, U) goes in as two f16 parts, high and low, 22 bits below the row's largest value, which is
// scaled to 2^14 .. 2^15 as well; so do fp32 inputs.  Products of low parts are left out (2^-22).  For bf16 outputs (2^-8) S q and P U
// take the high parts alone, 11 bits each.  Sums are fp32; decays are differences of sums kept in 48 bits.  A row's values have one scale
// and f16's steps end at 2^-24, so what a token writes is held to 2^-39 of the most that one of its chunk does; decays above one let it grow: up to
// 2^18 within a chunk it keeps its 22 bits, and a chunk with a larger product of decays is NaN.
#include <cuda_fp16.h>

#include "delta_rule.cuh"
#include "mma_sync.cuh"

namespace fdnn {
namespace {

constexpr int kChunk = 64;
constexpr int kChunkKeys = 128;      // the widest key that the chunks' kernels take
constexpr int kMostSegments = 32;    // that a row is cut into
constexpr float kMostGrowth = 18.0f; // log2 of a product of decays within a chunk
constexpr int kFactors = 6 * kChunk; // floats a chunk and head: -a, b, d, t, p, and e^(G_64)
constexpr int kLower = 10 * 512;     // bytes of a part of T or P

// How many 16-bit parts: of keys and queries, of S and P in what only y sees.
template <typename T>
struct Parts {
  static constexpr int kKey = std::is_same<T, float>::value ? 2 : 1;
  static constexpr int kOut = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;
};

// ---- small things --------------------------------------------------------------------------------------------------

// D = A B of f16 operands.
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// Four 8 x 8 matrices of 16-bit values, held as accumulators are, transposed to shared memory: 16-byte rows at each lane's address.
__device__ __forceinline__ void stmatrix_t(uint32_t at, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}
template <int THREADS>
__device__ __forceinline__ void barrier(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory"); }
template <int THREADS>
__device__ __forceinline__ void barrier_arrive(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(THREADS) : "memory"); }

// A power of two that takes `most` to 2^14 .. 2^15 (an exponent that it cannot have is cut).  Beside an infinity nothing else would be left of a
// row, as finite numbers that depend on a later token: its scale is NaN, and so is all that is made of the row.
__device__ __forceinline__ float raise(float most) {
  const int e = 268 - int((__float_as_uint(most) >> 23) & 255u);
  return __uint_as_float(e == 13 ? 0x7fffffffu : uint32_t(min(max(e, 1), 253)) << 23);
}
__device__ __forceinline__ float lower_of(float x, float y) {   // of two scales
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float inverse_of_power(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// Two values as f16 high parts, and what they leave as low parts.
__device__ __forceinline__ uint32_t high(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The largest of m, |x| and |y| (NaN is passed over).
__device__ __forceinline__ float most_of(float m, float x, float y) {
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
// The scales of an accumulator block's two rows (lane / 4, + 8).
template <int TILES>
__device__ __forceinline__ void row_scales(const float (&c)[TILES][4], float& lower, float& upper) {
  float m[2][2] = {};
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    m[0][i & 1] = most_of(m[0][i & 1], c[i][0], c[i][1]);
    m[1][i & 1] = most_of(m[1][i & 1], c[i][2], c[i][3]);
  }
  lower = raise(quad_max(fmaxf(m[0][0], m[0][1])));
  upper = raise(quad_max(fmaxf(m[1][0], m[1][1])));
}
// The two rows of an accumulator tile, as pairs.
__device__ __forceinline__ F2 first_row(const float (&c)[4]) { return f2_pack(c[0], c[1]); }
__device__ __forceinline__ F2 second_row(const float (&c)[4]) { return f2_pack(c[2], c[3]); }
__device__ __forceinline__ void set_rows(float (&c)[4], F2 first, F2 second) {
  f2_split(first, c[0], c[1]);
  f2_split(second, c[2], c[3]);
}
__device__ __forceinline__ uint32_t high(F2 v) {
  float x, y;
  f2_split(v, x, y);
  return high(x, y);
}
__device__ __forceinline__ uint32_t low(F2 v, uint32_t hi) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return high(f2_fma(f2_pack(h.x, h.y), f2_both(-1.0f), v));
}
// Accumulator tiles 2 s and 2 s + 1, their rows scaled, as the A operand of k-step s: high parts, and low ones.
__device__ __forceinline__ void operand(const float (&x)[4], const float (&y)[4], F2 s0, F2 s1, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  const F2 v[4] = {f2_mul(first_row(x), s0), f2_mul(second_row(x), s1), f2_mul(first_row(y), s0), f2_mul(second_row(y), s1)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi[i] = high(v[i]);
    lo[i] = low(v[i], hi[i]);
  }
}
__device__ __forceinline__ void operand(const float (&x)[4], const float (&y)[4], F2 s0, F2 s1, uint32_t (&hi)[4]) {
  hi[0] = high(f2_mul(first_row(x), s0));
  hi[1] = high(f2_mul(second_row(x), s1));
  hi[2] = high(f2_mul(first_row(y), s0));
  hi[3] = high(f2_mul(second_row(y), s1));
}

// 16-bit operands lie in blocks of 16 x 16 values, a block as its four 8 x 8 matrices (upper left, upper right, lower left, lower
// right) of eight 16-byte rows: what one ldmatrix reads is 512 bytes in a run, in no bank twice.  Byte offset of 16 bytes of a tile whose
// rows have `blocks` blocks: `at` counts 8 columns.
constexpr int kBlock = 512;
__host__ __device__ constexpr int piece(int row, int at, int blocks) {
  return ((row >> 4) * blocks + (at >> 1)) * kBlock + (((row >> 3) & 1) * 2 + (at & 1)) * 128 + (row & 7) * 16;
}
// Of a lower triangular 64 x 64 tile only the blocks (i, j <= i) are there.
__host__ __device__ constexpr int lower_block(int i, int j) { return i * (i + 1) / 2 + j; }

// ---- where things lie in the workspace -----------------------------------------------------------------------------

template <typename T, int KEYS>
struct Work {
  static constexpr int kKeyBytes = Parts<T>::kKey * kChunk * KEYS * 2;   // keys, and as many for the queries
  static constexpr int kHeadBytes = (2 + Parts<T>::kOut) * kLower + kFactors * 4;
  static constexpr int kStage = 2 * kKeyBytes + kHeadBytes;
};
struct Layout {
  int chunks;
  uint8_t *keys, *heads;   // [N, G, chunks] of kKeyBytes * 2, [N, H, chunks] of kHeadBytes
};
template <typename T, int KEYS>
__host__ __device__ inline Layout layout_of(const DeltaParams& p) {
  Layout w;
  w.chunks = (p.L + kChunk - 1) / kChunk;
  w.keys = static_cast<uint8_t*>(p.workspace);
  w.heads = w.keys + (long long)p.N * p.G * w.chunks * (2 * Work<T, KEYS>::kKeyBytes);
  return w;
}
template <typename T, int KEYS>
long long bytes_of(const DeltaParams& p) {
  const long long chunks = ((long long)p.L + kChunk - 1) / kChunk;
  return (long long)p.N * chunks * ((long long)p.G * 2 * Work<T, KEYS>::kKeyBytes + (long long)p.H * Work<T, KEYS>::kHeadBytes);
}
__device__ __forceinline__ int row_end(const DeltaParams& p, long long n) {
  return p.lengths != nullptr ? min(max(p.lengths[n], 0), p.L) : p.L;
}

// ---- what does not need the state ----------------------------------------------------------------------------------

// Eight warps to a chunk of a key head: four make a and solve it, four make P meanwhile.
constexpr int kPrepThreads = 256, kSolvers = 128, kSolveId = 1;
constexpr int kPitch = kChunk + 4;   // floats between rows of A, T

struct alignas(16) HeadGates {   // (pairs of each are read at once)
  float hi[kChunk], lo[kChunk], beta[kChunk];   // sums of log2 decays in two parts
  float whole;                                  // 1, or NaN where a product of decays is past kMostGrowth
};
template <typename T, int KEYS>
struct PrepShared {
  union {
    uint8_t keys[2 * Work<T, KEYS>::kKeyBytes];   // and the queries
    struct {
      float a[kChunk][kPitch], t[kChunk][kPitch], part[4][16][20];
    } solve;
  };
  float key_scale[kChunk], query_scale[kChunk];
  HeadGates gates[4];
};

// Keys or queries of a chunk, on their way to shared memory.  A warp takes 8 rows, four lanes a row, so that what they write is 128 bytes
// in a run.  All loads of a chunk are on their way before the first is waited for.
template <typename T, int KEYS, bool WHOLE>
struct Rows {
  static constexpr int kPieces = KEYS / 32, kV = WHOLE ? 16 / int(sizeof(T)) : 1;   // pieces of eight channels, to a lane
  Pack<T, kV> raw[kPieces][8 / kV];
  static __device__ __forceinline__ int row() { return (threadIdx.x >> 5) * 8 + (threadIdx.x & 7); }
  static __device__ __forceinline__ int channel(int n) { return (n * 4 + ((threadIdx.x & 31) >> 3)) * 8; }
  __device__ __forceinline__ void load(const T* x, const long long* s, int tokens, int K) {
#pragma unroll
    for (int n = 0; n < kPieces; ++n)
#pragma unroll
      for (int i = 0; i < 8 / kV; ++i) {
        const int at = channel(n) + i * kV;
        raw[n][i].clear();
        if (row() < tokens && at < K) raw[n][i].load(x + row() * s[1] + (WHOLE ? (long long)at : at * s[3]));
      }
  }
  // To their places, as parts, scaled; the factors that take the operands back (with the norm, if asked, and `scale`).
  __device__ __forceinline__ void stage(uint8_t* to, float* factor, int tokens, bool norm, float scale) const {
    float most = 0.0f, squares = 0.0f;
#pragma unroll
    for (int n = 0; n < kPieces; ++n)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = raw[n][j / kV].at(j % kV);
        most = fmaxf(most, fabsf(v));
        squares += v * v;
      }
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) {
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      squares += __shfl_xor_sync(0xffffffffu, squares, o);
    }
    const float up = raise(most);
    const int r = row();
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      uint4 hi, lo;
      uint32_t* h = reinterpret_cast<uint32_t*>(&hi);
      uint32_t* l = reinterpret_cast<uint32_t*>(&lo);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const F2 x = f2_mul(f2_pack(raw[n][2 * j / kV].at(2 * j % kV), raw[n][(2 * j + 1) / kV].at((2 * j + 1) % kV)), f2_both(up));
        h[j] = high(x);
        if constexpr (Parts<T>::kKey == 2) l[j] = low(x, h[j]);
      }
      const int at = piece(r, channel(n) / 8, KEYS / 16);
      *reinterpret_cast<uint4*>(to + at) = hi;
      if constexpr (Parts<T>::kKey == 2) *reinterpret_cast<uint4*>(to + kChunk * KEYS * 2 + at) = lo;
    }
    if ((threadIdx.x & 31) < 8) factor[r] = r < tokens ? scale * inverse_of_power(up) * (norm ? 1.0f / sqrtf(squares + kKeyEps) : 1.0f) : 0.0f;
  }
};

// c += the products of row block `i` of `x` with the row blocks up to it of `y`, over KEYS channels.
template <typename T, int KEYS>
__device__ __forceinline__ void dots(float (&c)[8][4], const uint8_t* x, const uint8_t* y, int i) {
  const int lane = threadIdx.x & 31, m = lane >> 3, r = lane & 7;
  const uint32_t xs = smem_u32(x) + i * (KEYS / 16) * kBlock + ((m & 1) * 2 + (m >> 1)) * 128 + r * 16, ys = smem_u32(y) + lane * 16;
  constexpr int kPart = kChunk * KEYS * 2;
#pragma unroll
  for (int s = 0; s < KEYS / 16; ++s) {
    uint32_t a[Parts<T>::kKey][4];
#pragma unroll
    for (int k = 0; k < Parts<T>::kKey; ++k) ldmatrix<false>(a[k], xs + k * kPart + s * kBlock);
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (n <= i) {
        uint32_t b[Parts<T>::kKey][4];
#pragma unroll
        for (int k = 0; k < Parts<T>::kKey; ++k) ldmatrix<false>(b[k], ys + k * kPart + (n * (KEYS / 16) + s) * kBlock);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mma<__half>(c[2 * n + j], a[0], b[0][2 * j], b[0][2 * j + 1]);
          if constexpr (Parts<T>::kKey == 2) {
            mma<__half>(c[2 * n + j], a[0], b[1][2 * j], b[1][2 * j + 1]);
            mma<__half>(c[2 * n + j], a[1], b[0][2 * j], b[0][2 * j + 1]);
          }
        }
      }
  }
}

// Sums of a head's log2 decays and its step sizes, by one warp, two tokens a lane.
struct RawGates {
  float delta[2], beta[2], A, bias;
};
template <typename T>
__device__ __forceinline__ void load_gates(const DeltaParams& p, RawGates& x, long long n, int begin, int tokens, int h) {
  x.A = p.A != nullptr ? p.A[h] : 1.0f;
  x.bias = p.delta_bias != nullptr ? p.delta_bias[h] : 0.0f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = 2 * (threadIdx.x & 31) + j;
    x.delta[j] = x.beta[j] = 0.0f;
    if (i < tokens) {
      x.delta[j] = gate_at<T>(p, p.delta, n * p.delta_s[0] + (begin + i) * p.delta_s[1] + h * p.delta_s[2]);
      x.beta[j] = gate_at<T>(p, p.beta, n * p.beta_s[0] + (begin + i) * p.beta_s[1] + h * p.beta_s[2]);
    }
  }
}
__device__ __forceinline__ void sum_gates(const DeltaParams& p, const RawGates& x, HeadGates& to, int tokens) {
  const int lane = threadIdx.x & 31;
  double v[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = 2 * lane + j;
    float g = log_decay(p, x.delta[j], x.bias, x.A);
    g = i < tokens ? (g < -1e5f ? -1e5f : g) : 0.0f;   // a decay of zero, whose difference to itself is a number; NaN stays
    v[j] = double(g) * 1.4426950408889634;
    to.beta[i] = i < tokens ? step_size(p, x.beta[j]) : 0.0f;
  }
  double sum = v[0] + v[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += other;
  }
  const double each[2] = {sum - v[1], sum};
  // how far a later sum is above an earlier one
  const float first = float(each[0]), second = float(each[1]);
  float most = fmaxf(first, second);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) most = fmaxf(most, __shfl_down_sync(0xffffffffu, most, o));   // (the last lanes' own again)
  const float later = fmaxf(second, __shfl_down_sync(0xffffffffu, most, 1)), behind = lane < 31 ? later : second;
  const bool grown = __any_sync(0xffffffffu, fmaxf(behind - first, behind - second) > kMostGrowth);
  if (lane == 0) to.whole = grown ? __uint_as_float(0x7fffffffu) : 1.0f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float hi = float(each[j]);
    to.hi[2 * lane + j] = hi;
    to.lo[2 * lane + j] = float(each[j] - double(hi));
  }
}
// 2^d to fp32's last place but two: what a state keeps over many chunks has no drift.  (What fp32 leaves of a d whose power is not zero is
// at most 2^-17.  The parts of a sum that has passed a token which forgets all are not: of 32 such tokens, 0.25.)
__device__ __forceinline__ float exp2_of(double d) {
  const float hi = float(d);
  return exp2f(hi) * fmaf(float(d - double(hi)), 0.6931471805599453f, 1.0f);
}

// d += x y of 16 x 16 blocks in fp32, by 3 x TF32 (2^-22).
__device__ __forceinline__ void block_product(float (&d)[2][4], const float* x, int x_pitch, const float* y, int y_pitch) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    uint32_t a[4], al[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      two_parts(x[(g + (i & 1) * 8) * x_pitch + s * 8 + t + (i >> 1) * 4], a[i], al[i]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      uint32_t b[2], bl[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) two_parts(y[(s * 8 + t + i * 4) * y_pitch + n * 8 + g], b[i], bl[i]);
      mma<float>(d[n], a, bl[0], bl[1]);
      mma<float>(d[n], al, b[0], b[1]);
      mma<float>(d[n], a, b[0], b[1]);
    }
  }
}
__device__ __forceinline__ void put_block(float* to, int pitch, const float (&d)[2][4], float sign) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) to[(g + (i >> 1) * 8) * pitch + n * 8 + 2 * t + (i & 1)] = sign * d[n][i];
}

// t = (1 + a)^-1 for a strictly lower triangular, 64 x 64: diagonal blocks of 16 by substitution, then blocks of 32 and 64 from
// [[X, 0], [-Y a X, Y]].  Called by four warps.
__device__ __forceinline__ void invert(const float (&a)[kChunk][kPitch], float (&t)[kChunk][kPitch], float (&part)[4][16][20]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  {
    const int at = warp * 16, c = lane & 15;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == c ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) v -= a[at + i][at + j] * x[j];
      x[i] = v;
    }
    if (lane < 16) {
#pragma unroll
      for (int i = 0; i < 16; ++i) t[at + i][at + c] = x[i];
    }
  }
  barrier<kSolvers>(kSolveId);
  if (warp < 2) {   // blocks (1, 0) and (3, 2)
    const int i = warp * 32 + 16, j = warp * 32;
    float d[2][4] = {};
    block_product(d, &a[i][j], kPitch, &t[j][j], kPitch);
    put_block(&part[warp][0][0], 20, d, 1.0f);
    __syncwarp();
    float e[2][4] = {};
    block_product(e, &t[i][i], kPitch, &part[warp][0][0], 20);
    put_block(&t[i][j], kPitch, e, -1.0f);
  }
  barrier<kSolvers>(kSolveId);
  {   // the lower left 32 x 32: part = a t, then t part
    const int i = 32 + (warp >> 1) * 16, j = (warp & 1) * 16;
    float d[2][4] = {};
    for (int m = j; m < 32; m += 16) block_product(d, &a[i][m], kPitch, &t[m][j], kPitch);
    put_block(&part[warp][0][0], 20, d, 1.0f);
    barrier<kSolvers>(kSolveId);
    float e[2][4] = {};
    for (int m = 32; m <= i; m += 16) block_product(e, &t[i][m], kPitch, &part[(m - 32) / 16 * 2 + (warp & 1)][0][0], 20);
    put_block(&t[i][j], kPitch, e, -1.0f);
  }
  barrier<kSolvers>(kSolveId);
}

template <typename T, int KEYS, bool WHOLE>
__global__ void __launch_bounds__(kPrepThreads, 2)
delta_prepare_kernel(const DeltaParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  PrepShared<T, KEYS>& s = *reinterpret_cast<PrepShared<T, KEYS>*>(smem_raw);
  chained();
  using W = Work<T, KEYS>;
  const Layout w = layout_of<T, KEYS>(p);
  const int g = int(blockIdx.x % p.G), c = int(blockIdx.x / p.G % w.chunks);   // (heads of a token lie together)
  const long long n = blockIdx.x / p.G / w.chunks;
  const int begin = c * kChunk, tokens = min(row_end(p, n) - begin, kChunk);
  if (tokens <= 0) return;
  const int tid = threadIdx.x, lane = tid & 31, q = lane >> 2, t = lane & 3;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0), block = warp & 3;   // of 16 tokens
  const bool solver = warp < 4;
  uint8_t* const queries = s.keys + W::kKeyBytes;
  const int group = p.H / p.G, h0 = g * group;
  {
    RawGates gates;
    if (warp < 4 && warp < group) load_gates<T>(p, gates, n, begin, tokens, h0 + warp);
    Rows<T, KEYS, WHOLE> rows, more;
    rows.load(static_cast<const T*>(p.k) + n * p.k_s[0] + begin * p.k_s[1] + g * p.k_s[2], p.k_s, tokens, p.K);
    more.load(static_cast<const T*>(p.q) + n * p.q_s[0] + begin * p.q_s[1] + g * p.q_s[2], p.q_s, tokens, p.K);
    if (warp < 4 && warp < group) sum_gates(p, gates, s.gates[warp], tokens);
    rows.stage(s.keys, s.key_scale, tokens, p.norm, 1.0f);
    more.stage(queries, s.query_scale, tokens, p.norm, p.scale);
  }
  fence_proxy_async_smem();
  __syncthreads();
  if (tid == 0) {
    bulk_store_1d(w.keys + ((n * p.G + g) * w.chunks + c) * (2ll * W::kKeyBytes), s.keys, 2 * W::kKeyBytes);
    bulk_commit_group();
  }
  float dot[8][4] = {};   // k_i . k_j of these 16 tokens, or q_i . k_j
  dots<T, KEYS>(dot, solver ? s.keys : queries, s.keys, block);
  const int r0 = block * 16 + q;
  {   // the factors of the rows and columns
    const float* of_row = solver ? s.key_scale : s.query_scale;
    const float f0 = of_row[r0], f1 = of_row[r0 + 8];
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const float2 f = *reinterpret_cast<const float2*>(&s.key_scale[m * 8 + 2 * t]);
      dot[m][0] *= f0 * f.x, dot[m][1] *= f0 * f.y, dot[m][2] *= f1 * f.x, dot[m][3] *= f1 * f.y;
    }
  }
  if (tid == 0) bulk_wait_group_read0();
  __syncthreads();   // the operands' place is taken by a and t

  for (int i = 0; i < group; ++i) {
    if (i > 0 && (i & 3) == 0) {
      __syncthreads();
      if (warp < 4 && i + warp < group) {
        RawGates raw;
        load_gates<T>(p, raw, n, begin, tokens, h0 + i + warp);
        sum_gates(p, raw, s.gates[warp], tokens);
      }
      __syncthreads();
    }
    const HeadGates& gates = s.gates[i & 3];
    uint8_t* out = w.heads + ((n * p.H + h0 + i) * w.chunks + c) * (long long)W::kHeadBytes;
    float* factors = reinterpret_cast<float*>(out + (2 + Parts<T>::kOut) * kLower);
    // a or P, of this warp's 16 tokens
    float hi[2], lo[2], beta[2], most[2] = {0.0f, 0.0f}, v[8][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      hi[j] = gates.hi[r0 + 8 * j];
      lo[j] = gates.lo[r0 + 8 * j];
      beta[j] = solver ? gates.beta[r0 + 8 * j] : 1.0f;
    }
#pragma unroll
    for (int m = 0; m < 8; ++m)
      if (m < 2 * (block + 1)) {
        const int col = m * 8 + 2 * t;
        const float2 chi = *reinterpret_cast<const float2*>(&gates.hi[col]), clo = *reinterpret_cast<const float2*>(&gates.lo[col]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = r0 + (j >> 1) * 8, at = col + (j & 1);
          const float d = ex2((hi[j >> 1] - ((j & 1) ? chi.y : chi.x)) + (lo[j >> 1] - ((j & 1) ? clo.y : clo.x)));
          v[m][j] = at < row || (at == row && !solver) ? dot[m][j] * (beta[j >> 1] * d) : 0.0f;
          most[j >> 1] = fmaxf(most[j >> 1], fabsf(v[m][j]));
        }
        if (solver) {
          *reinterpret_cast<float2*>(&s.solve.a[r0][col]) = make_float2(v[m][0], v[m][1]);
          *reinterpret_cast<float2*>(&s.solve.a[r0 + 8][col]) = make_float2(v[m][2], v[m][3]);
        }
      }
    if (solver) {
      barrier<kSolvers>(kSolveId);
      invert(s.solve.a, s.solve.t, s.solve.part);
      most[0] = most[1] = 0.0f;   // T = t diag(beta)
#pragma unroll
      for (int m = 0; m < 8; ++m)
        if (m < 2 * (block + 1)) {
          const int col = m * 8 + 2 * t;
          const float2 b = *reinterpret_cast<const float2*>(&gates.beta[col]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 x = *reinterpret_cast<const float2*>(&s.solve.t[r0 + 8 * j][col]);
            v[m][2 * j] = x.x * b.x;
            v[m][2 * j + 1] = x.y * b.y;
            most[j] = fmaxf(most[j], fmaxf(fabsf(v[m][2 * j]), fabsf(v[m][2 * j + 1])));
          }
        }
    } else if (tid - kSolvers < kChunk) {
      const int at = tid - kSolvers;
      const double sum = double(gates.hi[at]) + double(gates.lo[at]), all = double(gates.hi[kChunk - 1]) + double(gates.lo[kChunk - 1]);
      const float since = exp2_of(sum) * gates.whole;
      factors[at] = -since * s.key_scale[at];
      factors[kChunk + at] = since * s.query_scale[at];
      factors[2 * kChunk + at] = exp2_of(all - sum) * s.key_scale[at];
      if (at == kChunk - 1) factors[5 * kChunk] = since;
    }
    uint8_t* const parts = out + (solver ? 0 : 2 * kLower);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float up = raise(quad_max(most[j]));
      if (t == 0) factors[(solver ? 3 : 4) * kChunk + r0 + 8 * j] = inverse_of_power(up);
#pragma unroll
      for (int m = 0; m < 8; ++m)
        if (m < 2 * (block + 1)) {
          const F2 x = f2_mul(f2_pack(v[m][2 * j], v[m][2 * j + 1]), f2_both(up));
          const uint32_t h16 = high(x);
          uint8_t* at = parts + lower_block(block, m >> 1) * kBlock + (j * 2 + (m & 1)) * 128 + lane * 4;
          *reinterpret_cast<uint32_t*>(at) = h16;
          if (Parts<T>::kOut == 2 || solver) *reinterpret_cast<uint32_t*>(at + kLower) = low(x, h16);
        }
    }
    if (solver) barrier<kSolvers>(kSolveId);   // (t is read before the next head's a is solved)
  }
  if (tid == 0) bulk_wait_group0();
}

// ---- the chunks in order -------------------------------------------------------------------------------------------

// A block has SLICES slices of 16 rows of the state or fewer. Each has two warps that carry the state on and OUTS that make y.  Two slices
// with two of them leave each quarter of an SM one warp of either kind; four with one fill it.
constexpr int kMostSlices = 4, kMostStages = 3;
__host__ __device__ constexpr int outs_of(int slices) { return slices <= 2 ? 2 : 1; }
// What the warps of a slice leave for each other: S k of either half (8 tiles of 512 bytes each), S as operands (each half's, the high parts,
// then the low ones), U (8 tiles in fp32), the scales of the operands; and y on its way out.
template <typename T, int KEYS>
struct Exchange {
  static constexpr int kState = 2 * 8 * 512, kStatePart = KEYS / 32 * 512, kStateHalf = Parts<T>::kOut * kStatePart;
  static constexpr int kWritten = kState + 2 * kStateHalf, kScales = kWritten + 8 * 512, kStage = kScales + 2 * 32 * 8,
                       kBytes = kStage + (sizeof(T) == 2 ? 2048 : 0);
};

template <typename T>
__host__ __device__ constexpr int value_pitch(int slices) { return 16 * slices * int(sizeof(T)) + 16; }   // bytes; eight rows in different banks

__device__ __forceinline__ F2 pair_at(const float* p) { return *reinterpret_cast<const F2*>(p); }

// Outputs of BLOCKS x 16 tokens: o[i][..] holds rows (value channels) lane / 4, + 8 and tokens 8 i + 2 (lane % 4), + 1; `y` is at the first
// token.  16-bit ones go through `stage` (32 bytes a token) to 16-byte stores.
template <typename T, bool WHOLE, int BLOCKS>
__device__ __forceinline__ void put_outputs(const DeltaParams& p, T* y, const float (&o)[2 * BLOCKS][4], uint8_t* stage, int tokens, int channels) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if constexpr (sizeof(T) == 2) {
    const uint32_t to = smem_u32(stage) + (lane >> 4) * 256 + (lane & 7) * 32 + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)   // channels 0 .. 7 and 8 .. 15 of eight tokens, then of the next eight
      stmatrix_t(to + i * 512, pack2(from_f32<T>(o[2 * i][0]), from_f32<T>(o[2 * i][1])), pack2(from_f32<T>(o[2 * i][2]), from_f32<T>(o[2 * i][3])),
                 pack2(from_f32<T>(o[2 * i + 1][0]), from_f32<T>(o[2 * i + 1][1])), pack2(from_f32<T>(o[2 * i + 1][2]), from_f32<T>(o[2 * i + 1][3])));
    __syncwarp();
    if constexpr (WHOLE) {   // eight channels are whole, and 16 bytes
      const int token = lane >> 1, channel = (lane & 1) * 8;
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i) {
        const uint4 v = *reinterpret_cast<const uint4*>(stage + i * 512 + lane * 16);
        if (i * 16 + token < tokens && channel < channels) *reinterpret_cast<uint4*>(y + (i * 16 + token) * p.y_s[1] + channel) = v;
      }
    } else {
      const int channel = lane & 15;
      for (int token = lane >> 4; token < min(BLOCKS * 16, tokens); token += 2)
        if (channel < channels) y[token * p.y_s[1] + channel * p.y_s[3]] = reinterpret_cast<const T*>(stage)[token * 16 + channel];
    }
    __syncwarp();
  } else {
#pragma unroll
    for (int n = 0; n < 2 * BLOCKS; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int token = n * 8 + 2 * t + (i & 1), channel = g + (i >> 1) * 8;
        if (token < tokens && channel < channels) y[token * p.y_s[1] + channel * p.y_s[3]] = from_f32<T>(o[n][i]);
      }
  }
}

// d (+)= a b for the column tiles from FROM on, whose operands are b[tile / 2][2 (tile % 2)] and the next.
template <int TILES, int FROM = 0, int PAIRS>
__device__ __forceinline__ void mma_row(float (&d)[TILES][4], const uint32_t (&a)[4], const uint32_t (&b)[PAIRS][4], bool first = false) {
#pragma unroll
  for (int j = FROM; j < TILES; ++j) {
    if (first) mma_first(d[j], a, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
    else mma<__half>(d[j], a, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
  }
}

// A launch over the chunks.  Where few rows and heads leave SMs idle, a row is cut into segments of `per` chunks, which run side by side: first
// for their `ends` alone, from nothing, with the K rows of a unit matrix as further rows (the end of a segment is its start times their end
// plus the end from nothing: delta_join_kernel), then from their `starts`.
struct Run {
  int blocks_a_head, stages, per, segments;
  const float* starts;   // [N, H, segments - 1, V, K]: of all but the first
  float* ends;           // null, or [N, H, segments - 1, V rounded up to 16 + K, K]: of all but the last
  uint32_t* status;
  long long wait_limit;
  int skip_copies;       // a test of the bounded waits
};

// WHOLE: 16 bytes of neighbouring value channels are copied and stored at once.
template <typename T, int KEYS, int SLICES, bool WHOLE>
__global__ void __launch_bounds__((2 + outs_of(SLICES)) * SLICES * 32, 1)
delta_chunks_kernel(const DeltaParams p, const Run run) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ uint64_t full[kMostStages], empty[kMostStages];   // a stage's operands have landed; all warps are done with them
  __shared__ uint32_t abort_word;
  using W = Work<T, KEYS>;
  using E = Exchange<T, KEYS>;
  constexpr int kKeyPart = kChunk * KEYS * 2, kHalf = KEYS / 2, kSteps = KEYS / 16, kOuts = outs_of(SLICES), kShare = 64 + 32 * kOuts;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMostStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], blockDim.x / 32);
    }
    abort_word = 0;
    fence_barrier_init();
  }
  __syncthreads();
  chained();
  const Layout w = layout_of<T, KEYS>(p);
  const int lane = threadIdx.x & 31, slices = blockDim.x / kShare;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int stages = run.stages, made = run.ends != nullptr ? run.segments - 1 : run.segments;
  const int segment = int(blockIdx.x / run.blocks_a_head % made), h = int(blockIdx.x / run.blocks_a_head / made % p.H);
  const long long n = blockIdx.x / run.blocks_a_head / made / p.H;
  // the segment's tokens begin at `begin`, and are `end` (of the row's, which may be fewer)
  const int begin = int(min((long long)segment * run.per * kChunk, (long long)p.L)), row_tokens = row_end(p, n);
  const int end = max(0, min(row_tokens - begin, run.per * kChunk)), chunks = (end + kChunk - 1) / kChunk;
  const int chunk0 = segment * run.per;
  const int pitch = value_pitch<T>(slices), stage_bytes = W::kStage + kChunk * pitch;
  const uint32_t smem = smem_u32(smem_raw);
  const int g = lane >> 2, t = lane & 3, m = lane >> 3, r = lane & 7;
  const bool outputs = warp >= 2 * slices;
  const int slice = outputs ? (warp - 2 * slices) / kOuts : warp >> 1, half = warp & 1;
  // 16 rows: value channels, or behind them (where the segments' ends are made) the rows of what the segment makes of a state, a unit's
  // each, which meet no values
  const int number = int(blockIdx.x % run.blocks_a_head) * slices + slice, value_slices = (p.V + 15) / 16;
  const bool transition = run.ends != nullptr && number >= value_slices;
  const int row0 = (transition ? number - value_slices : number) * 16, rows = min(16, (transition ? p.K : p.V) - row0);
  const int channels = transition ? 0 : rows;
  uint8_t* const exchange = smem_raw + stages * stage_bytes + slice * E::kBytes;
  // named barriers of the slice's own: slices run at their own pace, `stages` chunks apart at most
  const int top_id = slice, pair_id = kMostSlices + slice, state_id = 2 * kMostSlices + slice, written_id = 3 * kMostSlices + slice;
  // The slice's warps, at the top of chunk c: it is there, and they are done with chunk c - 1.
  auto arrive_at = [&](int c) {
    barrier<kShare>(top_id);
    mbar_wait_warp(&full[c % stages], uint32_t(c / stages) & 1u, &abort_word, run.status, kIncidentDeltaWait, run.wait_limit);
  };
  auto leave = [&](int c) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[c % stages]);
  };

  if (outputs) {
    // ---- y, and the copies, stages - 1 chunks ahead: the first of these warps asks for the operands of all, each for its slice's values
    const int tid = kOuts == 2 ? threadIdx.x & 63 : lane;
    constexpr int kStep = 32 * kOuts;
    const bool loader = threadIdx.x == 2u * slices * 32;
    const uint8_t* keys_from = w.keys + ((n * p.G + h / (p.H / p.G)) * w.chunks + chunk0) * (2ll * W::kKeyBytes);
    const uint8_t* heads_from = w.heads + ((n * p.H + h) * w.chunks + chunk0) * (long long)W::kHeadBytes;
    const T* v0 = static_cast<const T*>(p.v) + n * p.v_s[0] + begin * p.v_s[1] + h * p.v_s[2] + row0 * p.v_s[3];
    int asked = 0;   // chunks, by the loader
    auto ask = [&](int c) {
      uint8_t* const to = smem_raw + (c % stages) * stage_bytes;
      if (loader && asked == c && !run.skip_copies) {
        uint64_t* bar = &full[c % stages];
        if (c < stages || mbar_wait_bounded(&empty[c % stages], uint32_t(c / stages - 1) & 1u, &abort_word, run.status, kIncidentDeltaWait, run.wait_limit)) {
          mbar_arrive_expect_tx(bar, W::kStage);
          bulk_load_1d(to, keys_from + c * (2ll * W::kKeyBytes), 2 * W::kKeyBytes, bar);
          bulk_load_1d(to + 2 * W::kKeyBytes, heads_from + c * (long long)W::kHeadBytes, W::kHeadBytes, bar);
          ++asked;
        }
      }
      __syncwarp();
      const int tokens = min(end - c * kChunk, kChunk);
      uint8_t* const values = to + W::kStage + slice * 16 * int(sizeof(T));
      if constexpr (WHOLE) {
        constexpr int kV = 16 / sizeof(T), kPieces = 16 / kV;
        const int at = tid % kPieces * kV, bytes = at < channels ? 16 : 0;
        const uint32_t first_row = smem_u32(values) + at * int(sizeof(T));
#pragma unroll 4
        for (int i = tid / kPieces; i < kChunk; i += kStep / kPieces) {
          const bool there = i < tokens && bytes > 0;
          copy16(first_row + i * pitch, there ? v0 + ((long long)c * kChunk + i) * p.v_s[1] + at : static_cast<const T*>(p.v), there ? bytes : 0);
        }
      } else {
        for (int i = tid; i < kChunk * 16; i += kStep) {
          const int row = i / 16, at = i % 16;
          reinterpret_cast<T*>(values + row * pitch)[at] =
              row < tokens && at < channels ? v0[((long long)c * kChunk + row) * p.v_s[1] + at * p.v_s[3]] : from_f32<T>(0.0f);
        }
      }
      async_commit();
    };
    T* const y_row = static_cast<T*>(p.y) + n * p.y_s[0] + h * p.y_s[2] + row0 * p.y_s[3];
    T* const y = y_row + begin * p.y_s[1];
    for (int c = 0; c < stages - 1; ++c) {
      if (c < chunks) ask(c);
      else async_commit();
    }
    for (int c = 0; c < chunks; ++c) {
      if (stages == 3) async_wait<1>();   // (a thread's groups: one a chunk, empty ones behind the last)
      else async_wait<0>();
      arrive_at(c);
      if (c + stages - 1 < chunks) ask(c + stages - 1);
      else async_commit();
      if (run.ends != nullptr) {   // (the state alone)
        barrier<kShare>(state_id);
        barrier<kShare>(written_id);
        leave(c);
        continue;
      }
      const uint8_t* const base = smem_raw + (c % stages) * stage_bytes;
      // this warp's tokens: all of the chunk's, or its first or last 32
      constexpr int kTiles = 8 / kOuts;
      const int tile0 = kOuts == 2 ? (warp & 1) * kTiles : 0;
      const uint32_t queries = smem_u32(base) + W::kKeyBytes + tile0 / 2 * kSteps * kBlock + lane * 16;
      const uint32_t weights = smem_u32(base) + 2 * W::kKeyBytes + 2 * kLower + lane * 16;
      const float* factors = reinterpret_cast<const float*>(base + 2 * W::kKeyBytes + (2 + Parts<T>::kOut) * kLower) + tile0 * 8 + 2 * t;
      float o[kTiles][4];
      barrier<kShare>(state_id);
#pragma unroll
      for (int half = 0; half < 2; ++half) {   // S q
        float z[kTiles][4];
        const uint4* from = reinterpret_cast<const uint4*>(exchange + E::kState + half * E::kStateHalf) + lane;
#pragma unroll
        for (int k = 0; k < kSteps / 2; ++k) {
          uint32_t hi[4], lo[4], b[kTiles / 2][4];
          const uint4 f = from[k * 32];
          hi[0] = f.x, hi[1] = f.y, hi[2] = f.z, hi[3] = f.w;
          if constexpr (Parts<T>::kOut == 2) {
            const uint4 l = from[(kSteps / 2 + k) * 32];
            lo[0] = l.x, lo[1] = l.y, lo[2] = l.z, lo[3] = l.w;
          }
#pragma unroll
          for (int j = 0; j < kTiles / 2; ++j) ldmatrix<false>(b[j], queries + (j * kSteps + half * (kSteps / 2) + k) * kBlock);
          mma_row<kTiles>(z, hi, b, k == 0);
          if constexpr (Parts<T>::kOut == 2) mma_row<kTiles>(z, lo, b);
          if constexpr (Parts<T>::kKey == 2) {
#pragma unroll
            for (int j = 0; j < kTiles / 2; ++j) ldmatrix<false>(b[j], queries + kKeyPart + (j * kSteps + half * (kSteps / 2) + k) * kBlock);
            mma_row<kTiles>(z, hi, b);
          }
        }
        const float2 down = reinterpret_cast<const float2*>(exchange + E::kScales)[half * 32 + lane];
        const F2 down0 = f2_both(down.x), down1 = f2_both(down.y);
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          if (half == 0) set_rows(o[j], f2_mul(first_row(z[j]), down0), f2_mul(second_row(z[j]), down1));
          else set_rows(o[j], f2_fma(first_row(z[j]), down0, first_row(o[j])), f2_fma(second_row(z[j]), down1, second_row(o[j])));
        }
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        const F2 b = pair_at(factors + kChunk + j * 8);
        set_rows(o[j], f2_mul(b, first_row(o[j])), f2_mul(b, second_row(o[j])));
      }
      barrier<kShare>(written_id);
      {   // U P^T, a lower triangle of blocks: the blocks on and next to the diagonal, and with the last tokens a square before them
        float u[kTiles][4], v[8 - kTiles + 1][4] = {}, z[kTiles][4] = {}, u0, u1, v0, v1;
        auto load = [&](float (&to)[4], int tile) {
          const float4 f = reinterpret_cast<const float4*>(exchange + E::kWritten)[tile * 32 + lane];
          to[0] = f.x, to[1] = f.y, to[2] = f.z, to[3] = f.w;
        };
#pragma unroll
        for (int j = 0; j < kTiles; ++j) load(u[j], tile0 + j);
        row_scales<kTiles>(u, u0, u1);
        if (tile0 != 0) {
#pragma unroll
          for (int j = 0; j < 8 - kTiles; ++j) load(v[j], j);
          row_scales<8 - kTiles + 1>(v, v0, v1);
          u0 = lower_of(u0, v0);
          u1 = lower_of(u1, v1);
        }
        const F2 up0 = f2_both(u0), up1 = f2_both(u1);
        auto products = [&](const float (&x)[4], const float (&y)[4], int k, auto from) {   // tokens 16 k ..: what they wrote, to blocks from .. on
          constexpr int j0 = decltype(from)::value;
          uint32_t hi[4], lo[4], b[kTiles / 2][4];
          if constexpr (Parts<T>::kOut == 2) operand(x, y, up0, up1, hi, lo);
          else operand(x, y, up0, up1, hi);
#pragma unroll
          for (int j = j0; j < kTiles / 2; ++j) ldmatrix<false>(b[j], weights + lower_block(tile0 / 2 + j, k) * kBlock);
          mma_row<kTiles, 2 * j0>(z, hi, b);
          if constexpr (Parts<T>::kOut == 2) {
            mma_row<kTiles, 2 * j0>(z, lo, b);
#pragma unroll
            for (int j = j0; j < kTiles / 2; ++j) ldmatrix<false>(b[j], weights + kLower + lower_block(tile0 / 2 + j, k) * kBlock);
            mma_row<kTiles, 2 * j0>(z, hi, b);
          }
        };
        products(u[0], u[1], tile0 / 2, std::integral_constant<int, 0>{});
        products(u[2], u[3], tile0 / 2 + 1, std::integral_constant<int, 1>{});
        if constexpr (kOuts == 1) {
          products(u[4], u[5], 2, std::integral_constant<int, 2>{});
          products(u[6], u[7], 3, std::integral_constant<int, 3>{});
        } else if (tile0 != 0) {
          products(v[0], v[1], 0, std::integral_constant<int, 0>{});
          products(v[2], v[3], 1, std::integral_constant<int, 0>{});
        }
        const F2 down0 = f2_both(inverse_of_power(u0)), down1 = f2_both(inverse_of_power(u1));
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          const F2 f = pair_at(factors + 4 * kChunk + j * 8);
          set_rows(o[j], f2_fma(f, f2_mul(first_row(z[j]), down0), first_row(o[j])), f2_fma(f, f2_mul(second_row(z[j]), down1), second_row(o[j])));
        }
      }
      uint8_t* const stage = exchange + E::kStage + tile0 * 256;
      const int token = c * kChunk + tile0 * 8;
      put_outputs<T, WHOLE, kTiles / 2>(p, y + (long long)token * p.y_s[1], o, stage, end - token, channels);
      leave(c);
    }
    // tokens behind the row's end
    if (run.ends == nullptr && segment == run.segments - 1)
      for (long long i = row_tokens * 16ll + (kOuts == 2 ? (warp & 1) * 32 : 0) + lane; i < p.L * 16ll; i += 32 * kOuts)
        if (i % 16 < channels) y_row[i / 16 * p.y_s[1] + i % 16 * p.y_s[3]] = from_f32<T>(0.0f);
    if (loader && *static_cast<volatile uint32_t*>(&abort_word) != 0) {   // after an incident: give the copies in flight time to land
      volatile uint32_t never = 0;
      for (int c = max(0, asked - stages); c < asked; ++c)
        mbar_wait_bounded(&full[c % stages], uint32_t(c / stages) & 1u, &never, run.status, kIncidentDrainWait, kWaitLimitCycles / 16);
    }
    return;
  }

  // ---- two warps hold 16 rows of the state, half of the keys' channels each: s[j] rows lane / 4, + 8, channels 8 j + 2 (lane % 4), + 1
  const long long head = n * p.H + h;
  const float* from = nullptr;   // the state before the first token: zeros, or a unit a row
  float* to = nullptr;
  if (run.ends != nullptr) {
    to = run.ends + ((head * (run.segments - 1) + segment) * (value_slices * 16 + p.K) + (transition ? value_slices * 16 : 0) + row0) * p.K;
  } else {
    if (segment > 0) from = run.starts + ((head * (run.segments - 1) + segment - 1) * p.V + row0) * p.K;
    else if (p.initial != nullptr) from = p.initial + (head * p.V + row0) * p.K;
    if (segment == run.segments - 1 && p.final_state != nullptr) to = p.final_state + (head * p.V + row0) * p.K;
  }
  float4 *const mine = reinterpret_cast<float4*>(exchange + half * 8 * 512) + lane, *const theirs = reinterpret_cast<float4*>(exchange + (half ^ 1) * 8 * 512) + lane;
  float s[kHalf / 8][4];
#pragma unroll
  for (int j = 0; j < kHalf / 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = g + (i >> 1) * 8, at = half * kHalf + j * 8 + 2 * t + (i & 1);
      s[j][i] = from != nullptr && row < rows && at < p.K ? from[(long long)row * p.K + at] : transition && row0 + row == at ? 1.0f : 0.0f;
    }

  for (int c = 0; c < chunks; ++c) {
    arrive_at(c);
    const uint8_t* const base = smem_raw + (c % stages) * stage_bytes;
    const uint32_t keys = smem_u32(base) + half * (kSteps / 2) * kBlock, solve = smem_u32(base) + 2 * W::kKeyBytes + lane * 16;
    const float* factors = reinterpret_cast<const float*>(base + 2 * W::kKeyBytes + (2 + Parts<T>::kOut) * kLower) + 2 * t;
    auto load_keys = [&](uint32_t (&b)[4][4], int k, int part) {
#pragma unroll
      for (int j = 0; j < 4; ++j) ldmatrix<false>(b[j], keys + part * kKeyPart + lane * 16 + (j * kSteps + k) * kBlock);
    };
    float x[8][4];
    uint32_t values[4][4];   // 16-bit: channels 0 .. 7 and 8 .. 15 of tokens 16 i .., then of 16 i + 8 ..
    {   // S k, of this warp's channels
      uint32_t b[2][4][4];
      load_keys(b[0], 0, 0);
      float s0, s1;
      row_scales<kHalf / 8>(s, s0, s1);
      const F2 up0 = f2_both(s0), up1 = f2_both(s1);
      uint4* const left = reinterpret_cast<uint4*>(exchange + E::kState + half * E::kStateHalf) + lane;
#pragma unroll
      for (int k = 0; k < kSteps / 2; ++k) {
        uint32_t hi[4], lo[4];
        if (k + 1 < kSteps / 2) load_keys(b[(k + 1) & 1], k + 1, 0);
        operand(s[2 * k], s[2 * k + 1], up0, up1, hi, lo);
        left[k * 32] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if constexpr (Parts<T>::kOut == 2) left[(kSteps / 2 + k) * 32] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        mma_row<8>(x, hi, b[k & 1], k == 0);
        mma_row<8>(x, lo, b[k & 1]);
        if constexpr (Parts<T>::kKey == 2) {
          load_keys(b[k & 1], k, 1);
          mma_row<8>(x, hi, b[k & 1]);
        }
      }
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ldmatrix<true>(values[i], smem_u32(base) + W::kStage + (i * 16 + (m >> 1) * 8 + r) * pitch + (slice * 16 + (m & 1) * 8) * 2);
      }
      const float i0 = inverse_of_power(s0), i1 = inverse_of_power(s1);
      reinterpret_cast<float2*>(exchange + E::kScales)[half * 32 + lane] = make_float2(i0, i1);
      barrier_arrive<kShare>(state_id);
      const F2 down0 = f2_both(i0), down1 = f2_both(i1);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        set_rows(x[j], f2_mul(first_row(x[j]), down0), f2_mul(second_row(x[j]), down1));
        mine[j * 32] = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
      }
    }
    F2 since[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) since[j] = pair_at(factors + j * 8);
    barrier<64>(pair_id);
    // v - e^G S k (the factors are negative)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 other = theirs[j * 32];
      float v[4];
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32<T>(reinterpret_cast<const T*>(values[j >> 1])[(j & 1) * 4 + i]);
      } else {
        const float* f = reinterpret_cast<const float*>(base + W::kStage);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = f[(j * 8 + 2 * t + (i & 1)) * (pitch / 4) + slice * 16 + g + (i >> 1) * 8];
      }
      set_rows(x[j], f2_fma(since[j], f2_add(first_row(x[j]), f2_pack(other.x, other.y)), first_row(v)),
               f2_fma(since[j], f2_add(second_row(x[j]), f2_pack(other.z, other.w)), second_row(v)));
    }
    // U = (v - ..) T^T: blocks 0 and 3 of 16 tokens by the first of the two warps, 1 and 2 by the second (T is lower triangular)
    {
      const int own[2] = {half, 3 - half};
      const uint32_t rows[2] = {solve + lower_block(own[0], 0) * kBlock, solve + lower_block(own[1], 0) * kBlock};
      float z[2][2][4], z2[2][2][4], r0, r1;
      uint32_t b[2][4], bl[2][4];
      auto load = [&](int i, int k) {
        ldmatrix<false>(b[i], rows[i] + k * kBlock);
        ldmatrix<false>(bl[i], rows[i] + kLower + k * kBlock);
      };
      load(0, 0);
      load(1, 0);
      row_scales<8>(x, r0, r1);
      const F2 up0 = f2_both(r0), up1 = f2_both(r1);
      auto products = [&](int i, int k, const uint32_t (&hi)[4], const uint32_t (&lo)[4]) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (k == 0) mma_first(z[i][j], hi, b[i][2 * j], b[i][2 * j + 1]);
          else mma<__half>(z[i][j], hi, b[i][2 * j], b[i][2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (k == 0) mma_first(z2[i][j], lo, b[i][2 * j], b[i][2 * j + 1]);
          else mma<__half>(z2[i][j], lo, b[i][2 * j], b[i][2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) mma<__half>(z[i][j], hi, bl[i][2 * j], bl[i][2 * j + 1]);
      };
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t hi[4], lo[4];
        operand(x[2 * k], x[2 * k + 1], up0, up1, hi, lo);
        if (k == 0 || (k == 1 && half != 0)) products(0, k, hi, lo);
        if (k == 0 && half != 0) load(0, 1);
        if (k < 3 || half == 0) products(1, k, hi, lo);
        if (k < 2 || (k == 2 && half == 0)) load(1, k + 1);
      }
      const F2 down0 = f2_both(inverse_of_power(r0)), down1 = f2_both(inverse_of_power(r1));
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int tile = 2 * own[i] + j;
          const F2 f = pair_at(factors + 3 * kChunk + tile * 8);
          float out[4];
          set_rows(out, f2_mul(f, f2_mul(f2_add(first_row(z[i][j]), first_row(z2[i][j])), down0)),
                   f2_mul(f, f2_mul(f2_add(second_row(z[i][j]), second_row(z2[i][j])), down1)));
          reinterpret_cast<float4*>(exchange + E::kWritten)[tile * 32 + lane] = make_float4(out[0], out[1], out[2], out[3]);
        }
    }
    // S = e^(G_64) S + (e^(G_64 - G) U) k, of this warp's channels
    {
      const uint32_t columns = keys + ((m & 1) * 2 + (m >> 1)) * 128 + r * 16;
      auto load_columns = [&](uint32_t (&b)[kSteps / 2][4], int k, int part) {
#pragma unroll
        for (int j = 0; j < kSteps / 2; ++j) ldmatrix<true>(b[j], columns + part * kKeyPart + (k * kSteps + j) * kBlock);
      };
      uint32_t b[2][kSteps / 2][4];
      load_columns(b[0], 0, 0);
      float u[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) since[j] = pair_at(factors + 2 * kChunk + j * 8);
      const F2 keep = f2_both(factors[5 * kChunk - 2 * t]);
      barrier<64>(pair_id);
      barrier_arrive<kShare>(written_id);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 f = reinterpret_cast<const float4*>(exchange + E::kWritten)[j * 32 + lane];
        set_rows(u[j], f2_mul(f2_pack(f.x, f.y), since[j]), f2_mul(f2_pack(f.z, f.w), since[j]));
      }
      float u0, u1, z[kHalf / 8][4];
      row_scales<8>(u, u0, u1);
      const F2 up0 = f2_both(u0), up1 = f2_both(u1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t hi[4], lo[4];
        if (k < 3) load_columns(b[(k + 1) & 1], k + 1, 0);
        operand(u[2 * k], u[2 * k + 1], up0, up1, hi, lo);
        mma_row<kHalf / 8>(z, hi, b[k & 1], k == 0);
        mma_row<kHalf / 8>(z, lo, b[k & 1]);
        if constexpr (Parts<T>::kKey == 2) {
          load_columns(b[k & 1], k, 1);
          mma_row<kHalf / 8>(z, hi, b[k & 1]);
        }
      }
      const F2 down0 = f2_both(inverse_of_power(u0)), down1 = f2_both(inverse_of_power(u1));
#pragma unroll
      for (int j = 0; j < kHalf / 8; ++j)
        set_rows(s[j], f2_fma(keep, first_row(s[j]), f2_mul(first_row(z[j]), down0)), f2_fma(keep, second_row(s[j]), f2_mul(second_row(z[j]), down1)));
    }
    leave(c);
  }

  if (to != nullptr) {
#pragma unroll
    for (int j = 0; j < kHalf / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = g + (i >> 1) * 8, at = half * kHalf + j * 8 + 2 * t + (i & 1);
        if (row < rows && at < p.K) to[(long long)row * p.K + at] = s[j][i];
      }
  }
}

// ---- segments put together -----------------------------------------------------------------------------------------

constexpr int kJoinRows = 8, kJoinThreads = 256;
constexpr int kJoinSmem = (2 * kChunkKeys + kJoinRows) * kChunkKeys * 4;
// start[j + 1] = start[j] unit_end[j] + end[j], from the row's initial state on: eight rows of the state to a block, two of them at two columns
// to a thread.  The next segment's ends are on their way meanwhile (64 KB of unit ends: read from L2 by each product they took 17 us
// a segment).
__global__ void __launch_bounds__(kJoinThreads)
delta_join_kernel(const DeltaParams p, const float* ends, float* starts, int segments) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  constexpr int kPlace = kChunkKeys * kChunkKeys;
  float* const units = reinterpret_cast<float*>(smem_raw);   // two of [K][K rounded up to 2]
  float* const s = units + 2 * kPlace;                       // [kJoinRows][kChunkKeys]
  chained();
  const int parts = (p.V + kJoinRows - 1) / kJoinRows, row0 = int(blockIdx.x % parts) * kJoinRows + threadIdx.x / 64 * 2;
  const long long head = blockIdx.x / parts;
  const int col = threadIdx.x % 64 * 2, tall = (p.V + 15) / 16 * 16 + p.K, wide = (p.K + 1) / 2 * 2;
  float* const mine = s + threadIdx.x / 64 * 2 * kChunkKeys;
  auto ask = [&](int j) {
    if (j < segments - 1) {
      const float* unit = ends + ((head * (segments - 1) + j) * tall + tall - p.K) * p.K;
      const uint32_t to = smem_u32(units + (j & 1) * kPlace);
      if (p.K % 4 == 0) {   // (as the workspace's addresses)
#pragma unroll 4
        for (int i = threadIdx.x; i < p.K * p.K / 4; i += kJoinThreads) copy16(to + i * 16, unit + i * 4, 16);
      } else {
        for (int i = threadIdx.x; i < p.K * p.K; i += kJoinThreads)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + (i / p.K * wide + i % p.K) * 4), "l"(unit + i) : "memory");
      }
    }
    async_commit();
  };
  auto load = [&](float (&x)[2][2], const float* from) {   // rows of a state, or of an end
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) x[r][c] = from != nullptr && row0 + r < p.V && col + c < p.K ? from[(long long)(row0 + r) * p.K + col + c] : 0.0f;
  };
  float x[2][2], next[2][2];
  ask(0);
  load(x, p.initial != nullptr ? p.initial + head * p.V * p.K : nullptr);
  load(next, ends + head * (segments - 1) * tall * p.K);
  for (int j = 0; j < segments - 1; ++j) {
    async_wait<0>();
    __syncthreads();   // the ends are there; all are done with the last segment's start
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      *reinterpret_cast<float2*>(mine + r * kChunkKeys + col) = make_float2(x[r][0], x[r][1]);   // (zeros behind K)
      x[r][0] = next[r][0];
      x[r][1] = next[r][1];
    }
    __syncthreads();
    ask(j + 1);
    if (j + 1 < segments - 1) load(next, ends + (head * (segments - 1) + j + 1) * tall * p.K);
    const float* unit = units + (j & 1) * kPlace + (col < p.K ? col : 0);
    int k = 0;
#pragma unroll 4
    for (; k + 4 <= p.K; k += 4) {
      float2 u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = *reinterpret_cast<const float2*>(unit + (k + i) * wide);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float4 v = *reinterpret_cast<const float4*>(mine + r * kChunkKeys + k);
        x[r][0] = fmaf(v.w, u[3].x, fmaf(v.z, u[2].x, fmaf(v.y, u[1].x, fmaf(v.x, u[0].x, x[r][0]))));
        x[r][1] = fmaf(v.w, u[3].y, fmaf(v.z, u[2].y, fmaf(v.y, u[1].y, fmaf(v.x, u[0].y, x[r][1]))));
      }
    }
    for (; k < p.K; ++k)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float2 u = *reinterpret_cast<const float2*>(unit + k * wide);
        x[r][0] = fmaf(mine[r * kChunkKeys + k], u.x, x[r][0]);
        x[r][1] = fmaf(mine[r * kChunkKeys + k], u.y, x[r][1]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (col + c >= p.K) x[r][c] = 0.0f;
        else if (row0 + r < p.V) starts[((head * (segments - 1) + j) * p.V + row0 + r) * p.K + col + c] = x[r][c];
      }
  }
}

// ---- launching -----------------------------------------------------------------------------------------------------

// Prompts that the chunks' kernels take.  Token by token prompts of 10 / 12 / 16 tokens take, in us, and a chunk:
//   16-bit   4 heads of 64 x 64 10.9 / 12.6 / 16.2, 12.6; 8 of them 11.0 / 12.9 / 16.6, 10.5; 100 rows of 4 17.9 / 20.9 / 26.9, 31.8
//            one of 128 x 128 9.2 / 10.6 / 13.5, 12.0; 32 of them 13.1 / 14.9 / 19.4, 15.5; 4 rows of 32 23.6 / 28.5 / 38.3, 28.3; 16 rows 66 / 78 / 101, 68
//   fp32     4 heads of 64 x 64 10.5 / 12.2 / 15.6, 11.5; 32 of 128 x 128 13.8 / 16.0 / 20.7, 22.2; 8 rows of 8 of them 15.4 / 18.1 / 23.1, 30.1
bool in_chunks(int dtype, const DeltaParams& p) { return p.K <= kChunkKeys && p.L > (dtype == FDNN_F32 && p.K > 64 ? 16 : 11); }

template <typename T>
bool eights(const void* q, const long long* s) {
  constexpr int kV = 16 / int(sizeof(T));
  return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && s[0] % kV == 0 && s[1] % kV == 0 && s[2] % kV == 0 && s[3] == 1;
}

constexpr int kMostSmem = 227 * 1024 - 256;   // (and the barriers)
template <typename T, int KEYS>
constexpr int smem_of(int slices, int stages) {
  return stages * (Work<T, KEYS>::kStage + kChunk * value_pitch<T>(slices)) + slices * Exchange<T, KEYS>::kBytes;
}

// Rounds of blocks of so many slices, for a number of slices to a head and of segments to a row.
long long rounds_of(const DeltaParams& p, int slices_a_head, int segments, int slices) {
  const long long blocks = (long long)p.N * p.H * segments * ((slices_a_head + slices - 1) / slices), sms = current_sm_count();
  return (blocks + sms - 1) / sms;
}
// Slices to a block.  Four take 1.7 times as long for a chunk as two (4100 and 7000 clocks: 128 x 128, bf16).
template <typename T, int KEYS>
int slices_of(const DeltaParams& p, int slices_a_head, int segments) {
  static_assert(smem_of<T, KEYS>(1, 2) <= kMostSmem, "one slice has two stages");
  int slices = slices_a_head < 2 ? slices_a_head : 2;
  if (slices_a_head > 2 && 17 * rounds_of(p, slices_a_head, segments, 4) < 10 * rounds_of(p, slices_a_head, segments, 2))
    slices = slices_a_head < 4 ? slices_a_head : 4;
  while (slices > 1 && smem_of<T, KEYS>(slices, 2) > kMostSmem) --slices;
  return slices;
}
// Segments to a row: the count with the least time, in chunks of two slices (2.2 us).  Two walks and what joins them, some 8 us and 2.4 us a
// segment and round of blocks, against one: worth it where a tenth is won.
struct Segments {
  int count, per;
};
template <typename T, int KEYS>
Segments segments_of(const DeltaParams& p) {
  const int chunks = int(((long long)p.L + kChunk - 1) / kChunk), values = (p.V + 15) / 16, keys = (p.K + 15) / 16;
  auto walk = [&](int slices_a_head, int segments, int per) {
    const int slices = slices_of<T, KEYS>(p, slices_a_head, segments);
    return per * (slices > 2 ? 1.7 : 1.0) * double(rounds_of(p, slices_a_head, segments, slices));
  };
  const long long join_blocks = (long long)p.N * p.H * ((p.V + 7) / 8), joins = (join_blocks + current_sm_count() - 1) / current_sm_count();
  Segments best = {1, chunks};
  double least = 0.9 * walk(values, 1, chunks);
  for (int count = 2; count <= kMostSegments && 2 * count <= chunks; ++count) {
    const int per = (chunks + count - 1) / count;
    if ((chunks + per - 1) / per != count) continue;   // (as many segments in pieces as long)
    const double time = walk(values + keys, count - 1, per) + walk(values, count, per) + (8.0 + 2.4 * count * double(joins)) / 2.2;
    if (time < least) least = time, best = {count, per};
  }
  return best;
}

template <typename T, int KEYS>
cudaError_t run(const DeltaParams& p, cudaStream_t stream) {
  const long long chunks = (p.L + kChunk - 1) / kChunk;
  const long long prep_blocks = (long long)p.N * p.G * chunks;
  if (prep_blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const bool keys_whole = p.K % (16 / int(sizeof(T))) == 0 && eights<T>(p.k, p.k_s) && eights<T>(p.q, p.q_s);
  constexpr int kPrepSmem = int(sizeof(PrepShared<T, KEYS>));
  auto* prep = keys_whole ? delta_prepare_kernel<T, KEYS, true> : delta_prepare_kernel<T, KEYS, false>;
  static std::atomic<uint64_t> done[2];
  cudaError_t e = allow_smem(prep, kPrepSmem, done[keys_whole]);
  if (e != cudaSuccess) return e;
  e = launch_seq(prep, dim3(unsigned(prep_blocks)), kPrepThreads, kPrepSmem, 1, stream, p);
  if (e != cudaSuccess) return e;

  const bool values_whole = p.V % (16 / int(sizeof(T))) == 0 && eights<T>(p.v, p.v_s) && eights<T>(p.y, p.y_s);
  Run r = {};
  bounded_wait_of(&r.status, &r.wait_limit, &r.skip_copies);
  if (r.status == nullptr) return cudaErrorInvalidSymbol;
  auto go = [&](auto* kernel, std::atomic<uint64_t>& allowed, int slices, long long blocks) -> cudaError_t {
    const cudaError_t err = allow_smem(kernel, kMostSmem, allowed);
    if (err != cudaSuccess) return err;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    return launch_seq(kernel, dim3(unsigned(blocks)), (2 + outs_of(slices)) * slices * 32, smem_of<T, KEYS>(slices, r.stages), 1, stream, p, r);
  };
  static std::atomic<uint64_t> allowed[4];
  auto walk = [&](int slices_a_head, int segments) -> cudaError_t {   // of each row
    const int slices = slices_of<T, KEYS>(p, slices_a_head, segments);
    r.blocks_a_head = (slices_a_head + slices - 1) / slices;
    r.stages = smem_of<T, KEYS>(slices, 3) <= kMostSmem ? 3 : 2;
    const long long blocks = (long long)p.N * p.H * segments * r.blocks_a_head;
    if (slices <= 2)
      return values_whole ? go(delta_chunks_kernel<T, KEYS, 2, true>, allowed[0], slices, blocks) : go(delta_chunks_kernel<T, KEYS, 2, false>, allowed[1], slices, blocks);
    return values_whole ? go(delta_chunks_kernel<T, KEYS, 4, true>, allowed[2], slices, blocks) : go(delta_chunks_kernel<T, KEYS, 4, false>, allowed[3], slices, blocks);
  };
  const Segments cut = segments_of<T, KEYS>(p);
  r.segments = cut.count;
  r.per = cut.per;
  if (cut.count > 1) {
    float* const ends = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + bytes_of<T, KEYS>(p));
    float* const starts = ends + (long long)p.N * p.H * (cut.count - 1) * ((p.V + 15) / 16 * 16 + p.K) * p.K;
    r.ends = ends;
    e = walk((p.V + 15) / 16 + (p.K + 15) / 16, cut.count - 1);
    if (e != cudaSuccess) return e;
    const long long joins = (long long)p.N * p.H * ((p.V + kJoinRows - 1) / kJoinRows);
    if (joins > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    static std::atomic<uint64_t> allowed_join;
    e = allow_smem(delta_join_kernel, kJoinSmem, allowed_join);
    if (e != cudaSuccess) return e;
    e = launch_seq(delta_join_kernel, dim3(unsigned(joins)), kJoinThreads, kJoinSmem, 1, stream, p, ends, starts, cut.count);
    if (e != cudaSuccess) return e;
    r.ends = nullptr;
    r.starts = starts;
  }
  return walk((p.V + 15) / 16, cut.count);
}

// f(TypeOf<T>, integral_constant<int, KEYS>)
template <typename F>
auto by_type(int dtype, const DeltaParams& p, F&& f) {
  auto go = [&](auto type) {
    if (p.K <= 64) return f(type, std::integral_constant<int, 64>{});
    return f(type, std::integral_constant<int, kChunkKeys>{});
  };
  if (dtype == FDNN_F16) return go(TypeOf<__half>{});
  if (dtype == FDNN_BF16) return go(TypeOf<__nv_bfloat16>{});
  return go(TypeOf<float>{});
}

}  // namespace

long long delta_rule_workspace(int dtype, const DeltaParams& p) {
  if (!in_chunks(dtype, p)) return 0;
  return by_type(dtype, p, [&](auto type, auto keys) -> long long {
    using T = typename decltype(type)::type;
    constexpr int kKeys = decltype(keys)::value;
    const long long cuts = segments_of<T, kKeys>(p).count - 1;
    return bytes_of<T, kKeys>(p) + (long long)p.N * p.H * cuts * ((p.V + 15) / 16 * 16 + p.K + p.V) * p.K * 4;
  });
}

cudaError_t launch_delta_rule(int dtype, const DeltaParams& p, cudaStream_t stream) {
  if (!in_chunks(dtype, p)) return launch_delta_rule_tokens(dtype, p, stream);
  return by_type(dtype, p, [&](auto type, auto keys) -> cudaError_t { return run<typename decltype(type)::type, decltype(keys)::value>(p, stream); });
}

}  // namespace fdnn
