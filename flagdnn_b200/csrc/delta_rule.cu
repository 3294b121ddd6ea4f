// The gated delta rule over prompts, in chunks of 64 tokens.
//
// With G_i = g_1 + .. + g_i within a chunk (g: logarithms of the decays), S the state before it ([V, K]) and D_ij = e^(G_i - G_j):
//   A_ij = b_i D_ij (k_i . k_j) for j < i                 what token j wrote is answered to key i
//   U    = T (v - e^G S k),   T = (1 + A)^-1 diag(b)      what each token writes
//   y_i  = scale (e^(G_i) S q_i + sum over j <= i of D_ij (q_i . k_j) U_j)
//   S    <- e^(G_64) S + sum over j of e^(G_64 - G_j) U_j k_j^T
// delta_prepare_kernel makes, for all chunks side by side, what does not need S: T, P_ij = scale D_ij (q_i . k_j), the keys and queries as
// 16-bit operands and the factors of each token.  delta_chunks_kernel then walks a head's chunks in order.  A state's rows do
// not meet, so a warp keeps 16 of them in registers, for the whole prompt, as the transposed accumulators of its own products: with rows
// as the M side, S, v - S k, U and e^.. U are in turn the accumulators of one product and the A operand of the next, without a
// word of shared memory between them, and no warp waits for another but for operands.
//
// Precision.  The tensor cores take 16 bits.  Keys and queries that come as f16 or bf16 are f16 operands exactly: each token's is
// scaled by a power of two to a largest value of 2^14 .. 2^15 (a bf16 value below 2^-29 of that loses bits that fp32 sums do not see).
// Everything made in fp32 (S, T, v - S k, U) goes in as two f16 parts, high and low, 22 bits below the row's largest value, which is
// scaled to 2^14 .. 2^15 as well; so do fp32 inputs.  Products of low parts are left out (2^-22).  For bf16 outputs (2^-8) S q and P U
// take the high parts alone, 11 bits each.  Sums are fp32; decays are differences of sums kept in 48 bits.
#include <cuda_fp16.h>

#include "delta_rule.cuh"

namespace fdnn {
namespace {

constexpr int kChunk = 64;
constexpr int kChunkKeys = 128;      // the widest key that the chunks' kernels take
constexpr int kFactors = 6 * kChunk; // floats a chunk and head: -a, b, d, t, p, and e^(G_64)
constexpr int kSquare = kChunk * kChunk * 2;   // bytes of a 64 x 64 part

// How many 16-bit parts: of keys and queries, of S and P in what only y sees.
template <typename T>
struct Parts {
  static constexpr int kKey = std::is_same<T, float>::value ? 2 : 1;
  static constexpr int kOut = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;
};

// ---- small things --------------------------------------------------------------------------------------------------

// D += A B, 16 x 8 x 16.  A: rows lane / 4 (+ 8 in a[1], a[3]), pairs of k at 2 (lane % 4) (+ 8 in a[2], a[3]); B: column lane / 4, pairs
// of k likewise; D: rows lane / 4 (+ 8 in d[2], d[3]), columns 2 (lane % 4) and the next.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// D = A B.
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// The same of 16 x 8 x 8 in TF32: A at (row, k = lane % 4), (row + 8, k), (row, k + 4), (row + 8, k + 4), B at k = lane % 4, + 4.
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// An 8 x 8 matrix of 16-bit values held as accumulators are, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {   // the rest of the 16 is zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// A power of two that takes `most` to 2^14 .. 2^15 (an exponent that it cannot have is cut; of infinity or NaN, some power).
__device__ __forceinline__ float raise(float most) {
  const int e = 268 - int((__float_as_uint(most) >> 23) & 255u);
  return __uint_as_float(uint32_t(min(max(e, 1), 253)) << 23);
}
__device__ __forceinline__ float inverse_of_power(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// Two values as f16 high parts, and what they leave as low parts.
__device__ __forceinline__ uint32_t high(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t low(float x, float y, uint32_t hi) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return high(x - h.x, y - h.y);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
// The scales of an accumulator block's two rows (lane / 4, + 8).
template <int TILES>
__device__ __forceinline__ void row_scales(const float (&c)[TILES][4], float& lower, float& upper) {
  float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    m0 = fmaxf(m0, fmaxf(fabsf(c[i][0]), fabsf(c[i][1])));
    m1 = fmaxf(m1, fmaxf(fabsf(c[i][2]), fabsf(c[i][3])));
  }
  lower = raise(quad_max(m0));
  upper = raise(quad_max(m1));
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

// Tiles of 16-bit operands: rows of COLS values, whose 16-byte pieces lie at piece ^ (row % 8), so that eight rows of a piece
// (one matrix of ldmatrix) are in different banks.  Byte offset of a piece.
template <int COLS>
__device__ __forceinline__ int piece(int row, int at) { return row * COLS * 2 + ((at ^ (row & 7)) << 4); }

// ---- where things lie in the workspace -----------------------------------------------------------------------------

template <typename T, int KEYS>
struct Work {
  static constexpr int kKeyBytes = Parts<T>::kKey * kChunk * KEYS * 2;   // keys, and as many for the queries
  static constexpr int kHeadBytes = (2 + Parts<T>::kOut) * kSquare + kFactors * 4;
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
  const long long chunks = (p.L + kChunk - 1) / kChunk;
  return (long long)p.N * chunks * ((long long)p.G * 2 * Work<T, KEYS>::kKeyBytes + (long long)p.H * Work<T, KEYS>::kHeadBytes);
}
__device__ __forceinline__ int row_end(const DeltaParams& p, long long n) {
  return p.lengths != nullptr ? min(max(p.lengths[n], 0), p.L) : p.L;
}

// ---- what does not need the state ----------------------------------------------------------------------------------

constexpr int kPrepThreads = 128;
constexpr int kPitch = kChunk + 4;   // floats between rows of A, T

template <typename T, int KEYS>
struct PrepShared {
  uint8_t keys[2 * Work<T, KEYS>::kKeyBytes];   // and the queries
  float a[kChunk][kPitch], t[kChunk][kPitch], part[4][16][20];
  float key_scale[kChunk], query_scale[kChunk], sum_hi[kChunk], sum_lo[kChunk], beta[kChunk];
  float end_hi, end_lo;
};

// A token's key or query: eight neighbouring channels of a row to their place, as parts, scaled; the factor that takes the operand
// back (with the norm, if asked, and `scale`).
template <typename T, int KEYS, bool WHOLE>
__device__ __forceinline__ void stage_rows(const DeltaParams& p, const T* x, const long long* s, int tokens, float scale, uint8_t* to,
                                           float* factor) {
  constexpr int kLanes = KEYS / 8, kRows = kPrepThreads / kLanes;
  const int at = threadIdx.x % kLanes;
#pragma unroll
  for (int r0 = 0; r0 < kChunk; r0 += kRows) {
    const int r = r0 + threadIdx.x / kLanes;
    float v[8];
    if constexpr (WHOLE) {
      constexpr int kV = 16 / sizeof(T);
#pragma unroll
      for (int i = 0; i < 8 / kV; ++i) {
        Pack<T, kV> q;
        q.clear();
        if (r < tokens && at * 8 + i * kV < p.K) q.load(x + r * s[1] + at * 8 + i * kV);
#pragma unroll
        for (int j = 0; j < kV; ++j) v[i * kV + j] = q.at(j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = r < tokens && at * 8 + j < p.K ? to_f32<T>(x[r * s[1] + (at * 8 + j) * s[3]]) : 0.0f;
    }
    float most = 0.0f, squares = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      most = fmaxf(most, fabsf(v[j]));
      squares += v[j] * v[j];
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) {
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      squares += __shfl_xor_sync(0xffffffffu, squares, o);
    }
    const float up = raise(most);
    uint4 hi, lo;
    uint32_t* h = reinterpret_cast<uint32_t*>(&hi);
    uint32_t* l = reinterpret_cast<uint32_t*>(&lo);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[j] = high(v[2 * j] * up, v[2 * j + 1] * up);
      l[j] = low(v[2 * j] * up, v[2 * j + 1] * up, h[j]);
    }
    *reinterpret_cast<uint4*>(to + piece<KEYS>(r, at)) = hi;
    if constexpr (Parts<T>::kKey == 2) *reinterpret_cast<uint4*>(to + kChunk * KEYS * 2 + piece<KEYS>(r, at)) = lo;
    if (at == 0) factor[r] = r < tokens ? scale * inverse_of_power(up) * (p.norm ? 1.0f / sqrtf(squares + kKeyEps) : 1.0f) : 0.0f;
  }
}

// c += the products of 16 rows of `x` (from row0) with the first `tiles` x 8 rows of `y`, over KEYS channels.
template <typename T, int KEYS>
__device__ __forceinline__ void dots(float (&c)[8][4], const uint8_t* x, const uint8_t* y, int row0, int pairs) {
  const int lane = threadIdx.x & 31, m = lane >> 3, r = lane & 7;
  const uint32_t xs = smem_u32(x), ys = smem_u32(y);
  constexpr int kPart = kChunk * KEYS * 2;
#pragma unroll
  for (int s = 0; s < KEYS / 16; ++s) {
    uint32_t a[Parts<T>::kKey][4];
#pragma unroll
    for (int i = 0; i < Parts<T>::kKey; ++i) ldmatrix(a[i], xs + i * kPart + piece<KEYS>(row0 + (m & 1) * 8 + r, 2 * s + (m >> 1)));
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (n < pairs) {
        uint32_t b[Parts<T>::kKey][4];
#pragma unroll
        for (int i = 0; i < Parts<T>::kKey; ++i) ldmatrix(b[i], ys + i * kPart + piece<KEYS>(n * 16 + (m >> 1) * 8 + r, 2 * s + (m & 1)));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mma(c[2 * n + j], a[0], b[0][2 * j], b[0][2 * j + 1]);
          if constexpr (Parts<T>::kKey == 2) {
            mma(c[2 * n + j], a[0], b[1][2 * j], b[1][2 * j + 1]);
            mma(c[2 * n + j], a[1], b[0][2 * j], b[0][2 * j + 1]);
          }
        }
      }
  }
}

// d += x y of 16 x 16 blocks in fp32, by 3 x TF32 (a high part is the number cut to TF32, what it leaves is exact; 2^-21).
__device__ __forceinline__ void block_product(float (&d)[2][4], const float* x, int x_pitch, const float* y, int y_pitch) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    uint32_t a[4], al[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = x[(g + (i & 1) * 8) * x_pitch + s * 8 + t + (i >> 1) * 4];
      a[i] = __float_as_uint(v) & 0xffffe000u;
      al[i] = __float_as_uint(v - __uint_as_float(a[i]));
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      uint32_t b[2], bl[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float v = y[(s * 8 + t + i * 4) * y_pitch + n * 8 + g];
        b[i] = __float_as_uint(v) & 0xffffe000u;
        bl[i] = __float_as_uint(v - __uint_as_float(b[i]));
      }
      mma_tf32(d[n], a, bl[0], bl[1]);
      mma_tf32(d[n], al, b[0], b[1]);
      mma_tf32(d[n], a, b[0], b[1]);
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
  __syncthreads();
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
  __syncthreads();
  {   // the lower left 32 x 32: part = a t, then t part
    const int i = 32 + (warp >> 1) * 16, j = (warp & 1) * 16;
    float d[2][4] = {};
    for (int m = j; m < 32; m += 16) block_product(d, &a[i][m], kPitch, &t[m][j], kPitch);
    put_block(&part[warp][0][0], 20, d, 1.0f);
    __syncthreads();
    float e[2][4] = {};
    for (int m = 32; m <= i; m += 16) block_product(e, &t[i][m], kPitch, &part[(m - 32) / 16 * 2 + (warp & 1)][0][0], 20);
    put_block(&t[i][j], kPitch, e, -1.0f);
  }
  __syncthreads();
}

template <typename T, int KEYS, bool WHOLE>
__global__ void __launch_bounds__(kPrepThreads)
delta_prepare_kernel(const DeltaParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  PrepShared<T, KEYS>& s = *reinterpret_cast<PrepShared<T, KEYS>*>(smem_raw);
  chained();
  using W = Work<T, KEYS>;
  const Layout w = layout_of<T, KEYS>(p);
  const int c = int(blockIdx.x % w.chunks), g = int(blockIdx.x / w.chunks % p.G);
  const long long n = blockIdx.x / w.chunks / p.G;
  const int begin = c * kChunk, tokens = min(row_end(p, n) - begin, kChunk);
  if (tokens <= 0) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q = lane >> 2, t = lane & 3;
  uint8_t* const queries = s.keys + W::kKeyBytes;
  stage_rows<T, KEYS, WHOLE>(p, static_cast<const T*>(p.k) + n * p.k_s[0] + begin * p.k_s[1] + g * p.k_s[2], p.k_s, tokens, 1.0f, s.keys,
                             s.key_scale);
  stage_rows<T, KEYS, WHOLE>(p, static_cast<const T*>(p.q) + n * p.q_s[0] + begin * p.q_s[1] + g * p.q_s[2], p.q_s, tokens, p.scale, queries,
                             s.query_scale);
  __syncthreads();
  {
    uint4* to = reinterpret_cast<uint4*>(w.keys + ((n * p.G + g) * w.chunks + c) * (2ll * W::kKeyBytes));
    const uint4* from = reinterpret_cast<const uint4*>(s.keys);
#pragma unroll 4
    for (int i = tid; i < 2 * W::kKeyBytes / 16; i += kPrepThreads) to[i] = from[i];
  }
  float kk[8][4] = {}, qk[8][4] = {};
  dots<T, KEYS>(kk, s.keys, s.keys, warp * 16, warp + 1);
  dots<T, KEYS>(qk, queries, s.keys, warp * 16, warp + 1);

  const int group = p.H / p.G;
  for (int h = g * group; h < (g + 1) * group; ++h) {
    if (warp == 0) {   // two tokens a lane
      const float A = p.A != nullptr ? p.A[h] : 1.0f, bias = p.delta_bias != nullptr ? p.delta_bias[h] : 0.0f;
      double v[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = 2 * lane + j;
        float gl = 0.0f, b = 0.0f;
        if (i < tokens) {
          gl = log_decay(p, gate_at<T>(p, p.delta, n * p.delta_s[0] + (begin + i) * p.delta_s[1] + h * p.delta_s[2]), bias, A);
          b = step_size(p, gate_at<T>(p, p.beta, n * p.beta_s[0] + (begin + i) * p.beta_s[1] + h * p.beta_s[2]));
          gl = gl < -1e5f ? -1e5f : gl;   // a decay of zero, whose difference to itself is a number; NaN stays
        }
        v[j] = double(gl);
        s.beta[i] = b;
      }
      double sum = v[0] + v[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double other = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += other;
      }
      const double each[2] = {sum - v[1], sum};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float hi = float(each[j]);
        s.sum_hi[2 * lane + j] = hi;
        s.sum_lo[2 * lane + j] = float(each[j] - double(hi));
      }
    }
    __syncthreads();
    uint8_t* out = w.heads + ((n * p.H + h) * w.chunks + c) * (long long)W::kHeadBytes;
    float* factors = reinterpret_cast<float*>(out + (2 + Parts<T>::kOut) * kSquare);
    if (tid < kChunk) {
      const float hi = s.sum_hi[tid], lo = s.sum_lo[tid], since = expf(hi + lo);
      factors[tid] = -since * s.key_scale[tid];
      factors[kChunk + tid] = since * s.query_scale[tid];
      factors[2 * kChunk + tid] = expf((s.sum_hi[kChunk - 1] - hi) + (s.sum_lo[kChunk - 1] - lo)) * s.key_scale[tid];
      if (tid == kChunk - 1) factors[5 * kChunk] = since;
    }
    // a and P, from this warp's 16 rows
    const int r0 = warp * 16 + q;
    float hi[2], lo[2], beta[2], most[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      hi[i] = s.sum_hi[r0 + 8 * i];
      lo[i] = s.sum_lo[r0 + 8 * i];
      beta[i] = s.beta[r0 + 8 * i] * s.key_scale[r0 + 8 * i];
    }
    float pm[8][4];
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = r0 + (i >> 1) * 8, col = m * 8 + 2 * t + (i & 1);
        float av = 0.0f, pv = 0.0f;
        if (m < 2 * (warp + 1) && col <= row) {
          const float d = expf((hi[i >> 1] - s.sum_hi[col]) + (lo[i >> 1] - s.sum_lo[col])) * s.key_scale[col];
          if (col < row) av = kk[m][i] * beta[i >> 1] * d;
          pv = qk[m][i] * s.query_scale[row] * d;
        }
        s.a[row][col] = av;
        pm[m][i] = pv;
        most[i >> 1] = fmaxf(most[i >> 1], fabsf(pv));
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float up = raise(quad_max(most[i]));
      if (t == 0) factors[4 * kChunk + r0 + 8 * i] = inverse_of_power(up);
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const float x = pm[m][2 * i] * up, y = pm[m][2 * i + 1] * up;
        const uint32_t h16 = high(x, y);
        uint8_t* at = out + 2 * kSquare + piece<kChunk>(r0 + 8 * i, m) + t * 4;
        *reinterpret_cast<uint32_t*>(at) = h16;
        if constexpr (Parts<T>::kOut == 2) *reinterpret_cast<uint32_t*>(at + kSquare) = low(x, y, h16);
      }
    }
    __syncthreads();
    invert(s.a, s.t, s.part);
    {   // T = t diag(beta), two threads a row
      const int row = tid >> 1, from = (tid & 1) * 32;
      float v[32], top = 0.0f;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        v[j] = from + j <= row ? s.t[row][from + j] * s.beta[from + j] : 0.0f;
        top = fmaxf(top, fabsf(v[j]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      const float up = raise(top);
      if (from == 0) factors[3 * kChunk + row] = inverse_of_power(up);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        uint4 h4, l4;
        uint32_t *hp = reinterpret_cast<uint32_t*>(&h4), *lp = reinterpret_cast<uint32_t*>(&l4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = v[m * 8 + 2 * j] * up, y = v[m * 8 + 2 * j + 1] * up;
          hp[j] = high(x, y);
          lp[j] = low(x, y, hp[j]);
        }
        uint8_t* at = out + piece<kChunk>(row, from / 8 + m);
        *reinterpret_cast<uint4*>(at) = h4;
        *reinterpret_cast<uint4*>(at + kSquare) = l4;
      }
    }
    __syncthreads();
  }
}

// ---- the chunks in order -------------------------------------------------------------------------------------------

constexpr int kMostSlices = 4;           // 16 rows of the state each, two warps to a slice
constexpr int kExchange = 2 * 16 * 512;  // bytes through which two warps add up their halves

template <typename T>
__host__ __device__ constexpr int value_pitch(int slices) { return 16 * slices * int(sizeof(T)) + 16; }   // bytes; eight rows in different banks

__device__ __forceinline__ void pair_barrier(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ F2 pair_at(const float* p) { return *reinterpret_cast<const F2*>(p); }

// Two output tiles: o[i][..] holds rows (value channels) lane / 4, + 8 and tokens 8 i + 2 (lane % 4), + 1.
template <typename T, bool WHOLE>
__device__ __forceinline__ void put_outputs(const DeltaParams& p, T* y, const float (&o)[2][4], int tokens, int channels) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    if constexpr (sizeof(T) == 2) {
      const uint32_t lower = transposed(pack2(from_f32<T>(o[n][0]), from_f32<T>(o[n][1])));
      const uint32_t upper = transposed(pack2(from_f32<T>(o[n][2]), from_f32<T>(o[n][3])));
      const int token = n * 8 + g;
      if (token < tokens) {
        T* at = y + token * p.y_s[1];
        if constexpr (WHOLE) {   // pairs of channels lie together and are whole
          if (2 * t < channels) *reinterpret_cast<uint32_t*>(at + 2 * t) = lower;
          if (8 + 2 * t < channels) *reinterpret_cast<uint32_t*>(at + 8 + 2 * t) = upper;
        } else {
          const T *l = reinterpret_cast<const T*>(&lower), *u = reinterpret_cast<const T*>(&upper);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (2 * t + j < channels) at[(2 * t + j) * p.y_s[3]] = l[j];
            if (8 + 2 * t + j < channels) at[(8 + 2 * t + j) * p.y_s[3]] = u[j];
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int token = n * 8 + 2 * t + (i & 1), channel = g + (i >> 1) * 8;
        if (token < tokens && channel < channels) y[token * p.y_s[1] + channel * p.y_s[3]] = from_f32<T>(o[n][i]);
      }
    }
  }
}

// WHOLE: 16 bytes of neighbouring value channels are copied at once, and pairs stored.
template <typename T, int KEYS, bool WHOLE>
__global__ void __launch_bounds__(2 * kMostSlices * 32, 1)
delta_chunks_kernel(const DeltaParams p, int blocks_a_head, int stages) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  chained();
  using W = Work<T, KEYS>;
  constexpr int kKeyPart = kChunk * KEYS * 2, kHalf = KEYS / 2;
  const Layout w = layout_of<T, KEYS>(p);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slices = blockDim.x >> 6;
  const int h = int(blockIdx.x / blocks_a_head % p.H);
  const long long n = blockIdx.x / blocks_a_head / p.H;
  const int end = row_end(p, n), chunks = (end + kChunk - 1) / kChunk;
  const int first = int(blockIdx.x % blocks_a_head) * slices * 16;   // the block's first value channel
  const int pitch = value_pitch<T>(slices), stage_bytes = W::kStage + kChunk * pitch;
  const uint32_t smem = smem_u32(smem_raw);

  const uint8_t* keys_from = w.keys + (n * p.G + h / (p.H / p.G)) * w.chunks * (2ll * W::kKeyBytes);
  const uint8_t* heads_from = w.heads + (n * p.H + h) * w.chunks * (long long)W::kHeadBytes;
  const T* v0 = static_cast<const T*>(p.v) + n * p.v_s[0] + h * p.v_s[2] + first * p.v_s[3];
  auto ask = [&](int c) {   // a chunk's operands, by all threads
    const int tid = threadIdx.x, step = blockDim.x;
    const uint32_t to = smem + (c % stages) * stage_bytes;
    const uint8_t* from = keys_from + c * (2ll * W::kKeyBytes);
#pragma unroll 8
    for (int i = tid; i < 2 * W::kKeyBytes / 16; i += step) copy16(to + i * 16, from + i * 16, 16);
    from = heads_from + c * (long long)W::kHeadBytes;
#pragma unroll 8
    for (int i = tid; i < W::kHeadBytes / 16; i += step) copy16(to + 2 * W::kKeyBytes + i * 16, from + i * 16, 16);
    const int here = min(slices * 16, p.V - first), tokens = min(end - c * kChunk, kChunk);
    const uint32_t values = to + W::kStage;
    if constexpr (WHOLE) {
      constexpr int kV = 16 / sizeof(T);
      const int pieces = slices * 16 / kV;   // a thread keeps its column: 64 slices threads are a multiple of it
      const int at = tid % pieces * kV, bytes = min(max(here - at, 0), kV) * int(sizeof(T));
#pragma unroll 4
      for (int r = tid / pieces; r < kChunk; r += step / pieces) {
        const bool there = r < tokens && bytes > 0;
        copy16(values + r * pitch + at * int(sizeof(T)), there ? v0 + (c * kChunk + r) * p.v_s[1] + at : v0, there ? bytes : 0);
      }
    } else {
      T* to_v = reinterpret_cast<T*>(smem_raw + (c % stages) * stage_bytes + W::kStage);
      for (int i = tid; i < kChunk * slices * 16; i += step) {
        const int r = i / (slices * 16), at = i % (slices * 16);
        to_v[r * (pitch / int(sizeof(T))) + at] =
            r < tokens && at < here ? v0[(c * kChunk + r) * p.v_s[1] + at * p.v_s[3]] : from_f32<T>(0.0f);
      }
    }
    async_commit();
  };
  if (chunks > 0) ask(0);

  // Two warps hold 16 rows of the state, half of the keys' channels each: s[j] rows lane / 4, + 8, channels 8 j + 2 (lane % 4), + 1.
  const int g = lane >> 2, t = lane & 3, m = lane >> 3, r = lane & 7;
  const int slice = warp >> 1, half = warp & 1;
  const int row0 = first + slice * 16, channels = min(16, p.V - row0);
  const long long state_at = ((n * p.H + h) * p.V + row0) * (long long)p.K;
  // what a warp leaves for the other one: its 8 tiles of S k, and its 8 of S q
  float4* const exchange = reinterpret_cast<float4*>(smem_raw + stages * stage_bytes + slice * kExchange) + lane;
  float4 *const mine = exchange + half * 16 * 32, *const theirs = exchange + (half ^ 1) * 16 * 32;
  float s[kHalf / 8][4];
#pragma unroll
  for (int j = 0; j < kHalf / 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = g + (i >> 1) * 8, at = half * kHalf + j * 8 + 2 * t + (i & 1);
      s[j][i] = p.initial != nullptr && row < channels && at < p.K ? p.initial[state_at + (long long)row * p.K + at] : 0.0f;
    }
  T* y = static_cast<T*>(p.y) + n * p.y_s[0] + h * p.y_s[2] + row0 * p.y_s[3];
  // y of 16-token blocks 0 and 3 is finished by the first of the two warps, of 1 and 2 by the second: P is lower triangular
  const int own[2] = {half, 3 - half};

  for (int c = 0; c < chunks; ++c) {
    async_wait<0>();
    __syncthreads();   // chunk c is there, and all are done with chunk c - 1
    if (stages > 1 && c + 1 < chunks) ask(c + 1);
    const int base_at = (c % stages) * stage_bytes;
    const uint32_t keys = smem + base_at, queries = keys + W::kKeyBytes, square = queries + W::kKeyBytes;
    const float* factors = reinterpret_cast<const float*>(smem_raw + base_at + 2 * W::kKeyBytes + (2 + Parts<T>::kOut) * kSquare) + 2 * t;
    float x[8][4];
    {   // S k and S q, of this warp's channels
      float s0, s1, o[8][4];
      row_scales<kHalf / 8>(s, s0, s1);
      const F2 up0 = f2_both(s0), up1 = f2_both(s1);
#pragma unroll
      for (int k = 0; k < kHalf / 16; ++k) {
        uint32_t hi[4], lo[4];
        operand(s[2 * k], s[2 * k + 1], up0, up1, hi, lo);
        const int at = half * (kHalf / 8) + 2 * k + (m & 1);
        uint32_t b[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) ldmatrix(b[j], keys + piece<KEYS>(j * 16 + (m >> 1) * 8 + r, at));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (k == 0) mma_first(x[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
          else mma(x[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) mma(x[j], lo, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
        if constexpr (Parts<T>::kKey == 2) {
#pragma unroll
          for (int j = 0; j < 4; ++j) ldmatrix(b[j], keys + kKeyPart + piece<KEYS>(j * 16 + (m >> 1) * 8 + r, at));
#pragma unroll
          for (int j = 0; j < 8; ++j) mma(x[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) ldmatrix(b[j], queries + piece<KEYS>(j * 16 + (m >> 1) * 8 + r, at));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (k == 0) mma_first(o[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
          else mma(o[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
        }
        if constexpr (Parts<T>::kOut == 2) {
#pragma unroll
          for (int j = 0; j < 8; ++j) mma(o[j], lo, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
        }
        if constexpr (Parts<T>::kKey == 2) {
#pragma unroll
          for (int j = 0; j < 4; ++j) ldmatrix(b[j], queries + kKeyPart + piece<KEYS>(j * 16 + (m >> 1) * 8 + r, at));
#pragma unroll
          for (int j = 0; j < 8; ++j) mma(o[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
        }
      }
      const F2 down0 = f2_both(inverse_of_power(s0)), down1 = f2_both(inverse_of_power(s1));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        set_rows(x[j], f2_mul(first_row(x[j]), down0), f2_mul(second_row(x[j]), down1));
        set_rows(o[j], f2_mul(first_row(o[j]), down0), f2_mul(second_row(o[j]), down1));
        mine[j * 32] = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
        mine[(8 + j) * 32] = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
      }
    }
    pair_barrier(1 + slice);
    // v - e^G S k (the factors are negative)
    const uint32_t values = smem + base_at + W::kStage;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float v[2][4];
      if constexpr (sizeof(T) == 2) {
        uint32_t b[4];   // channels 0 .. 7 and 8 .. 15 of tokens 8 j .., then of 8 (j + 1) ..
        ldmatrix_t(b, values + (j * 8 + (m >> 1) * 8 + r) * pitch + (slice * 16 + (m & 1) * 8) * 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i >> 2][i & 3] = to_f32<T>(reinterpret_cast<const T*>(b)[i]);
      } else {
        const float* f = reinterpret_cast<const float*>(smem_raw + base_at + W::kStage);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i >> 2][i & 3] = f[((j + (i >> 2)) * 8 + 2 * t + (i & 1)) * (pitch / 4) + slice * 16 + g + ((i >> 1) & 1) * 8];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const F2 a = pair_at(factors + (j + i) * 8);
        const float4 other = theirs[(j + i) * 32];
        set_rows(x[j + i], f2_fma(a, f2_add(first_row(x[j + i]), f2_pack(other.x, other.y)), first_row(v[i])),
                 f2_fma(a, f2_add(second_row(x[j + i]), f2_pack(other.z, other.w)), second_row(v[i])));
      }
    }
    // U = (v - ..) T^T, by both warps
    float u[8][4];
    {
      float r0, r1;
      row_scales<8>(x, r0, r1);
      const F2 up0 = f2_both(r0), up1 = f2_both(r1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t hi[4], lo[4], b[4][4], bl[4][4];
        operand(x[2 * k], x[2 * k + 1], up0, up1, hi, lo);
#pragma unroll
        for (int j = k; j < 4; ++j) {   // (T is lower triangular)
          const uint32_t at = square + piece<kChunk>(j * 16 + (m >> 1) * 8 + r, 2 * k + (m & 1));
          ldmatrix(b[j], at);
          ldmatrix(bl[j], at + kSquare);
        }
#pragma unroll
        for (int j = 2 * k; j < 8; ++j) {
          if (k == 0) mma_first(u[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
          else mma(u[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
        }
#pragma unroll
        for (int j = 2 * k; j < 8; ++j) mma(u[j], lo, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
#pragma unroll
        for (int j = 2 * k; j < 8; ++j) mma(u[j], hi, bl[j >> 1][2 * (j & 1)], bl[j >> 1][2 * (j & 1) + 1]);
      }
      const F2 down0 = f2_both(inverse_of_power(r0)), down1 = f2_both(inverse_of_power(r1));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const F2 f = pair_at(factors + 3 * kChunk + j * 8);
        set_rows(u[j], f2_mul(f, f2_mul(first_row(u[j]), down0)), f2_mul(f, f2_mul(second_row(u[j]), down1)));
      }
    }
    {   // y = e^G S q + U P^T
      float u0, u1, z[2][2][4] = {};
      row_scales<8>(u, u0, u1);
      const F2 up0 = f2_both(u0), up1 = f2_both(u1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t hi[4], lo[4];
        if constexpr (Parts<T>::kOut == 2) operand(u[2 * k], u[2 * k + 1], up0, up1, hi, lo);
        else operand(u[2 * k], u[2 * k + 1], up0, up1, hi);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (k <= own[i]) {
            const uint32_t at = square + 2 * kSquare + piece<kChunk>(own[i] * 16 + (m >> 1) * 8 + r, 2 * k + (m & 1));
            uint32_t b[4];
            ldmatrix(b, at);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mma(z[i][j], hi, b[2 * j], b[2 * j + 1]);
              if constexpr (Parts<T>::kOut == 2) mma(z[i][j], lo, b[2 * j], b[2 * j + 1]);
            }
            if constexpr (Parts<T>::kOut == 2) {
              ldmatrix(b, at + kSquare);
#pragma unroll
              for (int j = 0; j < 2; ++j) mma(z[i][j], hi, b[2 * j], b[2 * j + 1]);
            }
          }
      }
      const F2 down0 = f2_both(inverse_of_power(u0)), down1 = f2_both(inverse_of_power(u1));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int tile = own[i] * 2 + j;
          const F2 b = pair_at(factors + kChunk + tile * 8), f = pair_at(factors + 4 * kChunk + tile * 8);
          const float4 o = mine[(8 + tile) * 32], other = theirs[(8 + tile) * 32];
          const F2 q0 = f2_mul(b, f2_add(f2_pack(o.x, o.y), f2_pack(other.x, other.y)));
          const F2 q1 = f2_mul(b, f2_add(f2_pack(o.z, o.w), f2_pack(other.z, other.w)));
          set_rows(z[i][j], f2_fma(f, f2_mul(first_row(z[i][j]), down0), q0), f2_fma(f, f2_mul(second_row(z[i][j]), down1), q1));
        }
        const int token = c * kChunk + own[i] * 16;
        put_outputs<T, WHOLE>(p, y + token * p.y_s[1], z[i], end - token, channels);
      }
    }
    // S = e^(G_64) S + (e^(G_64 - G) U) k, of this warp's channels
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const F2 f = pair_at(factors + 2 * kChunk + j * 8);
      set_rows(u[j], f2_mul(first_row(u[j]), f), f2_mul(second_row(u[j]), f));
    }
    {
      const F2 keep = f2_both(factors[5 * kChunk - 2 * t]);
      float u0, u1, z[kHalf / 8][4];
      row_scales<8>(u, u0, u1);
      const F2 up0 = f2_both(u0), up1 = f2_both(u1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t hi[4], lo[4], b[kHalf / 16][4];
        operand(u[2 * k], u[2 * k + 1], up0, up1, hi, lo);
#pragma unroll
        for (int j = 0; j < kHalf / 16; ++j)
          ldmatrix_t(b[j], keys + piece<KEYS>(k * 16 + (m & 1) * 8 + r, half * (kHalf / 8) + 2 * j + (m >> 1)));
#pragma unroll
        for (int j = 0; j < kHalf / 8; ++j) {
          if (k == 0) mma_first(z[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
          else mma(z[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
        }
#pragma unroll
        for (int j = 0; j < kHalf / 8; ++j) mma(z[j], lo, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
        if constexpr (Parts<T>::kKey == 2) {
#pragma unroll
          for (int j = 0; j < kHalf / 16; ++j)
            ldmatrix_t(b[j], keys + kKeyPart + piece<KEYS>(k * 16 + (m & 1) * 8 + r, half * (kHalf / 8) + 2 * j + (m >> 1)));
#pragma unroll
          for (int j = 0; j < kHalf / 8; ++j) mma(z[j], hi, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
        }
      }
      const F2 down0 = f2_both(inverse_of_power(u0)), down1 = f2_both(inverse_of_power(u1));
#pragma unroll
      for (int j = 0; j < kHalf / 8; ++j)
        set_rows(s[j], f2_fma(keep, first_row(s[j]), f2_mul(first_row(z[j]), down0)), f2_fma(keep, second_row(s[j]), f2_mul(second_row(z[j]), down1)));
    }
    if (stages == 1) {
      __syncthreads();
      if (c + 1 < chunks) ask(c + 1);
    }
  }

  if (p.final_state != nullptr) {
#pragma unroll
    for (int j = 0; j < kHalf / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = g + (i >> 1) * 8, at = half * kHalf + j * 8 + 2 * t + (i & 1);
        if (row < channels && at < p.K) p.final_state[state_at + (long long)row * p.K + at] = s[j][i];
      }
  }
  // tokens behind the row's end
  for (long long i = end * 16ll + half * 32 + lane; i < p.L * 16ll; i += 64)
    if (i % 16 < channels) y[i / 16 * p.y_s[1] + i % 16 * p.y_s[3]] = from_f32<T>(0.0f);
}

// ---- launching -----------------------------------------------------------------------------------------------------

// Prompts that the chunks' kernels take.
bool in_chunks(const DeltaParams& p) { return p.K <= kChunkKeys && p.L > 16; }

template <typename T>
bool eights(const void* q, const long long* s) {
  constexpr int kV = 16 / int(sizeof(T));
  return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && s[0] % kV == 0 && s[1] % kV == 0 && s[2] % kV == 0 && s[3] == 1;
}

template <typename T, int KEYS>
cudaError_t run(const DeltaParams& p, cudaStream_t stream) {
  const long long chunks = (p.L + kChunk - 1) / kChunk;
  const long long prep_blocks = (long long)p.N * p.G * chunks;
  if (prep_blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const bool keys_whole = p.K % (16 / int(sizeof(T))) == 0 && eights<T>(p.k, p.k_s) && eights<T>(p.q, p.q_s);
  constexpr int kPrepSmem = int(sizeof(PrepShared<T, KEYS>));
  auto* prep = keys_whole ? delta_prepare_kernel<T, KEYS, true> : delta_prepare_kernel<T, KEYS, false>;
  static std::atomic<uint64_t> done[4];
  cudaError_t e = allow_smem(prep, kPrepSmem, done[keys_whole]);
  if (e != cudaSuccess) return e;
  e = launch_seq(prep, dim3(unsigned(prep_blocks)), kPrepThreads, kPrepSmem, 1, stream, p);
  if (e != cudaSuccess) return e;

  const int most = (p.V + 15) / 16;
  auto blocks_of = [&](int slices) { return (long long)p.N * p.H * ((most + slices - 1) / slices); };
  auto smem_of = [&](int slices, int stages) {
    return stages * (Work<T, KEYS>::kStage + kChunk * value_pitch<T>(slices)) + slices * kExchange;
  };
  constexpr int kMostSmem = 227 * 1024;
  // Four slices to a block put two warps on a quarter of an SM: a chunk takes longer, but twice the rows
  int slices = most < 2 ? most : 2;
  if (most > 2 && 5 * ((blocks_of(4) + current_sm_count() - 1) / current_sm_count()) < 3 * ((blocks_of(2) + current_sm_count() - 1) / current_sm_count()))
    slices = most < 4 ? most : 4;
  while (slices > 1 && smem_of(slices, 2) > kMostSmem) --slices;
  const int stages = smem_of(slices, 2) <= kMostSmem ? 2 : 1;
  const long long blocks = blocks_of(slices);
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const bool values_whole = eights<T>(p.v, p.v_s) && p.V % 2 == 0 && p.y_s[3] == 1 && p.y_s[0] % 2 == 0 && p.y_s[1] % 2 == 0 &&
                            p.y_s[2] % 2 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 3u) == 0;
  auto* kernel = values_whole ? delta_chunks_kernel<T, KEYS, true> : delta_chunks_kernel<T, KEYS, false>;
  e = allow_smem(kernel, kMostSmem, done[2 + values_whole]);
  if (e != cudaSuccess) return e;
  return launch_seq(kernel, dim3(unsigned(blocks)), 2 * slices * 32, smem_of(slices, stages), 1, stream, p,
                    (most + slices - 1) / slices, stages);
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
  if (!in_chunks(p)) return 0;
  return by_type(dtype, p, [&](auto type, auto keys) -> long long { return bytes_of<typename decltype(type)::type, decltype(keys)::value>(p); });
}

cudaError_t launch_delta_rule(int dtype, const DeltaParams& p, cudaStream_t stream) {
  if (!in_chunks(p)) return launch_delta_rule_tokens(dtype, p, stream);
  return by_type(dtype, p, [&](auto type, auto keys) -> cudaError_t { return run<typename decltype(type)::type, decltype(keys)::value>(p, stream); });
}

}  // namespace fdnn
