// Quantisation to microscaled 4-bit floating point, optionally behind a modulated layer norm, and back.
//
//   y = (x - mean) rsqrt(var + eps) (1 + scale) + shift          where shift and scale are given
//   block scale from the block's largest magnitude, codes = y / scale to the nearest (ties to even), saturating
//
// One pass over x.  Bound by memory: 2 bytes in, 0.5 + 1/16 (or 1/32) out for each 16-bit element.
#include "fp4.cuh"
#include "internal.h"

namespace t2t {

// Quantises the 16 elements from column `at` of a row, one or half a block, and writes their codes (where the row has room for
// them); `on`: there is such a unit, up to the last whole atom.  The first lane of an atom's word writes it.
template <int FMT, bool EXACT>
__device__ __forceinline__ void put_unit(float* y, bool on, int row, int at, int pitch, int atoms, float g, float inv_g,
                                         uint8_t* codes, uint8_t* scales) {
  constexpr int B = fp4_block(FMT);
  uint32_t word;
  const uint2 c = fp4_unit<FMT, EXACT>(y, g, inv_g, word);
  if (!on) return;
  if ((at & (4 * B - 1)) == 0) *reinterpret_cast<uint32_t*>(scales + fp4_scale_offset(row, at / B, atoms)) = word;
  if (at / 2 < pitch) *reinterpret_cast<uint2*>(codes + (long long)row * pitch + at / 2) = c;
}

// Walks the items (row, column) of rows x columns in steps of 256 threads without a division per item.
struct Walk {
  int row, col, dr, dc, cols;
  __device__ __forceinline__ Walk(int first_row, int columns) : cols(columns) {
    dr = 256 / columns;
    dc = 256 - dr * columns;
    row = threadIdx.x / columns;
    col = threadIdx.x - row * columns;
    row += first_row;
  }
  __device__ __forceinline__ void next() {
    row += dr;
    col += dc;
    if (col >= cols) {
      col -= cols;
      ++row;
    }
  }
};

// A thread takes 16 elements, rows are rounded up to whole atoms.  A CTA takes `rows` whole rows.  (A block of 32 to a thread: 128
// bytes a lane of a 32-bit matrix, 4.1 TB/s.)
template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(256) fp4_quantize_kernel(const T* __restrict__ x, long long x_row, int M, int K, float g,
                                                           float inv_g, int rows, int pitch, int atoms,
                                                           uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int row0 = blockIdx.x * rows, end = min(row0 + rows, M);
  Walk w(row0, atoms * (fp4_block(FMT) / 4));
  const int items = (end - row0) * w.cols;
  grid_release();
  for (int i = 0; i < items; i += 256, w.next()) {
    const bool on = w.row < end;
    const int at = w.col * 16;
    float y[16];
    load16<T, VEC>(x + (on ? w.row : row0) * x_row + at, on ? K - at : 0, y);
    put_unit<FMT, true>(y, on, w.row, at, pitch, atoms, g, inv_g, codes, scales);
  }
}

// 16 elements of a shift or scale from column `at`: of x's type, or of 32 bits.
template <typename T, bool VEC>
__device__ __forceinline__ void load_vector(const void* v, bool wide, int at, int K, float* y) {
  if (sizeof(T) == 2 && wide) load16<float, VEC>(static_cast<const float*>(v) + at, K - at, y);
  else load16<T, VEC>(static_cast<const T*>(v) + at, K - at, y);
}

// Modulated rows.  A thread owns U x 16 columns and walks down the CTA's rows, R at a time, the next ones on their way meanwhile; shift
// and 1 + scale lie in shared memory in 32 bits, read once for all R.  Mean, then mean square about it, from registers: one pass over x.
// Bound by instructions and the latency of its sums (two meetings of the block for R rows): 75,600 x 5,120 bf16 nvfp4 takes 255 us,
// 3.9 TB/s; a row to a warp, which reads and converts the vectors for every row, 554.
// The values come out of 32-bit arithmetic, so their quotients are not corrected as fp4_divide's: a value within rounding
// of the middle between two codes may take either, with and without the correction (20 million values, nvfp4: 16 and 17 codes other than
// in 64 bits; 32,760 x 5,120: 127 us with it, 113 without).
__host__ __device__ constexpr int mod_threads(int U, int R) { return R == 1 ? 640 : U == 1 ? 384 : 512; }
__host__ __device__ constexpr int mod_regs(int U, int R) { return R == 1 ? 96 : U == 1 ? 80 : 128; }
// The sums of one or two values over the block, in every thread; of two, a half of each warp takes one.
template <int R>
__device__ __forceinline__ void mod_sums(float (&v)[R], float (&to)[R][32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if constexpr (R == 1) {
    v[0] = warp_sum(v[0]);
    if (lane == 0) to[0][warp] = v[0];
    __syncthreads();
    v[0] = warp_sum(lane < warps ? to[0][lane] : 0.f);
  } else {
    const int half = lane >> 4, l = lane & 15;
    float s = (half ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, half ? v[0] : v[1], 16);
#pragma unroll
    for (int d = 8; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (l == 0) to[half][warp] = s;
    __syncthreads();
    s = l < warps ? to[half][l] : 0.f;
#pragma unroll
    for (int d = 8; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float o = __shfl_xor_sync(0xffffffffu, s, 16);
    v[0] = half ? o : s;
    v[1] = half ? s : o;
  }
}
template <typename T, int FMT, bool VEC, int U, int R>
__global__ void __launch_bounds__(mod_threads(U, R), U == 1 ? 2 : 1)
    fp4_modulate_kernel(const T* __restrict__ x, long long x_row, int M, int K, const void* __restrict__ shift,
                        const void* __restrict__ scale, bool wide, float eps, float g, float inv_g, int rows, int pitch, int atoms,
                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr int B = fp4_block(FMT);
  static_assert(R == 1 || mod_threads(U, R) <= 512, "mod_sums: a half warp takes the warps' sums");
  extern __shared__ ulonglong2 vectors[];      // [1 + scale, shift][unit][four columns][thread]
  __shared__ float red[2][R][32];
  const int row0 = blockIdx.x * rows, end = min(row0 + rows, M);
  const float inv_n = 1.f / (float)K;
  grid_release();
  auto column = [&](int u) { return (u * (int)blockDim.x + (int)threadIdx.x) * 16; };
  auto vector = [&](int v, int u, int c) -> ulonglong2& { return vectors[((v * U + u) * 4 + c) * blockDim.x + threadIdx.x]; };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float m[16], s[16];
    load_vector<T, VEC>(scale, wide, column(u), K, m);
    load_vector<T, VEC>(shift, wide, column(u), K, s);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      vector(0, u, c) = make_ulonglong2(pair_of(1.f + m[4 * c], 1.f + m[4 * c + 1]), pair_of(1.f + m[4 * c + 2], 1.f + m[4 * c + 3]));
      vector(1, u, c) = make_ulonglong2(pair_of(s[4 * c], s[4 * c + 1]), pair_of(s[4 * c + 2], s[4 * c + 3]));
    }
  }
  Eight<T> next[R][U][2];
  auto fetch = [&](int row) {      // behind an odd last row: that row again
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u) load_raw<T, VEC>(x + min(row + r, end - 1) * x_row + column(u), K - column(u), next[r][u]);
  };
  fetch(row0);
  for (int row = row0; row < end; row += R) {
    uint64_t y[R][U][8], sum2[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sum2[r] = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[16];
        unpack8(next[r][u][0], f);
        unpack8(next[r][u][1], f + 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[r][u][e] = pair_of(f[2 * e], f[2 * e + 1]);
          sum2[r] = add2(sum2[r], y[r][u][e]);
        }
      }
    }
    if (row + R < end) fetch(row + R);
    float a, b, stat[R];
#pragma unroll
    for (int r = 0; r < R; ++r) pair_to(sum2[r], a, b), stat[r] = a + b;
    mod_sums<R>(stat, red[0]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float mean = stat[r] * inv_n;
      const uint64_t minus = pair_of(-mean, -mean);
      sum2[r] = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[r][u][e] = add2(y[r][u][e], minus);
        if (column(u) + 16 > K) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            pair_to(y[r][u][e], a, b);
            y[r][u][e] = pair_of(column(u) + 2 * e < K ? a : 0.f, column(u) + 2 * e + 1 < K ? b : 0.f);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum2[r] = fma2(y[r][u][e], y[r][u][e], sum2[r]);
      }
      pair_to(sum2[r], a, b);
      stat[r] = a + b;
    }
    mod_sums<R>(stat, red[1]);
#pragma unroll
    for (int r = 0; r < R; ++r) stat[r] = rsqrtf(fmaf(stat[r], inv_n, eps));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = column(u);
#pragma unroll
      for (int c = 0; c < 4; ++c) {      // columns behind the last one: 0
        const ulonglong2 m = vector(0, u, c), s = vector(1, u, c);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint64_t rr = pair_of(stat[r], stat[r]);
          y[r][u][2 * c] = fma2(mul2(y[r][u][2 * c], rr), m.x, s.x);
          y[r][u][2 * c + 1] = fma2(mul2(y[r][u][2 * c + 1], rr), m.y, s.y);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float f[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) pair_to(y[r][u][e], f[2 * e], f[2 * e + 1]);
        put_unit<FMT, false>(f, at < atoms * 4 * B, min(row + r, end - 1), at, pitch, atoms, g, inv_g, codes, scales);
      }
    }
  }
}

// The same for rows that are too long for a block's registers: 256 threads a row, every look reads it again.  WIDE: 32-bit vectors.
template <typename T, int FMT, bool VEC, bool WIDE>
__global__ void __launch_bounds__(256) fp4_modulate_long_kernel(const T* __restrict__ x, long long x_row, int K,
                                                                const void* __restrict__ shift, const void* __restrict__ scale,
                                                                float eps, float g, float inv_g, int pitch, int atoms,
                                                                uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  __shared__ float red[2][8];
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* p = x + row * x_row;
  grid_release();
  float stat[2];      // mean, then the mean square about it
#pragma unroll
  for (int look = 0; look < 2; ++look) {
    const float mean = look ? stat[0] : 0.f;
    float sum = 0.f;
    for (int at = threadIdx.x * 16; at < K; at += 256 * 16) {
      float y[16];
      load16<T, VEC>(p + at, K - at, y);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float d = y[e] - mean;
        if (at + e < K) sum += look ? d * d : d;
      }
    }
    sum = warp_sum(sum);
    if (lane == 0) red[look][warp] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += red[look][w];
    stat[look] = sum / (float)K;
  }
  const float mean = stat[0], r = rsqrtf(stat[1] + eps);
  const int width = atoms * 4 * fp4_block(FMT);
  for (int u = 0; u < width; u += 256 * 16) {
    const int at = u + threadIdx.x * 16;
    float y[16], sc[16], sh[16];
    load16<T, VEC>(p + at, K - at, y);
    load_vector<T, VEC>(scale, WIDE, at, K, sc);
    load_vector<T, VEC>(shift, WIDE, at, K, sh);
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = at + e < K ? fmaf((y[e] - mean) * r, 1.f + sc[e], sh[e]) : 0.f;
    put_unit<FMT, false>(y, at < width, row, at, pitch, atoms, g, inv_g, codes, scales);
  }
}

// A thread writes 32 bytes (16 or 8 elements), a CTA `rows` whole rows.  WIDTH: of its stores (32 or 16).
// 32-byte stores fill whole sectors at once: with 16 bytes at a time 226 us instead of 156 at 75,600 x 5,120 nvfp4, and with a
// block of 32 to a thread 311.
template <typename T, int FMT, int WIDTH>
__global__ void __launch_bounds__(256) fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             int M, int K, float g, int rows, int pitch, int atoms,
                                                             T* __restrict__ out, long long out_row) {
  constexpr int B = fp4_block(FMT), E = 32 / sizeof(T);
  const int row0 = blockIdx.x * rows, end = min(row0 + rows, M);
  for (Walk w(row0, cdiv(K, E)); w.row < end; w.next()) {
    const int at = w.col * E;
    const uint32_t s = scales[fp4_scale_offset(w.row, at / B, atoms)];
    const uint8_t* c = codes + (long long)w.row * pitch + at / 2;
    uint32_t code[E / 8];
    if (E == 16) {
      *reinterpret_cast<uint2*>(code) = *reinterpret_cast<const uint2*>(c);
    } else {
      code[0] = *reinterpret_cast<const uint32_t*>(c);
    }
    const float f = (FMT == T2T_MXFP4 ? e8m0_to_f(s) : e4m3_to_f(s)) * g;
    T* p = out + w.row * out_row + at;
    float y[E];
#pragma unroll
    for (int i = 0; i < E; i += 8) fp4_unpack8(code[i / 8], y + i);
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] *= f;
    if (at + E <= K) {
      Eight<T> v[E / 8];
#pragma unroll
      for (int i = 0; i < E / 8; ++i) v[i] = pack8<T>(y + 8 * i);
      const uint4 lo = v[0].w[0], hi = E == 16 ? v[E / 8 - 1].w[0] : v[0].w[sizeof(T) / 2 - 1];
      if (WIDTH == 32) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "r"(lo.x), "r"(lo.y), "r"(lo.z),
                     "r"(lo.w), "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w)
                     : "memory");
      } else {
        reinterpret_cast<uint4*>(p)[0] = lo;
        reinterpret_cast<uint4*>(p)[1] = hi;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (at + e < K) p[e] = from_f<T>(y[e]);
    }
  }
}

// Rows that are not 16-byte aligned: a thread writes the two elements of a byte, so that neighbouring threads write neighbouring
// elements (16 elements to a thread: 333 us at 37,121 x 1,481 bf16).
template <typename T, int FMT>
__global__ void __launch_bounds__(256) fp4_dequantize_any_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                 int M, int K, float g, int rows, int pitch, int atoms,
                                                                 T* __restrict__ out, long long out_row) {
  constexpr int B = fp4_block(FMT);
  const int row0 = blockIdx.x * rows, end = min(row0 + rows, M);
  for (Walk w(row0, cdiv(K, 2)); w.row < end; w.next()) {
    const int at = w.col * 2;
    const uint32_t s = scales[fp4_scale_offset(w.row, at / B, atoms)];
    const float f = (FMT == T2T_MXFP4 ? e8m0_to_f(s) : e4m3_to_f(s)) * g;
    const uint32_t c = codes[(long long)w.row * pitch + w.col];
    T* p = out + w.row * out_row + at;
    p[0] = from_f<T>(fp4_unpack(c) * f);
    if (at + 1 < K) p[1] = from_f<T>(fp4_unpack(c >> 4) * f);
  }
}

// Whole rows per CTA of 256 threads: about eight blocks a thread where the matrix is large enough to fill the SMs with such CTAs.
static int rows_per_cta(int M, int blocks) {
  const int most = cdiv(8 * 256, blocks), fill = M / (148 * 8);
  return most < fill ? most : (fill > 1 ? fill : 1);
}

// Threads of a block whose threads own U units of 16 columns: whole atoms.
static int mod_block(int K, int fmt, int U) { return cdiv(4 * fp4_atoms(K, fmt) * fp4_block(fmt) / 16, 32 * U) * 32; }

template <typename T, int FMT, bool VEC, int U, int R>
static int modulate_t(const T* x, long long x_row, int M, int K, const void* shift, const void* scale, bool wide, float eps, float g,
                      uint8_t* codes, uint8_t* scales, cudaStream_t st) {
  const int threads = mod_block(K, FMT, U), smem = 2 * U * 4 * threads * 16;
  auto* k = fp4_modulate_kernel<T, FMT, VEC, U, R>;
  static std::atomic<unsigned long long> allowed{0};
  if (!allow_smem(k, 2 * U * 4 * mod_threads(U, R) * 16, allowed)) return T2T_ERR_CUDA;
  // one wave: as many CTAs as registers, shared memory and thread slots of the SMs hold
  const int by_regs = 65536 / (mod_regs(U, R) * threads), by_smem = 224 * 1024 / (smem + 2048), by_slots = 32;
  const int ctas = by_regs < by_smem ? (by_regs < by_slots ? by_regs : by_slots) : (by_smem < by_slots ? by_smem : by_slots);
  const int share = cdiv(M, 148 * (ctas > 1 ? ctas : 1)), rows = share > R ? share : R;
  k<<<cdiv(M, rows), threads, smem, st>>>(x, x_row, M, K, shift, scale, wide, eps, g, 1.f / g, rows, fp4_pitch(K), fp4_atoms(K, FMT),
                                          codes, scales);
  return cudaGetLastError() == cudaSuccess ? T2T_OK : T2T_ERR_CUDA;
}

template <typename T, int FMT>
static int quantize_t(const void* x, long long x_row, int M, int K, const void* shift, const void* scale, bool wide, float eps,
                      float g, uint8_t* codes, uint8_t* scales, cudaStream_t st) {
  const int pitch = fp4_pitch(K), atoms = fp4_atoms(K, FMT);
  const T* p = static_cast<const T*>(x);
  const uintptr_t at = (uintptr_t)x | (uintptr_t)shift | (uintptr_t)scale;
  const bool vec = at % 16 == 0 && x_row * (long long)sizeof(T) % 16 == 0;
  if (shift) {
    // Two rows at a time where 16-bit rows are aligned: 114 us for 32,760 x 5,120 bf16, 122 with one row and two units, 112 with two
    // rows and two units, which at 1,536 columns take 46 against 34.  Longer rows need the second unit (8,000 x 16,384: 92 us, 115 one
    // by one).  32-bit rows do not leave the registers for two (180 us, 168 one by one), nor do the words of unaligned ones
    // (32,759 x 5,119 fp16: 226 and 205).
    if constexpr (sizeof(T) == 2) {
      if (vec && mod_block(K, FMT, 1) <= mod_threads(1, 2))
        return modulate_t<T, FMT, true, 1, 2>(p, x_row, M, K, shift, scale, wide, eps, g, codes, scales, st);
      if (vec && mod_block(K, FMT, 2) <= mod_threads(2, 2))
        return modulate_t<T, FMT, true, 2, 2>(p, x_row, M, K, shift, scale, wide, eps, g, codes, scales, st);
    }
    if (mod_block(K, FMT, 2) <= mod_threads(2, 1)) {
      if (vec) return modulate_t<T, FMT, true, 2, 1>(p, x_row, M, K, shift, scale, wide, eps, g, codes, scales, st);
      return modulate_t<T, FMT, false, 2, 1>(p, x_row, M, K, shift, scale, wide, eps, g, codes, scales, st);
    }
    constexpr bool narrow = sizeof(T) == 2;
    auto* k = wide && narrow ? (vec ? fp4_modulate_long_kernel<T, FMT, true, narrow> : fp4_modulate_long_kernel<T, FMT, false, narrow>)
                             : (vec ? fp4_modulate_long_kernel<T, FMT, true, false> : fp4_modulate_long_kernel<T, FMT, false, false>);
    k<<<M, 256, 0, st>>>(p, x_row, K, shift, scale, eps, g, 1.f / g, pitch, atoms, codes, scales);
  } else {
    const int rows = rows_per_cta(M, atoms * (fp4_block(FMT) / 4));
    auto* k = vec ? fp4_quantize_kernel<T, FMT, true> : fp4_quantize_kernel<T, FMT, false>;
    k<<<cdiv(M, rows), 256, 0, st>>>(p, x_row, M, K, g, 1.f / g, rows, pitch, atoms, codes, scales);
  }
  return cudaGetLastError() == cudaSuccess ? T2T_OK : T2T_ERR_CUDA;
}

template <typename T, int FMT>
static int dequantize_t(const uint8_t* codes, const uint8_t* scales, int M, int K, float g, void* out, long long out_row,
                        cudaStream_t st) {
  const uintptr_t at = (uintptr_t)out | (uintptr_t)(out_row * (long long)sizeof(T));
  const int rows = rows_per_cta(M, at % 16 == 0 ? cdiv(K, 32 / sizeof(T)) : cdiv(K, 2));
  auto* k = at % 32 == 0 ? fp4_dequantize_kernel<T, FMT, 32>
                         : at % 16 == 0 ? fp4_dequantize_kernel<T, FMT, 16> : fp4_dequantize_any_kernel<T, FMT>;
  k<<<cdiv(M, rows), 256, 0, st>>>(codes, scales, M, K, g, rows, fp4_pitch(K), fp4_atoms(K, FMT), static_cast<T*>(out), out_row);
  return cudaGetLastError() == cudaSuccess ? T2T_OK : T2T_ERR_CUDA;
}

// Sizes whose indexes the kernels hold in 32 bits: rows, elements of a row, blocks of threads.
static bool fp4_shape_ok(int M, int K) { return M > 0 && K > 0 && K <= (1 << 24) && M <= (1 << 30); }

}  // namespace t2t

using namespace t2t;

extern "C" size_t t2t_fp4_codes_bytes(int M, int K) { return M > 0 && K > 0 ? (size_t)M * fp4_pitch(K) : 0; }

extern "C" size_t t2t_fp4_scales_bytes(int M, int K, int fmt) {
  return M > 0 && K > 0 && fp4_known(fmt) ? (size_t)cdiv(M, 128) * fp4_atoms(K, fmt) * 512 : 0;
}

extern "C" int t2t_fp4_quantize(const void* x, long long x_row_stride, const void* shift, const void* scale, float eps, int M,
                                int K, int dtype, int fmt, float tensor_scale, void* codes, void* scales, cudaStream_t stream) {
  const bool wide = dtype & T2T_WIDE_VECTORS;
  dtype &= ~T2T_WIDE_VECTORS;
  if (!x || !codes || !scales || !fp4_shape_ok(M, K) || !elem_known(dtype) || !fp4_known(fmt)) return T2T_ERR_ARG;
  if (!shift != !scale || x_row_stride < 0 || (uintptr_t)codes % 16) return T2T_ERR_ARG;
  if (!(tensor_scale >= 0x1p-100f && tensor_scale <= 0x1p100f) || (fmt == T2T_MXFP4 && tensor_scale != 1.f)) return T2T_ERR_ARG;
  uint8_t *c = static_cast<uint8_t*>(codes), *s = static_cast<uint8_t*>(scales);
#define T2T_CALL(T)                                                                                                       \
  return fmt == T2T_MXFP4                                                                                                 \
             ? quantize_t<T, T2T_MXFP4>(x, x_row_stride, M, K, shift, scale, wide, eps, tensor_scale, c, s, stream)             \
             : quantize_t<T, T2T_NVFP4>(x, x_row_stride, M, K, shift, scale, wide, eps, tensor_scale, c, s, stream)
  if (dtype == T2T_BF16) T2T_CALL(__nv_bfloat16);
  if (dtype == T2T_FP16) T2T_CALL(__half);
  T2T_CALL(float);
#undef T2T_CALL
}

extern "C" int t2t_fp4_dequantize(const void* codes, const void* scales, int M, int K, int fmt, float tensor_scale, void* out,
                                  long long out_row_stride, int dtype, cudaStream_t stream) {
  if (!out || !codes || !scales || !fp4_shape_ok(M, K) || !elem_known(dtype) || !fp4_known(fmt)) return T2T_ERR_ARG;
  if (out_row_stride < K || (uintptr_t)codes % 16) return T2T_ERR_ARG;
  const uint8_t *c = static_cast<const uint8_t*>(codes), *s = static_cast<const uint8_t*>(scales);
#define T2T_CALL(T)                                                                                                     \
  return fmt == T2T_MXFP4 ? dequantize_t<T, T2T_MXFP4>(c, s, M, K, tensor_scale, out, out_row_stride, stream)           \
                          : dequantize_t<T, T2T_NVFP4>(c, s, M, K, tensor_scale, out, out_row_stride, stream)
  if (dtype == T2T_BF16) T2T_CALL(__nv_bfloat16);
  if (dtype == T2T_FP16) T2T_CALL(__half);
  T2T_CALL(float);
#undef T2T_CALL
}
