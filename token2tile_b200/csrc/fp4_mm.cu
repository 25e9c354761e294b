// Products of microscaled 4-bit matrices with a fused epilogue:
//
//   out[m, n] = residual[m, n] + gate[n] * act(alpha * sum_k A[m, k] W[n, k] + bias[n])
//
// Sums in 32 bits, one rounding at the end.  The tensor cores read the codes from shared memory (TMA, 128-byte swizzle:
// 256 codes a row) and the scales from tensor memory, where tcgen05.cp puts them atom by atom.
//
// Pairs of CTAs share 256 x 256 tiles (cta_group::2): each holds 128 rows of A and half of the rows of W, 37 KB a stage
// of 256 codes of K with nvfp4.  Pairs are persistent and take tiles in bands of eight row tiles, so that 74 pairs read
// about 8 x 9 of them at a time.  Roles of a CTA: warp 0 copies, warp 1 of the leader issues products, the
// others run the epilogue.
//
// Tensor memory: two accumulators of 256 columns do not fit beside the scales (48 columns), so they overlap by 64:
//   columns 0 .. 255  even tiles, 192 .. 447  odd tiles, 448 .. 495  scales of the stage at hand
// The epilogue reads the 64 common columns first and hands them over; the next tile's products start then and run beside
// the rest of the epilogue.
//
// Bound by the SM's port to L2 (64 bytes a cycle: 608 cycles a step of 256 codes, its products 512) and, in a loop of calls, by power:
// 75,600 x 5,120 x 5,120 nvfp4 with gate and residual takes 950 us, 4,170 TFLOP/s at 1,245 MHz.
#include <cuda.h>

#include "fp4.cuh"
#include "internal.h"

namespace t2t {

struct MmMaps {
  CUtensorMap a, w, sa, sw, out, res;
};

struct MmArgs {
  const void *bias, *gate, *residual;
  void* out;
  long long res_row, out_row;
  int M, N, K, act, vec_dtype;
  bool wide;      // rows of out and residual are 16-byte aligned
  float alpha, out_scale, inv_out_scale;
  uint8_t* out_scales;      // of quantised results
  int* status;
  const void* x;            // A as it is, where the few-rows kernel quantises it
  long long x_row;
  int x_dtype;
  bool x_wide;              // its rows are 16-byte aligned
  int stuck;                // give-up self-test: what never arrives
};
// 1: bytes of the first operands; 2: bytes of the residuals of every CTA's last tile.
enum { MM_STUCK_NONE, MM_STUCK_OPERANDS, MM_STUCK_RESIDUAL };
// Limit of the waits: the self-test's run out within milliseconds.
template <bool GIVE_UP>
__device__ __forceinline__ bool mm_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_wait_warp(bar, parity, abort_flag, GIVE_UP ? 1u << 12 : kWaitSpinLimit);
}

constexpr int MM_TILE = 256;                       // rows and columns of a pair's tile
constexpr int MM_K = 256;                          // codes of K a stage: 128 bytes a row
constexpr int MM_STAGES = 5;
constexpr int MM_HALF = 128 * 128;                 // bytes of 128 rows of codes
// How a pair's results leave: MM_TMA by tiles of 128 rows x 128 bytes, where rows are 16-byte aligned and residuals' rows apart; MM_LANES
// by element, where they are not; MM_CODES quantised.
enum MmEpilogue { MM_TMA, MM_LANES, MM_CODES };
__host__ __device__ constexpr int mm_warps(MmEpilogue e) { return e == MM_TMA ? 8 : 16; }
__host__ __device__ constexpr int mm_threads(MmEpilogue e) { return 32 * (2 + mm_warps(e)); }
constexpr int MM_OVERLAP = 64;
constexpr int MM_ACC1 = MM_TILE - MM_OVERLAP;      // first column of the odd tiles' accumulator
constexpr int MM_SFA = MM_ACC1 + MM_TILE;          // scales of A: 4 columns an atom
constexpr int MM_SFB = MM_SFA + 16;                // of W: 8 columns an atom
__host__ __device__ constexpr int mm_stage_atoms(int fmt) { return MM_K / (4 * fp4_block(fmt)); }
__host__ __device__ constexpr int mm_stage_bytes(int fmt) { return 2 * MM_HALF + 3 * mm_stage_atoms(fmt) * 512; }
constexpr int MM_STAGING = 2 * 16 * 1024;          // results (and residuals) on their way
constexpr int MM_VECTORS = 2 * 2 * 256 * 4;        // bias and gate of a tile's columns, in 32 bits; two tiles in turn
enum { MB_FULL = 0, MB_EMPTY = MM_STAGES, MB_ACC = 2 * MM_STAGES, MB_DRAINED = MB_ACC + 2, MB_RES, MB_COUNT = MB_RES + 2 };
__host__ __device__ constexpr int mm_smem(int fmt) {
  return MM_STAGES * mm_stage_bytes(fmt) + MM_STAGING + MB_COUNT * 8 + 16 + 1024;
}
// MM_CODES keeps the vectors where the others stage their results, MM_TMA (one tile's) behind its barriers.
__host__ __device__ constexpr int mm_smem(int fmt, MmEpilogue e) { return mm_smem(fmt) + (e == MM_TMA ? MM_VECTORS / 2 + 16 : 0); }
static_assert(mm_smem(T2T_NVFP4, MM_TMA) <= 227 * 1024, "shared memory of an SM");
static_assert(MM_SFB + 32 <= 512, "tensor memory");

// ---- block-scaled products ------------------------------------------------------
// Instruction descriptor: E2M1 x E2M1 -> fp32, scales E8M0 (mxfp4) or E4M3 (nvfp4); `id` is the byte of a scale word that
// the product's first block is in (0 or 2: two of an atom's four blocks make 64 codes of mxfp4).
__host__ __device__ constexpr uint32_t mm_idesc(int fmt, int M, int N, int id) {
  return ((uint32_t)id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (fmt == T2T_MXFP4 ? 1u << 23 : 0u) |
         ((uint32_t)(M >> 4) << 24) | ((uint32_t)id << 29);
}
// Descriptor of an atom of scales (512 contiguous bytes, no swizzle): 8-lane groups 128 bytes apart.
__device__ __forceinline__ uint64_t mm_scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(128u >> 4) << 32) | (1ull << 46);
}
__device__ __forceinline__ void scales_to_tmem_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(desc) : "memory");
}
template <int FMT>
__device__ __forceinline__ void mm_product_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                                uint32_t accumulate) {
  if (FMT == T2T_MXFP4)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tma_load_tile3_pair(uint32_t dst, const void* map, int col, int row, int slab, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(row), "r"(slab), "r"(bar)
      : "memory");
}

// ---- epilogue ---------------------------------------------------------------------
// tanh(u) = 2 / (1 + exp(-2 u)) - 1, so both activations are x / (1 + 2^-z).  ex2 and rcp are good to 2^-22; z, of a few
// tens at most where the result is not x or 0, adds 2^-20 at worst.  Large arguments: z overflows to an infinity of the right sign
// and the result is x or -0.  GELU's x^2 may overflow in it; SiLU has no such term (times a factor of 0 it would be a NaN).
template <int ACT, int n>
__device__ __forceinline__ void mm_act_of(float (&y)[n]) {
  constexpr float log2e = 1.4426950408889634f, c1 = ACT == T2T_ACT_SILU ? -log2e : -1.5957691216057308f * log2e,
                  c3 = 0.044715f * -1.5957691216057308f * log2e;
  const uint64_t k1 = pair_of(c1, c1), k3 = pair_of(c3, c3), one = pair_of(1.f, 1.f);
#pragma unroll
  for (int e = 0; e < n; e += 2) {
    const uint64_t x = pair_of(y[e], y[e + 1]);
    float p, q;
    pair_to(mul2(x, ACT == T2T_ACT_SILU ? k1 : fma2(k3, mul2(x, x), k1)), p, q);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(p));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(q));
    pair_to(add2(pair_of(p, q), one), p, q);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(p));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(q));
    pair_to(mul2(x, pair_of(p, q)), y[e], y[e + 1]);
  }
}
template <int n>
__device__ __forceinline__ void mm_act(float (&y)[n], int act) {
  if (act == T2T_ACT_GELU_TANH) mm_act_of<T2T_ACT_GELU_TANH>(y);
  else if (act == T2T_ACT_SILU) mm_act_of<T2T_ACT_SILU>(y);
}
// y * a + b, by pairs.
template <int n>
__device__ __forceinline__ void mm_affine(float (&y)[n], float a, const float (&b)[n]) {
  const uint64_t aa = pair_of(a, a);
#pragma unroll
  for (int e = 0; e < n; e += 2) pair_to(fma2(pair_of(y[e], y[e + 1]), aa, pair_of(b[e], b[e + 1])), y[e], y[e + 1]);
}

// 32 accumulator columns of a row in one thread: y = gate * act(alpha * v + bias).  The vectors lie in shared memory; every lane reads
// the same.
__device__ __forceinline__ void mm_row(const MmArgs& p, const uint32_t (&v)[32], const float* bias, const float* gate, float (&y)[32]) {
  const uint64_t alpha = pair_of(p.alpha, p.alpha);
#pragma unroll
  for (int e = 0; e < 32; e += 4) {
    const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(bias + e);
    pair_to(fma2(pair_of(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), alpha, b.x), y[e], y[e + 1]);
    pair_to(fma2(pair_of(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), alpha, b.y), y[e + 2], y[e + 3]);
  }
  mm_act(y, p.act);
  if (p.gate) {
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      const ulonglong2 g = *reinterpret_cast<const ulonglong2*>(gate + e);
      pair_to(mul2(pair_of(y[e], y[e + 1]), g.x), y[e], y[e + 1]);
      pair_to(mul2(pair_of(y[e + 2], y[e + 3]), g.y), y[e + 2], y[e + 3]);
    }
  }
}

// MM_TMA: 32 results of row `row` into a tile of 128-byte rows (128-byte swizzle) from 16-byte chunk `c`, on top of the residuals that lie
// there.
template <typename T>
__device__ __forceinline__ void mm_to_tile(const MmArgs& p, float (&y)[32], uint8_t* tile, int row, int c) {
  constexpr int V = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    Eight<T> r;
    uint4* at[sizeof(T) / 2];
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) at[j] = reinterpret_cast<uint4*>(tile + sw128(row, c + i / V + j));
    if (p.residual) {
      float z[8];
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; ++j) r.w[j] = *at[j];
      unpack8(r, z);
#pragma unroll
      for (int e = 0; e < 8; e += 2) pair_to(add2(pair_of(y[i + e], y[i + e + 1]), pair_of(z[e], z[e + 1])), y[i + e], y[i + e + 1]);
    }
    r = pack8<T>(y + i);
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) *at[j] = r.w[j];
  }
}
__device__ __forceinline__ void tma_store_tile(const void* map, int col, int row, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(col), "r"(row), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
}
__device__ __forceinline__ void tma_prefetch_tile(const void* map, int col, int row) {      // into L2
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(col),
               "r"(row)
               : "memory");
}
template <bool READ>      // this thread's stores have read their shared memory, or have landed
__device__ __forceinline__ void tma_store_wait() {
  if (READ) asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
  else asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
}
// The four warps of an epilogue group; every one of them comes here as often as the others, whatever its waits have answered.
__device__ __forceinline__ void mm_meet(int group) { asm volatile("bar.sync %0, 128;\n" ::"r"(group + 1) : "memory"); }

// MM_LANES: 16 columns of a warp's 32 rows through shared memory, so that a lane takes one column and walks down the rows: neighbouring
// lanes write neighbouring elements.  16-byte chunk c of row r lies at c ^ (r / 2 % 4) of its 64 bytes.
template <typename T>
__device__ __forceinline__ void mm_lanes(const MmArgs& p, const uint32_t (&v)[16], uint8_t* staging, int m0, int n0) {
  constexpr int C = 16;
  const int lane = threadIdx.x & 31;
  auto at = [&](int r, int c) { return reinterpret_cast<float4*>(staging + r * (C * 4) + ((c ^ (r >> 1 & 3)) << 4)); };
#pragma unroll
  for (int c = 0; c < C / 4; ++c)
    *at(lane, c) = make_float4(__uint_as_float(v[4 * c]), __uint_as_float(v[4 * c + 1]), __uint_as_float(v[4 * c + 2]),
                               __uint_as_float(v[4 * c + 3]));
  const int col = n0 + lane % C;
  const bool on = col < p.N;
  const float bias = p.bias && on ? load_elem(p.bias, col, p.vec_dtype) : 0.f;
  const float gate = p.gate && on ? load_elem(p.gate, col, p.vec_dtype) : 1.f;
  __syncwarp();
#pragma unroll 1
  for (int r0 = lane / C; r0 < 32; r0 += 8 * (32 / C)) {      // eight rows' residuals before the first store, which may overwrite them
    float y[8];
    bool row[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + i * (32 / C);
      row[i] = on && m0 + r < p.M;
      y[i] = p.residual && row[i] ? to_f(static_cast<const T*>(p.residual)[(m0 + r) * p.res_row + col]) : 0.f;
    }
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      z[i] = fmaf(reinterpret_cast<const float*>(at(r0 + i * (32 / C), lane % C >> 2))[lane & 3], p.alpha, bias);
    mm_act(z, p.act);
#pragma unroll
    for (int i = 0; i < 8; ++i) {      // as MM_TMA: a zero keeps its sign, and the residual is added to the rounded product
      z[i] = __fmul_rn(z[i], gate);
      if (p.residual) z[i] = __fadd_rn(z[i], y[i]);
      if (row[i]) static_cast<T*>(p.out)[(m0 + r0 + i * (32 / C)) * p.out_row + col] = from_f<T>(z[i]);
    }
  }
  __syncwarp();
}

// MM_CODES: 32 columns of row m, one or two whole blocks, to codes and scales.
template <int FMT>
__device__ __forceinline__ void mm_codes(const MmArgs& p, float (&y)[32], int m, int n0) {
  constexpr int B = fp4_block(FMT);
  const int pitch = fp4_pitch(p.N), atoms = fp4_atoms(p.N, FMT);
  if (n0 + 32 > p.N) {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (n0 + e >= p.N) y[e] = 0.f;
  }
  uint32_t s[32 / B];
#pragma unroll
  for (int b = 0; b < 32 / B; ++b) {
    float inv, eff;
    const float top = fp4_top<B>(y + b * B);
    s[b] = fp4_scale<FMT>(top, p.out_scale, p.inv_out_scale, inv, eff);
    fp4_divide<FMT, B>(y + b * B, top, inv, eff);
  }
  if (m >= p.M) return;
  uint8_t* to = p.out_scales + fp4_scale_offset(m, n0 / B, atoms);
  if (n0 / B < 4 * atoms) {
    if (FMT == T2T_MXFP4) *to = (uint8_t)s[0];
    else *reinterpret_cast<unsigned short*>(to) = (unsigned short)(s[0] | s[32 / B - 1] << 8);
  }
  if (n0 / 2 < pitch)
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + (long long)m * pitch + n0 / 2) =
        make_uint4(fp4_pack8(y), fp4_pack8(y + 8), fp4_pack8(y + 16), fp4_pack8(y + 24));
}

// Tile number -> first row and column: bands of eight row tiles, all column tiles of a band before the next.
__device__ __forceinline__ void mm_tile(int tile, int mt, int nt, int& m0, int& n0) {
  constexpr int BAND = 8;
  const int band = tile / (BAND * nt), first = band * BAND, rows = min(BAND, mt - first), at = tile - band * BAND * nt;
  m0 = (first + at % rows) * MM_TILE;
  n0 = at / rows * MM_TILE;
}

// Behind a barrier of the CTA after its last wait: reports one that gave up, and lets copies still in flight land before the shared memory
// is released.
__device__ __forceinline__ void mm_gave_up(const MmArgs& p, volatile int* abort_flag) {
  if (*abort_flag) {
    if (threadIdx.x == 0 && p.status) *reinterpret_cast<volatile int*>(p.status) = ST_WAIT_TIMEOUT;
    for (int i = 0; i < 100; ++i) __nanosleep(1000);
  }
  __syncwarp();
}

template <int FMT, typename T, MmEpilogue EPI, bool GIVE_UP = false>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(mm_threads(EPI), 1)
    fp4_mm_pair_kernel(const __grid_constant__ MmMaps maps, const MmArgs p) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int STAGE = mm_stage_bytes(FMT), ATOMS = mm_stage_atoms(FMT), WARPS = mm_warps(EPI);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - smem_u32(smem_raw));
  // codes of all stages and staged results first (1024-byte aligned tiles), then scales and barriers
  constexpr int OFF_STAGING = MM_STAGES * 2 * MM_HALF, OFF_SCALES = OFF_STAGING + MM_STAGING, OFF_BARS = MM_STAGES * STAGE + MM_STAGING;
  const uint32_t s_scales = base + OFF_SCALES;
  uint8_t* staging = sm + OFF_STAGING;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + OFF_BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + MB_COUNT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* vectors = reinterpret_cast<float*>(EPI == MM_TMA ? sm + (OFF_BARS + MB_COUNT * 8 + 16 + 15) / 16 * 16 : staging);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();

  if (warp == 0) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  if (tid == 0) {
    *abort_flag = 0;
    for (int i = 0; i < MB_COUNT; ++i) mbar_init(bars + i, i == MB_DRAINED ? 2 * WARPS : 1);
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  grid_release();
  grid_wait();
  cluster_sync();      // both CTAs' barriers exist
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t lead = cluster_addr(smem_u32(bars), 0);

  const int mt = cdiv(p.M, MM_TILE), nt = cdiv(p.N, MM_TILE), tiles = mt * nt, steps = cdiv(p.K, MM_K);
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

  if (warp == 0) {
    // ================= copies =================
    uint32_t it = 0;
    bool ok = true;
    for (int tile = first; ok && tile < tiles; tile += stride) {
      int m0, n0;
      mm_tile(tile, mt, nt, m0, n0);
      for (int k = 0; k < steps; ++k, ++it) {
        const uint32_t s = it % MM_STAGES;
        ok = it < MM_STAGES || mm_wait<GIVE_UP>(bars + MB_EMPTY + s, (it / MM_STAGES - 1u) & 1u, abort_flag);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t full = lead + (MB_FULL + s) * 8, codes = base + s * 2 * MM_HALF, sc = s_scales + s * 3 * ATOMS * 512;
          if (rank == 0) mbar_arrive_expect_tx(bars + MB_FULL + s, 2 * STAGE + (GIVE_UP && p.stuck == MM_STUCK_OPERANDS && it == 0 ? 16 : 0));
          tma_load_tile_pair(codes, &maps.a, k * 128, m0 + (int)rank * 128, full);
          tma_load_tile_pair(codes + MM_HALF, &maps.w, k * 128, n0 + (int)rank * 128, full);
          tma_load_tile3_pair(sc, &maps.sa, 0, k * ATOMS, m0 / 128 + (int)rank, full);
          tma_load_tile3_pair(sc + ATOMS * 512, &maps.sw, 0, k * ATOMS, n0 / 128, full);
        }
        __syncwarp();
      }
    }
    // the products that read the last stages have arrived here too before this CTA leaves
    for (uint32_t i = it < MM_STAGES ? 0 : it - MM_STAGES; ok && i < it; ++i)
      ok = mm_wait<GIVE_UP>(bars + MB_EMPTY + i % MM_STAGES, (i / MM_STAGES) & 1u, abort_flag);
  } else if (warp == 1 && rank == 0) {
    // ================= products =================
    constexpr uint32_t dhi = sdesc_hi(1024);
    uint32_t it = 0, n = 0;
    bool ok = true;
    for (int tile = first; tile < tiles; tile += stride, ++n) {
      // the epilogue has read the columns that this tile shares with the one before (and all of the one before that)
      if (n > 0 && !mm_wait<GIVE_UP>(bars + MB_DRAINED, (n - 1u) & 1u, abort_flag)) break;
      tc_fence_after();
      const uint32_t acc = tmem + (n & 1u) * MM_ACC1;
      for (int k = 0; k < steps; ++k, ++it) {
        const uint32_t s = it % MM_STAGES;
        ok = mm_wait<GIVE_UP>(bars + MB_FULL + s, (it / MM_STAGES) & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t codes = base + s * 2 * MM_HALF, sc = s_scales + s * 3 * ATOMS * 512;
          // products and copies of one thread run in the order of their issue, so the columns are written after the products
          // of the stage before have read them
#pragma unroll
          for (int j = 0; j < ATOMS; ++j) {
            scales_to_tmem_pair(tmem + MM_SFA + j * 4, mm_scale_desc(sc + j * 512));
            scales_to_tmem_pair(tmem + MM_SFB + j * 8, mm_scale_desc(sc + (ATOMS + j) * 512));
            scales_to_tmem_pair(tmem + MM_SFB + j * 8 + 4, mm_scale_desc(sc + (2 * ATOMS + j) * 512));
          }
          const uint32_t alo = sdesc_lo(codes, 16), blo = sdesc_lo(codes + MM_HALF, 16);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int j = FMT == T2T_MXFP4 ? q >> 1 : q, id = FMT == T2T_MXFP4 ? (q & 1) * 2 : 0;
            mm_product_pair<FMT>(acc, ((uint64_t)dhi << 32) | (alo + q * 2), ((uint64_t)dhi << 32) | (blo + q * 2),
                                 mm_idesc(FMT, MM_TILE, MM_TILE, id), tmem + MM_SFA + j * 4, tmem + MM_SFB + j * 8,
                                 k + q > 0 ? 1u : 0u);
          }
          umma_commit_pair(bars + MB_EMPTY + s);
          if (k + 1 == steps) umma_commit_pair(bars + MB_ACC + (n & 1u));
        }
        __syncwarp();
      }
      if (!ok) break;
    }
  } else if (warp >= 2) {
    // ================= epilogue =================
    // A warp reads the 32 lanes of its number modulo 4; the four warps of a group share columns.  The common columns come first.
    const int ew = warp - 2, quad = warp & 3, group = ew >> 2, row = quad * 32 + lane;
    uint32_t n = 0, loads = 0;
    bool ok = true;
    for (int tile = first; tile < tiles; tile += stride, ++n) {
      int m0, n0;
      mm_tile(tile, mt, nt, m0, n0);
      const int rows0 = m0 + (int)rank * 128;
      const bool odd = n & 1u;
      const uint32_t acc = tmem_addr(tmem + (n & 1u) * MM_ACC1, quad * 32, 0);
      auto wait_acc = [&] {
        ok = ok && mm_wait<GIVE_UP>(bars + MB_ACC + (n & 1u), (n >> 1) & 1u, abort_flag);
        tc_fence_after();
      };
      auto drained = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_peer(lead + MB_DRAINED * 8);
      };
      auto vector = [&](const void* v, int col, float fill) { return v && col < p.N ? load_elem(v, col, p.vec_dtype) : fill; };
      if constexpr (EPI == MM_TMA) {
        // tiles of 128 bytes of columns, every second one each group's: of an even tile the last 64 columns are common, of an odd one the
        // first.  A group's tile in shared memory takes the residuals and, in their place, the results.
        constexpr int SUB = 128 / sizeof(T), PER = 128 / SUB;
        auto sub = [&](int i) { return (odd ? 2 * i + group : 2 * (PER - 1 - i) + group) * SUB; };
        uint8_t* buffer = staging + group * 16384;
        float *bias = vectors + group * 128, *gate = vectors + 256 + group * 128;
        bias[row] = vector(p.bias, n0 + sub(row / SUB) + row % SUB, 0.f);
        gate[row] = vector(p.gate, n0 + sub(row / SUB) + row % SUB, 1.f);
        if (row == 0 && p.residual && tile + stride < tiles) {      // the next tile's residuals are in L2 when they are asked for
          int m1, n1;
          mm_tile(tile + stride, mt, nt, m1, n1);
          m1 += (int)rank * 128;
          for (int i = 0; i < PER; ++i)
            if (m1 < p.M && n1 + (2 * i + group) * SUB < p.N) tma_prefetch_tile(&maps.res, n1 + (2 * i + group) * SUB, m1);
        }
        __syncwarp();
#pragma unroll 1
        for (int i = 0; i < PER; ++i) {
          const int col = n0 + sub(i);
          const bool there = rows0 < p.M && col < p.N;
          if (row == 0) {
            tma_store_wait<true>();      // the tile before has left the buffer
            if (p.residual && there && ok) {
              const bool stuck = GIVE_UP && p.stuck == MM_STUCK_RESIDUAL && tile + stride >= tiles && i + 1 == PER;
              mbar_arrive_expect_tx(bars + MB_RES + group, 16384 + (stuck ? 16 : 0));
              tma_load_tile(smem_u32(buffer), &maps.res, col, rows0, bars + MB_RES + group);
            }
          }
          __syncwarp();
          if (i == 0) wait_acc();
          uint32_t v[SUB / 32][32];
          if (ok) {
#pragma unroll
            for (int q = 0; q < SUB / 32; ++q) tmem_ld32(acc + sub(i) + q * 32, v[q]);
            tmem_wait_ld();
          }
          if (i == 0) drained();
          mm_meet(group);
          if (p.residual && there) {
            ok = ok && mm_wait<GIVE_UP>(bars + MB_RES + group, loads & 1u, abort_flag);
            ++loads;
          }
          if (ok && there) {
#pragma unroll
            for (int q = 0; q < SUB / 32; ++q) {
              float y[32];
              mm_row(p, v[q], bias + i * SUB + q * 32, gate + i * SUB + q * 32, y);
              mm_to_tile<T>(p, y, buffer, row, q * 4);
            }
            fence_proxy_async();
          }
          mm_meet(group);
          if (row == 0 && ok && there) tma_store_tile(&maps.out, col, rows0, smem_u32(buffer));
        }
      } else if constexpr (EPI == MM_CODES) {
        // chunks of 32 columns, two a warp: 6, 7 of an even tile are common, 0, 1 of an odd one; groups 2 and 3 have none
        auto chunk = [&](int i) {
          return (group < 2 ? (odd ? group + 2 * i : group + 6 * (1 - i)) : 2 * group - (odd ? 0 : 2) + i) * 32;
        };
        float *bias = vectors + (n & 1u) * 512 + group * 64, *gate = bias + 256;
        if (row < 64) bias[row] = vector(p.bias, n0 + chunk(row >> 5) + (row & 31), 0.f);
        else gate[row - 64] = vector(p.gate, n0 + chunk((row - 64) >> 5) + (row & 31), 1.f);
        mm_meet(group);      // two tiles' vectors in turn: nobody is more than one meeting behind
        wait_acc();
#pragma unroll 1
        for (int i = 0; i < 2 && ok; ++i) {
          uint32_t v[32];
          tmem_ld32(acc + chunk(i), v);
          tmem_wait_ld();
          if (i == 0) drained();
          if (rows0 + quad * 32 >= p.M) continue;
          float y[32];
          mm_row(p, v, bias + i * 32, gate + i * 32, y);
          mm_codes<FMT>(p, y, rows0 + row, n0 + chunk(i));
        }
      } else {
        // chunks of 16 columns, four a warp: 12 .. 15 of an even tile are common, 0 .. 3 of an odd one
        auto chunk = [&](int i) { return (i == 0 ? group + (odd ? 0 : 12) : group * 3 + i - 1 + (odd ? 4 : 0)) * 16; };
        wait_acc();
#pragma unroll 1
        for (int i = 0; i < 4 && ok; ++i) {
          uint32_t v[16];
          tmem_ld16(acc + chunk(i), v);
          tmem_wait_ld();
          if (i == 0) drained();
          if (rows0 + quad * 32 < p.M) mm_lanes<T>(p, v, staging + ew * 2048, rows0 + quad * 32, n0 + chunk(i));
        }
      }
    }
    if (EPI == MM_TMA && row == 0) tma_store_wait<false>();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();      // every wait of the CTA has ended, those for the last residuals too
  mm_gave_up(p, abort_flag);
  cluster_sync();      // the other CTA no longer arrives here, and both are done with tensor memory
  if (warp == 0) tmem_dealloc_pair(tmem, 512);
}

// ---- few rows ---------------------------------------------------------------------------
// With few rows of A the product is bound by reading W, and by latency.  The operands change sides: 128 rows of W fill the
// tensor core's rows and the rows of A, T of them (16 to 128, the next power of two), are its columns, so one row costs no
// more than sixteen.  Where the slabs of W are fewer than the SMs hold CTAs, a cluster splits K between up to four of them and
// adds their sums up over distributed shared memory in the order of their ranks.  CTAs of up to 32 columns leave room for
// two on an SM.
// A step of 256 codes takes 0.28 us whatever T is: its four products, 125 cycles each down to 16 columns, follow one another
// (without the copies of the scales 0.26; with nine steps in flight instead of four 0.28).  1 x 30,720 x 5,120 nvfp4 takes
// 15.8 us (5.6 TB/s), 1 x 5,120 x 5,120 6.0, of which 4 are the launch and the first step's way through memory.
constexpr int MR_THREADS = 192;      // warps: copies, products, four that bring the sums to shared memory
__host__ __device__ constexpr int mr_stage_bytes(int fmt, int T) { return MM_HALF + T * 128 + 2 * mm_stage_atoms(fmt) * 512; }
__host__ __device__ constexpr int mr_stages(int T) { return T <= 32 ? 4 : 5; }
__host__ __device__ constexpr int mr_smem(int fmt, int T) { return mr_stages(T) * mr_stage_bytes(fmt, T) + 128 + 1024; }
__host__ __device__ constexpr int mr_columns(int T) { return T + 32 <= 64 ? 64 : T + 32 <= 128 ? 128 : 256; }
static_assert(2 * (mr_smem(T2T_NVFP4, 32) + 1024) <= 228 * 1024, "two CTAs on an SM");
static_assert(mr_smem(T2T_NVFP4, 128) <= 227 * 1024 && 128 * 128 * 4 <= mr_stages(128) * mr_stage_bytes(T2T_MXFP4, 128), "");

__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(desc) : "memory");
}
template <int FMT>
__device__ __forceinline__ void mm_product(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                           uint32_t accumulate) {
  if (FMT == T2T_MXFP4)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ float4 cluster_load4(uint32_t caddr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(caddr));
  return v;
}

// Four neighbouring elements of a vector or row; `fill` behind its end.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int left, float fill, float (&y)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = e < left ? to_f(p[e]) : fill;
}
__device__ __forceinline__ void load4(const void* p, int n, int N, int dtype, float fill, float (&y)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = p && n + e < N ? load_elem(p, n + e, dtype) : fill;
}

// Columns n .. n + 3 of row m, the whole warp.
template <int FMT, typename T>
__device__ __forceinline__ void mr_finish(const MmArgs& p, int m, int n, float (&y)[4], const float (&bias)[4], const float (&gate)[4]) {
  mm_affine(y, p.alpha, bias);
  mm_act(y, p.act);
  if (p.gate) {
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= gate[e];
  }
  if constexpr (std::is_same<T, uint8_t>::value) {
    constexpr int B = fp4_block(FMT);      // in four or eight lanes
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e >= p.N) y[e] = 0.f;
    float top = fp4_top<4>(y), inv, eff;
#pragma unroll
    for (int d = 1; d < B / 4; d <<= 1) top = fp4_max(top, __shfl_xor_sync(0xffffffffu, top, d));
    const uint32_t s = fp4_scale<FMT>(top, p.out_scale, p.inv_out_scale, inv, eff);
    const int pitch = fp4_pitch(p.N), atoms = fp4_atoms(p.N, FMT);
    if ((n & (B - 1)) == 0 && n / B < 4 * atoms) p.out_scales[fp4_scale_offset(m, n / B, atoms)] = (uint8_t)s;
    if (n / 2 >= pitch) return;
    fp4_divide<FMT, 4>(y, top, inv, eff);
    const float z[8] = {y[0], y[1], y[2], y[3], 0.f, 0.f, 0.f, 0.f};
    *reinterpret_cast<unsigned short*>(static_cast<uint8_t*>(p.out) + (long long)m * pitch + n / 2) = (unsigned short)fp4_pack8(z);
  } else {
    if (n >= p.N) return;
    if (p.residual) {
      float r[4];
      load4(static_cast<const T*>(p.residual) + m * p.res_row + n, p.N - n, 0.f, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += r[e];
    }
    T* out = static_cast<T*>(p.out) + m * p.out_row + n;
    if (p.wide && n + 4 <= p.N) {
      Vec<T, 4> v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v.e[e] = from_f<T>(y[e]);
      store_vec<T, 4>(out, v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) out[e] = from_f<T>(y[e]);
    }
  }
}

// Up to T2T_FP4_FEW_ROWS rows of A that are not quantised yet: the four warps that wait for the sums do it, a step to a warp in turn and
// 16 elements to a lane.  The codes and scales are those of the quantisation on its own.  They run beside the
// copies of W: 4 x 5,120 x 5,120 nvfp4 takes 5.9 us like this, 6.0 from codes and 7.7 with the quantisation as a launch of its own (one
// row 5.7, 6.2 and 7.3).  Sixteen rows fell behind the products (11.6 us, 8.8 in two launches).
template <int FMT, int STAGES, typename X, bool GIVE_UP>
__device__ __forceinline__ void mr_quantize(const MmArgs& p, int w, int first, int last, uint8_t* codes, int codes_stage, uint8_t* scales,
                                            int scales_stage, uint64_t* full, uint64_t* empty, volatile int* abort_flag) {
  constexpr int B = fp4_block(FMT), ATOMS = mm_stage_atoms(FMT), UNITS = MM_K / 16, ROWS = 32 / UNITS, LOOKS = T2T_FP4_FEW_ROWS / ROWS;
  const int lane = threadIdx.x & 31, unit = lane % UNITS, row0 = lane / UNITS;
  const X* x = static_cast<const X*>(p.x);
  for (int k = first + w; k < last; k += 4) {
    const uint32_t it = k - first, s = it % STAGES;
    const int at = k * MM_K + unit * 16;
    Eight<X> raw[LOOKS][2];
#pragma unroll
    for (int j = 0; j < LOOKS; ++j) {
      const int row = row0 + j * ROWS, left = row < p.M ? p.K - at : 0;
      const X* q = x + (row < p.M ? row : 0) * p.x_row + at;
      if (p.x_wide) load_raw<X, true>(q, left, raw[j]);
      else load_raw<X, false>(q, left, raw[j]);
    }
    if (it >= STAGES && !mm_wait<GIVE_UP>(empty + s, (it / STAGES - 1u) & 1u, abort_flag)) return;
#pragma unroll
    for (int j = 0; j < LOOKS; ++j) {
      if (j * ROWS >= p.M) break;
      const int row = row0 + j * ROWS;
      float y[16];
      uint32_t word;
      unpack8(raw[j][0], y);
      unpack8(raw[j][1], y + 8);
      const uint2 c = fp4_unit<FMT, true>(y, 1.f, 1.f, word);
      if (row < p.M) {
        *reinterpret_cast<uint2*>(codes + s * codes_stage + sw128(row, unit / 2) + unit % 2 * 8) = c;
        if (unit * 16 % (4 * B) == 0)
          *reinterpret_cast<uint32_t*>(scales + s * scales_stage + fp4_scale_offset(row, unit * 16 / B, ATOMS)) = word;
      }
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(full + s);
    __syncwarp();
  }
}

// Grid: (splits x slabs of 128 rows of W, tiles of T rows of A); clusters of `splits` CTAs.  X: void, or the type of an A that is quantised
// here (one tile of rows).
template <int FMT, int T, typename OUT, typename X, bool GIVE_UP = false>
__global__ void __launch_bounds__(MR_THREADS) fp4_mm_rows_kernel(const __grid_constant__ MmMaps maps, const MmArgs p, int splits) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int STAGES = mr_stages(T), STAGE = mr_stage_bytes(FMT, T), ATOMS = mm_stage_atoms(FMT), COLUMNS = mr_columns(T);
  constexpr bool QUANTIZE = !std::is_same<X, void>::value;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t s_rows = base + STAGES * MM_HALF, s_scales = s_rows + STAGES * T * 128;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + STAGES * STAGE);      // full, empty, sums
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = splits > 1 ? (int)cluster_rank() : 0, n0 = (int)blockIdx.x / splits * 128, m0 = (int)blockIdx.y * T;
  const int steps = cdiv(p.K, MM_K), first = steps * rank / splits, last = steps * (rank + 1) / splits;

  if (warp == 0) {
    tmem_alloc(tmem_slot, COLUMNS);
    tmem_relinquish();
  }
  if (tid == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 2 * STAGES + 1; ++i) mbar_init(bars + i, QUANTIZE && i < STAGES ? 2 : 1);
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  grid_release();
  grid_wait();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, sfa = tmem + T, sfb = tmem + T + 16;

  if (warp == 0) {
    for (int k = first; k < last; ++k) {
      const uint32_t it = k - first, s = it % STAGES;
      if (it >= STAGES && !mm_wait<GIVE_UP>(bars + STAGES + s, (it / STAGES - 1u) & 1u, abort_flag)) break;
      if (elect_one()) {
        uint64_t* full = bars + s;
        const uint32_t sc = s_scales + s * 2 * ATOMS * 512;
        const int stuck = GIVE_UP && p.stuck == MM_STUCK_OPERANDS && it == 0 ? 16 : 0;
        mbar_arrive_expect_tx(full, (QUANTIZE ? MM_HALF + ATOMS * 512 : STAGE) + stuck);
        tma_load_tile(base + s * MM_HALF, &maps.w, k * 128, n0, full);
        tma_load_tile3(sc, &maps.sw, 0, k * ATOMS, n0 / 128, full);
        if (!QUANTIZE) {
          tma_load_tile(s_rows + s * T * 128, &maps.a, k * 128, m0, full);
          tma_load_tile3(sc + ATOMS * 512, &maps.sa, 0, k * ATOMS, m0 / 128, full);
        }
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    constexpr uint32_t dhi = sdesc_hi(1024);
    for (int k = first; k < last; ++k) {
      const uint32_t it = k - first, s = it % STAGES;
      if (!mm_wait<GIVE_UP>(bars + s, (it / STAGES) & 1u, abort_flag)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t sc = s_scales + s * 2 * ATOMS * 512;
#pragma unroll
        for (int j = 0; j < ATOMS; ++j) {
          scales_to_tmem(sfa + j * 4, mm_scale_desc(sc + j * 512));
          scales_to_tmem(sfb + j * 4, mm_scale_desc(sc + (ATOMS + j) * 512));
        }
        const uint32_t alo = sdesc_lo(base + s * MM_HALF, 16), blo = sdesc_lo(s_rows + s * T * 128, 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int j = FMT == T2T_MXFP4 ? q >> 1 : q, id = FMT == T2T_MXFP4 ? (q & 1) * 2 : 0;
          mm_product<FMT>(tmem, ((uint64_t)dhi << 32) | (alo + q * 2), ((uint64_t)dhi << 32) | (blo + q * 2),
                          mm_idesc(FMT, 128, T, id), sfa + j * 4, sfb + j * 4, it + q > 0 ? 1u : 0u);
        }
        umma_commit(bars + STAGES + s);
        if (k + 1 == last) umma_commit(bars + 2 * STAGES);
      }
      __syncwarp();
    }
  } else if constexpr (QUANTIZE) {
    mr_quantize<FMT, STAGES, X, GIVE_UP>(p, warp - 2, first, last, sm + (s_rows - base), T * 128, sm + (s_scales - base) + ATOMS * 512,
                                2 * ATOMS * 512, bars, bars + STAGES, abort_flag);
  }
  // every warp waits for the sums: all copies have been read then, so that their memory is free (a rank without steps has none)
  const bool any = last > first, ok = !any || mm_wait<GIVE_UP>(bars + 2 * STAGES, 0, abort_flag);
  tc_fence_after();
  float* part = reinterpret_cast<float*>(sm);      // [T][128]
  if (warp >= 2 && ok) {
    const int quad = warp & 3;
#pragma unroll 1
    for (int c = 0; c < T; c += 16) {
      uint32_t v[16] = {};
      if (any) {
        tmem_ld16(tmem_addr(tmem, quad * 32, c), v);
        tmem_wait_ld();
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) part[(c + i) * 128 + quad * 32 + lane] = __uint_as_float(v[i]);
    }
  }
  __syncwarp();
  tc_fence_before();
  if (splits > 1) cluster_sync();
  else __syncthreads();
  mm_gave_up(p, abort_flag);
  if (warp == 0) tmem_dealloc(tmem, COLUMNS);

  const int n = n0 + lane * 4, rows = min(T, p.M - m0);
  float bias[4], gate[4];
  load4(p.bias, n, p.N, p.vec_dtype, 0.f, bias);
  load4(p.gate, n, p.N, p.vec_dtype, 1.f, gate);
  for (int t = rank + warp * splits; t < rows; t += splits * (MR_THREADS / 32)) {
    const uint32_t at = smem_u32(part + t * 128 + lane * 4);
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < splits; ++r) {
      const float4 v = splits > 1 ? cluster_load4(cluster_addr(at, r)) : *reinterpret_cast<const float4*>(part + t * 128 + lane * 4);
      y[0] += v.x, y[1] += v.y, y[2] += v.z, y[3] += v.w;
    }
    mr_finish<FMT, OUT>(p, m0 + t, n, y, bias, gate);
  }
  if (splits > 1) cluster_sync();      // the others have read this CTA's sums
}

// SMs of the current device, looked up once.
static int sm_count() {
  static int n[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (!n[dev] && cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n[dev];
}

// How a product is run.  T = 0: by pairs of CTAs; else the few-rows kernel with T columns and `splits` parts of K.
struct MmPlan {
  int T, splits;
};
static MmPlan mm_plan(int M, int N, int K) {
  const int sms = sm_count(), T = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  const long long ctas = (long long)cdiv(N, 128) * cdiv(M, T);
  // More than 128 rows: few-rows CTAs as long as all fit the SMs at once (256 x 5,120 x 5,120: 14.5 us, pairs 15.5; 512 rows
  // 27.3 and 15.7).
  if (M > 128 && ctas > sms) return {0, 1};
  // Clusters of more than four do not pack: 40 clusters of 7 or 8 CTAs, two on an SM, ran one behind the other (1 x 5,120 x 5,120:
  // 11.3 us, 6.5 with four).
  long long splits = (T <= 32 ? 2 : 1) * sms / ctas;
  if (splits > 4) splits = 4;
  if (splits > cdiv(K, MM_K)) splits = cdiv(K, MM_K);
  return {T, splits > 1 ? (int)splits : 1};
}

// A grid that may be set up while the kernel in front of it still runs; `cluster` CTAs together (0: as the kernel says).
struct MmLaunch {
  cudaLaunchAttribute attrs[2] = {};
  cudaLaunchConfig_t cfg = {};
  MmLaunch(dim3 grid, int threads, int smem, int cluster, cudaStream_t st) {
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = cluster;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attrs;
    cfg.numAttrs = cluster ? 2 : 1;
  }
};

template <int FMT, int T, typename OUT, typename X = void, bool GIVE_UP = false>
static int mm_launch_rows(const MmMaps& maps, const MmArgs& p, int splits, cudaStream_t st) {
  auto* k = fp4_mm_rows_kernel<FMT, T, OUT, X, GIVE_UP>;
  constexpr int smem = mr_smem(FMT, T);
  static std::atomic<unsigned long long> allowed{0};
  if (!allow_smem(k, smem, allowed)) return T2T_ERR_CUDA;
  MmLaunch l(dim3(cdiv(p.N, 128) * splits, cdiv(p.M, T)), MR_THREADS, smem, splits, st);
  return cudaLaunchKernelEx(&l.cfg, k, maps, p, splits) == cudaSuccess ? T2T_OK : T2T_ERR_CUDA;
}

template <int FMT, typename T, MmEpilogue EPI, bool GIVE_UP = false>
static int mm_launch_pairs(const MmMaps& maps, const MmArgs& p, cudaStream_t st) {
  auto* k = fp4_mm_pair_kernel<FMT, T, EPI, GIVE_UP>;
  static std::atomic<unsigned long long> allowed{0};
  if (!allow_smem(k, mm_smem(FMT, EPI), allowed)) return T2T_ERR_CUDA;
  const long long tiles = (long long)cdiv(p.M, MM_TILE) * cdiv(p.N, MM_TILE);
  const int pairs = (int)(tiles < sm_count() / 2 ? tiles : sm_count() / 2);
  if (pairs < 1) return T2T_ERR_CUDA;
  MmLaunch l(dim3(2 * pairs), mm_threads(EPI), mm_smem(FMT, EPI), 0, st);
  return cudaLaunchKernelEx(&l.cfg, k, maps, p) == cudaSuccess ? T2T_OK : T2T_ERR_CUDA;
}

template <typename T>
static bool mm_result_maps(MmMaps& maps, const MmArgs& p) {
  constexpr int size = sizeof(T);
  constexpr bool half = std::is_same<T, __half>::value;
  return make_result_map(&maps.out, p.out, size, half, p.N, p.M, p.out_row) &&
         (!p.residual || make_result_map(&maps.res, p.residual, size, half, p.N, p.M, p.res_row));
}

template <int FMT, typename T>
static int mm_launch(MmMaps& maps, const MmArgs& p, const MmPlan& plan, cudaStream_t st) {
  if (p.x) {
    if constexpr (!std::is_same<T, uint8_t>::value) {      // of the result's type
      return mm_launch_rows<FMT, 16, T, T>(maps, p, plan.splits, st);
    } else {
      if (p.x_dtype == T2T_BF16) return mm_launch_rows<FMT, 16, T, __nv_bfloat16>(maps, p, plan.splits, st);
      if (p.x_dtype == T2T_FP16) return mm_launch_rows<FMT, 16, T, __half>(maps, p, plan.splits, st);
      return mm_launch_rows<FMT, 16, T, float>(maps, p, plan.splits, st);
    }
  }
  if (plan.T == 16) return mm_launch_rows<FMT, 16, T>(maps, p, plan.splits, st);
  if (plan.T == 32) return mm_launch_rows<FMT, 32, T>(maps, p, plan.splits, st);
  if (plan.T == 64) return mm_launch_rows<FMT, 64, T>(maps, p, plan.splits, st);
  if (plan.T == 128) return mm_launch_rows<FMT, 128, T>(maps, p, plan.splits, st);
  if constexpr (std::is_same<T, uint8_t>::value) {
    return mm_launch_pairs<FMT, T, MM_CODES>(maps, p, st);
  } else {
    // rows of a residual that overlap (one row for all: stride 0) are no tensor that TMA describes
    if (!p.wide || (p.residual && p.res_row < p.N)) return mm_launch_pairs<FMT, T, MM_LANES>(maps, p, st);
    if (!mm_result_maps<T>(maps, p)) return T2T_ERR_CUDA;
    return mm_launch_pairs<FMT, T, MM_TMA>(maps, p, st);
  }
}

}  // namespace t2t

using namespace t2t;

static bool mm_operand_maps(MmMaps& maps, const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales, int fmt,
                            const MmArgs& p, const MmPlan& plan) {
  const int pitch = fp4_pitch(p.K), atoms = fp4_atoms(p.K, fmt), box = mm_stage_atoms(fmt);
  return (p.x || (make_bytes_tile_map(&maps.a, a_codes, pitch, p.M, plan.T ? plan.T : 128) &&
                  make_scale_map(&maps.sa, a_scales, atoms, cdiv(p.M, 128), box, 1))) &&
         make_bytes_tile_map(&maps.w, w_codes, pitch, p.N, 128) &&
         make_scale_map(&maps.sw, w_scales, atoms, cdiv(p.N, 128), box, plan.T ? 1 : 2);
}
// Bytes [p, p + n) and [q, q + m) have some in common.
static bool mm_shares(const void* p, size_t n, const void* q, size_t m) {
  return (uintptr_t)p < (uintptr_t)q + m && (uintptr_t)q < (uintptr_t)p + n;
}
// Checks and launch common to the two entry points; dtype < 0: quantised results.
static int mm_run(const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales, int fmt, int dtype,
                  const MmArgs& p, cudaStream_t stream) {
  if ((!p.x && (!a_codes || !a_scales)) || !w_codes || !w_scales || !p.out || p.M <= 0 || p.N <= 0 || p.K <= 0 || p.K > (1 << 24))
    return T2T_ERR_ARG;
  if (!(p.alpha - p.alpha == 0.f)) return T2T_ERR_ARG;      // an infinity would make NaN of sums that are 0
  if (!fp4_known(fmt) || !elem_known(p.vec_dtype) || p.act < T2T_ACT_NONE || p.act > T2T_ACT_SILU) return T2T_ERR_ARG;
  if (((uintptr_t)a_codes | (uintptr_t)a_scales | (uintptr_t)w_codes | (uintptr_t)w_scales) % 16) return T2T_ERR_ARG;
  if ((long long)cdiv(p.M, MM_TILE) * cdiv(p.N, MM_TILE) > 0x3fffffffLL) return T2T_ERR_ARG;
  // factors that the result overlaps would be overwritten while other CTAs still read them
  const struct { const void* at; size_t bytes; } in[4] = {
      {a_codes, p.x ? 0 : t2t_fp4_codes_bytes(p.M, p.K)}, {a_scales, p.x ? 0 : t2t_fp4_scales_bytes(p.M, p.K, fmt)},
      {w_codes, t2t_fp4_codes_bytes(p.N, p.K)}, {w_scales, t2t_fp4_scales_bytes(p.N, p.K, fmt)}};
  const size_t written = dtype < 0 ? t2t_fp4_codes_bytes(p.M, p.N) : ((p.M - 1) * (size_t)p.out_row + p.N) * elem_bytes(dtype);
  for (const auto& t : in)
    if (t.bytes && (mm_shares(t.at, t.bytes, p.out, written) ||
                    (dtype < 0 && mm_shares(t.at, t.bytes, p.out_scales, t2t_fp4_scales_bytes(p.M, p.N, fmt)))))
      return T2T_ERR_ARG;
  if (sm_count() < 2) return T2T_ERR_CUDA;
  const MmPlan plan = mm_plan(p.M, p.N, p.K);
  MmMaps maps;
  if (!mm_operand_maps(maps, a_codes, a_scales, w_codes, w_scales, fmt, p, plan)) return T2T_ERR_CUDA;
#define T2T_CALL(T) return fmt == T2T_MXFP4 ? mm_launch<T2T_MXFP4, T>(maps, p, plan, stream) : mm_launch<T2T_NVFP4, T>(maps, p, plan, stream)
  if (dtype < 0) T2T_CALL(uint8_t);
  if (dtype == T2T_BF16) T2T_CALL(__nv_bfloat16);
  if (dtype == T2T_FP16) T2T_CALL(__half);
  T2T_CALL(float);
#undef T2T_CALL
}

// A quantised, or x as it is.
struct MmInput {
  const void *codes, *scales, *x;
  long long x_row;
  int x_dtype;
};
static bool mm_wide(const void* x, long long row, int dtype) {
  return (uintptr_t)x % 16 == 0 && row * elem_bytes(dtype) % 16 == 0;
}
static int mm_values(const MmInput& a, const void* w_codes, const void* w_scales, int M, int N, int K, int fmt, float alpha,
                     const void* bias, int act, const void* gate, int vec_dtype, const void* residual, long long residual_row,
                     void* out, long long out_row, int dtype, int* d_status, cudaStream_t stream) {
  if (!elem_known(dtype) || out_row < N || (residual && residual_row < 0)) return T2T_ERR_ARG;
  const MmArgs p = {bias, gate, residual, out, residual_row, out_row, M, N, K, act, vec_dtype,
                    mm_wide(out, out_row, dtype) && (!residual || mm_wide(residual, residual_row, dtype)), alpha,
                    1.f, 1.f, nullptr, d_status, a.x, a.x_row, a.x_dtype, a.x && mm_wide(a.x, a.x_row, a.x_dtype)};
  return mm_run(a.codes, a.scales, w_codes, w_scales, fmt, dtype, p, stream);
}
static int mm_codes(const MmInput& a, const void* w_codes, const void* w_scales, int M, int N, int K, int fmt, float alpha,
                    const void* bias, int act, const void* gate, int vec_dtype, float tensor_scale, void* codes, void* scales,
                    int* d_status, cudaStream_t stream) {
  if (!scales || (uintptr_t)codes % 16) return T2T_ERR_ARG;
  if (!(tensor_scale >= 0x1p-100f && tensor_scale <= 0x1p100f) || (fmt == T2T_MXFP4 && tensor_scale != 1.f)) return T2T_ERR_ARG;
  const MmArgs p = {bias, gate, nullptr, codes, 0, 0, M, N, K, act, vec_dtype, false, alpha, tensor_scale, 1.f / tensor_scale,
                    static_cast<uint8_t*>(scales), d_status, a.x, a.x_row, a.x_dtype, a.x && mm_wide(a.x, a.x_row, a.x_dtype)};
  return mm_run(a.codes, a.scales, w_codes, w_scales, fmt, -1, p, stream);
}

extern "C" int t2t_fp4_matmul(const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales, int M, int N,
                              int K, int fmt, float alpha, const void* bias, int act, const void* gate, int vec_dtype,
                              const void* residual, long long residual_row_stride, void* out, long long out_row_stride,
                              int dtype, int* d_status, cudaStream_t stream) {
  return mm_values({a_codes, a_scales, nullptr, 0, 0}, w_codes, w_scales, M, N, K, fmt, alpha, bias, act, gate, vec_dtype, residual,
                   residual_row_stride, out, out_row_stride, dtype, d_status, stream);
}

extern "C" int t2t_fp4_matmul_quantize(const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales, int M,
                                       int N, int K, int fmt, float alpha, const void* bias, int act, const void* gate,
                                       int vec_dtype, float tensor_scale, void* codes, void* scales, int* d_status,
                                       cudaStream_t stream) {
  return mm_codes({a_codes, a_scales, nullptr, 0, 0}, w_codes, w_scales, M, N, K, fmt, alpha, bias, act, gate, vec_dtype, tensor_scale,
                  codes, scales, d_status, stream);
}

// x as the input of a product: as it is where the product quantises it, else quantised here.  `out` [M, N]: what the product writes
// in x's type, or null; where it overlaps x, some CTAs would write what others have yet to read.
static int mm_input(MmInput& a, const void* x, long long x_row, const void* shift, const void* scale, float eps, int M, int K, int dtype,
                    int fmt, const void* out, long long out_row, int N, void* ws, size_t ws_bytes, cudaStream_t stream) {
  const int vectors = dtype & T2T_WIDE_VECTORS;
  dtype &= ~T2T_WIDE_VECTORS;
  if (!x || x_row < 0 || !elem_known(dtype)) return T2T_ERR_ARG;
  auto end = [&](const void* y, long long row, int n) { return (uintptr_t)y + ((M - 1) * row + n) * elem_bytes(dtype); };
  const bool apart = !out || end(x, x_row, K) <= (uintptr_t)out || end(out, out_row, N) <= (uintptr_t)x;
  a = {nullptr, nullptr, x, x_row, dtype};
  if (M <= T2T_FP4_FEW_ROWS && !shift && !scale && apart) return T2T_OK;
  if (!ws) return T2T_ERR_ARG;
  if (ws_bytes < t2t_fp4_linear_ws_bytes(M, K, fmt)) return T2T_ERR_WORKSPACE;
  uint8_t* scales = static_cast<uint8_t*>(ws) + t2t_fp4_codes_bytes(M, K);
  a = {ws, scales, nullptr, 0, 0};
  return t2t_fp4_quantize(x, x_row, shift, scale, eps, M, K, dtype | vectors, fmt, 1.f, ws, scales, stream);
}

extern "C" size_t t2t_fp4_linear_ws_bytes(int M, int K, int fmt) {
  return t2t_fp4_codes_bytes(M, K) + t2t_fp4_scales_bytes(M, K, fmt);
}

extern "C" int t2t_fp4_linear(const void* x, long long x_row_stride, const void* shift, const void* scale, float eps, int M, int K,
                              int dtype, int fmt, const void* w_codes, const void* w_scales, float w_scale, int N,
                              const void* bias, int act, const void* gate, int vec_dtype, const void* residual,
                              long long residual_row_stride, void* out, long long out_row_stride, void* ws, size_t ws_bytes,
                              int* d_status, cudaStream_t stream) {
  if (!fp4_known(fmt) || M <= 0 || K <= 0 || N <= 0 || !out) return T2T_ERR_ARG;
  MmInput a;
  const int rc = mm_input(a, x, x_row_stride, shift, scale, eps, M, K, dtype, fmt, out, out_row_stride, N, ws, ws_bytes, stream);
  if (rc != T2T_OK) return rc;
  return mm_values(a, w_codes, w_scales, M, N, K, fmt, w_scale, bias, act, gate, vec_dtype, residual, residual_row_stride, out,
                   out_row_stride, dtype & ~T2T_WIDE_VECTORS, d_status, stream);
}

extern "C" size_t t2t_fp4_feed_forward_ws_bytes(int M, int K, int F, int fmt) {
  return t2t_fp4_linear_ws_bytes(M, K, fmt) + t2t_fp4_linear_ws_bytes(M, F, fmt);      // multiples of 16 bytes
}

extern "C" int t2t_fp4_feed_forward(const void* x, long long x_row_stride, const void* shift, const void* scale, float eps, int M,
                                    int K, int dtype, int fmt, const void* up_codes, const void* up_scales, float up_scale, int F,
                                    const void* up_bias, int up_vec_dtype, int act, const void* down_codes,
                                    const void* down_scales, float down_scale, int N, const void* down_bias, const void* gate,
                                    int down_vec_dtype, const void* residual, long long residual_row_stride, void* out,
                                    long long out_row_stride, void* ws, size_t ws_bytes, int* d_status, cudaStream_t stream) {
  if (!fp4_known(fmt) || M <= 0 || K <= 0 || F <= 0 || !ws) return T2T_ERR_ARG;
  if (ws_bytes < t2t_fp4_feed_forward_ws_bytes(M, K, F, fmt)) return T2T_ERR_WORKSPACE;
  uint8_t *h = static_cast<uint8_t*>(ws) + t2t_fp4_linear_ws_bytes(M, K, fmt), *hs = h + t2t_fp4_codes_bytes(M, F);
  MmInput a;
  int rc = mm_input(a, x, x_row_stride, shift, scale, eps, M, K, dtype, fmt, nullptr, 0, 0, ws, ws_bytes, stream);
  if (rc != T2T_OK) return rc;
  rc = mm_codes(a, up_codes, up_scales, M, F, K, fmt, up_scale, up_bias, act, nullptr, up_vec_dtype, 1.f, h, hs, d_status, stream);
  if (rc != T2T_OK) return rc;
  return t2t_fp4_matmul(h, hs, down_codes, down_scales, M, N, F, fmt, down_scale, down_bias, T2T_ACT_NONE, gate, down_vec_dtype,
                        residual, residual_row_stride, out, out_row_stride, dtype & ~T2T_WIDE_VECTORS, d_status, stream);
}

extern "C" int t2t_fp4_give_up_selftest(int stuck, const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales,
                                        int M, int N, int K, const void* residual, void* out, int* d_status, cudaStream_t stream) {
  if (!a_codes || !a_scales || !w_codes || !w_scales || !residual || !out || !d_status) return T2T_ERR_ARG;
  if (M <= 0 || N <= 0 || K <= 0 || N % 8 || K > (1 << 24) || stuck < MM_STUCK_NONE || stuck > MM_STUCK_RESIDUAL) return T2T_ERR_ARG;
  if (((uintptr_t)a_codes | (uintptr_t)a_scales | (uintptr_t)w_codes | (uintptr_t)w_scales | (uintptr_t)residual | (uintptr_t)out) % 16)
    return T2T_ERR_ARG;
  if (sm_count() < 2) return T2T_ERR_CUDA;
  const MmPlan plan = mm_plan(M, N, K);
  if (plan.T && (plan.T != 16 || stuck == MM_STUCK_RESIDUAL)) return T2T_ERR_ARG;
  MmArgs p = {};
  p.residual = residual;
  p.out = out;
  p.res_row = p.out_row = N;
  p.M = M;
  p.N = N;
  p.K = K;
  p.wide = true;
  p.alpha = p.out_scale = p.inv_out_scale = 1.f;
  p.status = d_status;
  p.stuck = stuck;
  MmMaps maps;
  if (!mm_operand_maps(maps, a_codes, a_scales, w_codes, w_scales, T2T_NVFP4, p, plan)) return T2T_ERR_CUDA;
  if (plan.T) return mm_launch_rows<T2T_NVFP4, 16, __nv_bfloat16, void, true>(maps, p, plan.splits, stream);
  if (!mm_result_maps<__nv_bfloat16>(maps, p)) return T2T_ERR_CUDA;
  return mm_launch_pairs<T2T_NVFP4, __nv_bfloat16, MM_TMA, true>(maps, p, stream);
}
