// Rotary positions of queries and keys, with an optional RMS norm in front, and the gradient of both.
//
//   theta = position[axis(j)] * f_j,   j = 0 .. rotary_dim / 2 - 1
//   (a, b) -> m (a cos theta - b sin theta, a sin theta + b cos theta)
//
// on the pairs (2 j, 2 j + 1) or (j, j + rotary_dim / 2) of every head; the rest of the head passes unchanged.  The
// frequencies come as turns per position in units of 2^-64: the 64-bit product with the position drops whole turns
// without rounding, so what is off is the position times the error of the frequency itself.  Rotary's, out of 64-bit floats, are right to
// 2^-55 turns, and the angle to 32 bits up to 2^29 positions (position * f in 32 bits is off by 0.008 rad at 131,072).
// Statistics, angles and the rotation are held in 32 bits; each output is rounded once.
//
// An item is two vectors of V elements that hold V pairs.  L lanes (a power of two) work on one head of one token, a
// block on all heads of q and k of one token: the cosines are computed once per token and shared by all heads.
#include "elem.cuh"
#include "internal.h"

namespace t2t {

struct RotarySide {                   // one tensor: q or k
  const void* x;
  const void* dy;                     // gradient only
  void* out;
  const void* weight;                 // null: no norm
  int heads;
  long long x_batch, x_token, x_head, d_batch, d_token, d_head, o_batch, o_token, o_head;      // strides in elements
};
struct RotaryArgs {
  RotarySide side[2];
  const void* pos;
  const long long* turns;
  const int* axis;
  long long pos_axis, pos_batch;      // strides of the positions (a token's is 1)
  int pos_bytes, N, D, rd, inverse, norm, weight_dtype;
  long long rows;                     // batch * N
  float mscale, eps;
  float* partial;                     // gradient of the weights, one row per block
};

constexpr int ROT_MAX_PAIRS = 256;
constexpr int ROT_SMEM = 200 * 1024;      // dynamic shared memory a block may ask for, beside up to 7 KB of its own

// cos and sin (times m) of the rd / 2 angles of one token, by all threads.
__device__ __forceinline__ void rotary_table(const RotaryArgs& a, long long b, long long n, float2* table) {
  for (int j = threadIdx.x; j < a.rd / 2; j += blockDim.x) {
    const long long at = a.axis[j] * a.pos_axis + b * a.pos_batch + n;
    const long long p = a.pos_bytes == 8 ? static_cast<const long long*>(a.pos)[at] : static_cast<const int*>(a.pos)[at];
    const unsigned long long phase = (unsigned long long)p * (unsigned long long)a.turns[j];
    float s, c;
    sincospif((float)(int)(phase >> 32) * 0x1p-31f, &s, &c);      // half turns in [-1, 1]
    table[j] = make_float2(c * a.mscale, (a.inverse ? -s : s) * a.mscale);
  }
}

// Offsets within a head of item i's two vectors; pairs j0 .. j0 + V - 1, or j0 < 0 behind the rotated part.
template <int V, bool INTER>
__device__ __forceinline__ void item_at(int i, int rd, int& lo, int& hi, int& j0) {
  const int rot = rd / (2 * V);
  if (i >= rot) {
    lo = rd + (i - rot) * 2 * V;
    hi = lo + V;
    j0 = -1;
  } else if (INTER) {
    lo = i * 2 * V;
    hi = lo + V;
    j0 = i * V;
  } else {
    lo = i * V;
    hi = lo + rd / 2;
    j0 = lo;
  }
}

// Turns the item x[0 .. 2 V): the first V elements are the vector at lo.
template <int V, bool INTER>
__device__ __forceinline__ void turn(float (&x)[2 * V], const float2* table, int j0) {
  if (j0 < 0) return;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float2 cs = table[j0 + e];
    float& a = INTER ? x[2 * e] : x[e];
    float& b = INTER ? x[2 * e + 1] : x[V + e];
    const float u = a * cs.x - b * cs.y, v = a * cs.y + b * cs.x;
    a = u;
    b = v;
  }
}

template <typename T, int V>
__device__ __forceinline__ void load_item(const T* p, int lo, int hi, float (&x)[2 * V]) {
  const Vec<T, V> a = load_vec<T, V>(p + lo), b = load_vec<T, V>(p + hi);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    x[e] = to_f(a.e[e]);
    x[V + e] = to_f(b.e[e]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_item(T* p, int lo, int hi, const float (&x)[2 * V]) {
  Vec<T, V> a, b;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    a.e[e] = from_f<T>(x[e]);
    b.e[e] = from_f<T>(x[V + e]);
  }
  store_vec<T, V>(p + lo, a);
  store_vec<T, V>(p + hi, b);
}

__device__ __forceinline__ float group_sum(float v, int L) {
  for (int d = L >> 1; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Sum over the block of n values; every thread gets them.  red: 32 * n floats.
template <int n>
__device__ __forceinline__ void block_sum(float (&v)[n], float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    v[i] = warp_sum(v[i]);
    if (lane == 0) red[i * 32 + warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < n; ++i) {
    float s = 0.f;
    for (int w = 0; w < warps; ++w) s += red[i * 32 + w];
    v[i] = s;
  }
}

// ---- every item in a register ------------------------------------------------------
// Where each lane has at most one item of a head (2 V elements, V elements 16 bytes), a thread meets item i = its number
// modulo L in every head it works on, at most R of them, so its angles are the same for all and x stays in registers
// between the norm's sum and the rotation: one pass over x.  Arithmetic goes by pairs of elements (f32x2).
// Neighbouring lanes take neighbouring vectors, so an instruction moves whole sectors: the item's two vectors are half a head apart
// (half the rotated part, half the rest in the "half" layout, whose first vector holds the first elements of its pairs and
// the second the second ones).  32 bytes a lane in two instructions of 16 took 914 us instead of 604.
template <int V, bool INTER>
__device__ __forceinline__ void vectors_at(int i, int D, int rd, int& lo, int& hi, int& j_lo, int& j_hi) {
  const int rot = rd / (2 * V);
  if (INTER) {
    lo = i * V;
    hi = lo + D / 2;
    j_lo = lo < rd ? lo / 2 : -1;      // first of the V / 2 pairs of each vector
    j_hi = hi < rd ? hi / 2 : -1;
  } else {
    lo = i < rot ? i * V : rd + (i - rot) * V;
    hi = lo + (i < rot ? rd / 2 : (D - rd) / 2);
    j_lo = i < rot ? lo : -1;
    j_hi = i < rot ? lo + V / 2 : -1;
  }
}
template <typename T, int V>
struct Item {      // as stored
  uint4 lo, hi;
};
template <typename T>
__device__ __forceinline__ void words_to_f(const uint4& v, float (&y)[16 / sizeof(T)]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 4) {
      y[e] = __uint_as_float(w[e]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(w + e));
      y[2 * e] = f.x;
      y[2 * e + 1] = f.y;
    } else {
      y[2 * e] = bf_lo(w[e]);
      y[2 * e + 1] = bf_hi(w[e]);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 f_to_words(const float (&y)[16 / sizeof(T)]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 4) {
      w[e] = __float_as_uint(y[e]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(y[2 * e], y[2 * e + 1]);
      w[e] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      w[e] = pack_bf2(y[2 * e], y[2 * e + 1]);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// First and second elements of the V pairs, two pairs to an operand.
template <int V>
struct Pairs {
  uint64_t a[V / 2], b[V / 2];
};
template <int V, bool INTER>
__device__ __forceinline__ Pairs<V> pairs_of(const float (&lo)[V], const float (&hi)[V]) {
  Pairs<V> p;
#pragma unroll
  for (int e = 0; e < V / 2; ++e) {
    if (INTER) {
      const float* y = e < V / 4 ? lo + 4 * e : hi + 4 * (e - V / 4);
      p.a[e] = pair_of(y[0], y[2]);
      p.b[e] = pair_of(y[1], y[3]);
    } else {
      p.a[e] = pair_of(lo[2 * e], lo[2 * e + 1]);
      p.b[e] = pair_of(hi[2 * e], hi[2 * e + 1]);
    }
  }
  return p;
}
template <typename T, int V, bool INTER>
__device__ __forceinline__ Pairs<V> unpack_item(const Item<T, V>& x) {
  float lo[V], hi[V];
  words_to_f<T>(x.lo, lo);
  words_to_f<T>(x.hi, hi);
  return pairs_of<V, INTER>(lo, hi);
}
template <typename T, int V, bool INTER>
__device__ __forceinline__ Item<T, V> pack_item(const Pairs<V>& p) {
  float lo[V], hi[V];
#pragma unroll
  for (int e = 0; e < V / 2; ++e) {
    if (INTER) {
      float* y = e < V / 4 ? lo + 4 * e : hi + 4 * (e - V / 4);
      pair_to(p.a[e], y[0], y[2]);
      pair_to(p.b[e], y[1], y[3]);
    } else {
      pair_to(p.a[e], lo[2 * e], lo[2 * e + 1]);
      pair_to(p.b[e], hi[2 * e], hi[2 * e + 1]);
    }
  }
  return {f_to_words<T>(lo), f_to_words<T>(hi)};
}
// Norm weights at the item's two vectors.
template <typename T, int V, bool INTER>
__device__ __forceinline__ Pairs<V> load_weights(const void* w, long long lo, long long hi, bool wide) {      // wide: 32 bits
  float x[V], y[V];
  if (!wide) {
    words_to_f<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(w) + lo), x);
    words_to_f<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(w) + hi), y);
  } else {
    const float4 *p = reinterpret_cast<const float4*>(static_cast<const float*>(w) + lo),
                 *q = reinterpret_cast<const float4*>(static_cast<const float*>(w) + hi);
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 f = p[i], g = q[i];
      x[4 * i] = f.x, x[4 * i + 1] = f.y, x[4 * i + 2] = f.z, x[4 * i + 3] = f.w;
      y[4 * i] = g.x, y[4 * i + 1] = g.y, y[4 * i + 2] = g.z, y[4 * i + 3] = g.w;
    }
  }
  return pairs_of<V, INTER>(x, y);
}
// What a thread works on: item i of head `group` + round * groups of q and k together, for every token.  Where the items start is kept as
// addresses within a token; worked out for every item again, they and the 64-bit products with the strides were two
// thirds of the instructions.
struct Place {
  int side, head;
  bool on;
};
__device__ __forceinline__ Place place_of(const RotaryArgs& a, int head, bool on_item) {
  const int side = head >= a.side[0].heads;
  head -= side ? a.side[0].heads : 0;
  return {side, head, on_item && head < a.side[side].heads};
}
template <typename T, int V, bool INTER, int R, bool GRAD>
struct Work {
  int group, groups, lo, hi, j_lo, j_hi;
  bool on_item;
  uint32_t on, second;      // bits of the rounds: there is an item, it is k's
  const T *x[R], *dy[GRAD ? R : 1];
  T* out[R];
  __device__ __forceinline__ Work(const RotaryArgs& a, int L) {
    const int i = threadIdx.x % L;
    group = threadIdx.x / L;
    groups = blockDim.x / L;
    on_item = i < a.D / (2 * V);
    vectors_at<V, INTER>(on_item ? i : 0, a.D, a.rd, lo, hi, j_lo, j_hi);
    on = second = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const Place w = place_of(a, group + r * groups, on_item);
      const RotarySide& z = a.side[w.side];
      on |= (uint32_t)w.on << r;
      second |= (uint32_t)w.side << r;
      x[r] = static_cast<const T*>(z.x) + w.head * z.x_head + lo;
      if (GRAD) dy[r] = static_cast<const T*>(z.dy) + w.head * z.d_head + lo;
      out[r] = static_cast<T*>(z.out) + w.head * z.o_head + lo;
    }
    hi -= lo;      // from here on: the second vector's distance from the first
  }
  __device__ __forceinline__ bool has(int r) const { return on >> r & 1u; }
  __device__ __forceinline__ bool is_k(int r) const { return second >> r & 1u; }
};
// Offset of a token in a tensor of q and one of k.
struct Token {
  long long q, k;
  __device__ __forceinline__ long long of(bool is_k) const { return is_k ? k : q; }
};
enum { TENSOR_X, TENSOR_DY, TENSOR_OUT };
template <int WHICH>
__device__ __forceinline__ Token token_at(const RotaryArgs& a, long long row) {
  const RotarySide &q = a.side[0], &k = a.side[1];
  const long long qt = WHICH == TENSOR_X ? q.x_token : WHICH == TENSOR_DY ? q.d_token : q.o_token;
  const long long kt = WHICH == TENSOR_X ? k.x_token : WHICH == TENSOR_DY ? k.d_token : k.o_token;
  if (a.rows == a.N) return {row * qt, row * kt};
  const long long qb = WHICH == TENSOR_X ? q.x_batch : WHICH == TENSOR_DY ? q.d_batch : q.o_batch;
  const long long kb = WHICH == TENSOR_X ? k.x_batch : WHICH == TENSOR_DY ? k.d_batch : k.o_batch;
  const long long b = row / a.N, n = row - b * a.N;
  return {b * qb + n * qt, b * kb + n * kt};
}

// The thread's norm weights: kept as they are stored (KEEP), or read for every token: where a thread has four items, and where
// they have 32 bits and x has 16.
template <typename T, int V, bool INTER, int R, bool KEEP>
struct Weights {
  Item<T, V> kept[KEEP ? R : 1];
  const void* at[R];
  bool wide;
  __device__ __forceinline__ Weights(const RotaryArgs& a, const Place (&place)[R], int lo, int hi) {
    wide = a.weight_dtype == T2T_FP32 && sizeof(T) == 2;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long i = lo + (a.norm == T2T_NORM_ROW ? (long long)place[r].head * a.D : 0);
      at[r] = static_cast<const uint8_t*>(a.side[place[r].side].weight) + i * (wide ? 4 : (int)sizeof(T));
      if (KEEP && !wide && a.norm && place[r].on) {
        kept[r].lo = *static_cast<const uint4*>(at[r]);
        kept[r].hi = *reinterpret_cast<const uint4*>(static_cast<const T*>(at[r]) + hi);
      }
    }
  }
  __device__ __forceinline__ Pairs<V> get(int r, int hi) const {
    if (KEEP && !wide) return unpack_item<T, V, INTER>(kept[KEEP ? r : 0]);
    return load_weights<T, V, INTER>(at[r], 0, hi, wide);
  }
};
template <int V>
__device__ __forceinline__ float sum_products(const Pairs<V>& x, const Pairs<V>& y) {
  uint64_t s = 0;
#pragma unroll
  for (int e = 0; e < V / 2; ++e) s = fma2(x.b[e], y.b[e], fma2(x.a[e], y.a[e], s));
  float lo, hi;
  pair_to(s, lo, hi);
  return lo + hi;
}
template <int V>
__device__ __forceinline__ void scale_pairs(Pairs<V>& x, const Pairs<V>& y) {
#pragma unroll
  for (int e = 0; e < V / 2; ++e) {
    x.a[e] = mul2(x.a[e], y.a[e]);
    x.b[e] = mul2(x.b[e], y.b[e]);
  }
}
template <int V>
__device__ __forceinline__ void scale_pairs(Pairs<V>& x, float f) {
  const uint64_t ff = pair_of(f, f);
#pragma unroll
  for (int e = 0; e < V / 2; ++e) {
    x.a[e] = mul2(x.a[e], ff);
    x.b[e] = mul2(x.b[e], ff);
  }
}
// Angles of an item's pairs: cosines and sines, 1 and 0 behind the rotated part.
template <int V>
struct Angles {
  uint64_t c[V / 2], s[V / 2], minus[V / 2];      // minus: -s
};
struct alignas(16) AngleTable {
  float c[ROT_MAX_PAIRS], s[ROT_MAX_PAIRS];
};
template <int V>
__device__ __forceinline__ Angles<V> load_angles(const AngleTable& table, int j_lo, int j_hi) {
  Angles<V> t;
#pragma unroll
  for (int e = 0; e < V / 2; ++e) {
    const int j = e < V / 4 ? j_lo : j_hi, at = 2 * (e < V / 4 ? e : e - V / 4);
    if (e % 2 == 0 && V == 8) {
      const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(table.c + max(j, 0));
      const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(table.s + max(j, 0));
      t.c[e] = c.x, t.c[e + 1] = c.y, t.s[e] = s.x, t.s[e + 1] = s.y;
    } else if (V != 8) {
      t.c[e] = *reinterpret_cast<const uint64_t*>(table.c + max(j, 0) + at);
      t.s[e] = *reinterpret_cast<const uint64_t*>(table.s + max(j, 0) + at);
    }
  }
#pragma unroll
  for (int e = 0; e < V / 2; ++e) {
    if ((e < V / 4 ? j_lo : j_hi) < 0) t.c[e] = pair_of(1.f, 1.f), t.s[e] = 0;
    t.minus[e] = t.s[e] ^ 0x8000000080000000ull;
  }
  return t;
}
template <int V>
__device__ __forceinline__ void turn_pairs(Pairs<V>& x, const Angles<V>& t) {
#pragma unroll
  for (int e = 0; e < V / 2; ++e) {
    const uint64_t u = fma2(x.a[e], t.c[e], mul2(x.b[e], t.minus[e]));
    x.b[e] = fma2(x.a[e], t.s[e], mul2(x.b[e], t.c[e]));
    x.a[e] = u;
  }
}

// Angles of the tokens that a block meets, one pair a thread.  Frequency and axis stay in registers and a position is read a token
// before its angle is computed: read when they were needed, the three one after the other took longer than the token's rotation.
struct AngleMaker {
  unsigned long long turns;
  long long next;      // position of the token that `make` comes to
  long long at;        // of the thread's axis
  bool on;
  __device__ __forceinline__ AngleMaker(const RotaryArgs& a, long long row) : turns(0), next(0), at(0) {
    on = threadIdx.x < a.rd / 2;
    if (on) {
      turns = (unsigned long long)a.turns[threadIdx.x];
      at = a.axis[threadIdx.x] * a.pos_axis;
    }
    read(a, row);
  }
  __device__ __forceinline__ void read(const RotaryArgs& a, long long row) {
    if (!on || row >= a.rows) return;
    const long long b = a.rows == a.N ? 0 : row / a.N, i = at + b * a.pos_batch + row - b * a.N;
    next = a.pos_bytes == 8 ? static_cast<const long long*>(a.pos)[i] : static_cast<const int*>(a.pos)[i];
  }
  // the token read before into `table`; `row` is read
  __device__ __forceinline__ void make(const RotaryArgs& a, AngleTable& table, long long row) {
    const unsigned long long phase = (unsigned long long)next * turns;
    read(a, row);
    if (!on) return;
    float s, c;
    sincospif((float)(int)(phase >> 32) * 0x1p-31f, &s, &c);
    table.c[threadIdx.x] = c * a.mscale;
    table.s[threadIdx.x] = (a.inverse ? -s : s) * a.mscale;
  }
};

// A thread's items of the tokens ahead, brought to shared memory by cp.async: written and read by the same thread, so nothing but
// its own copies has to be waited for.  [stage][round][x, dy][first, second vector][thread].
template <typename T, int V, int R, bool GRAD>
struct Ahead {
  static constexpr int TENSORS = GRAD ? 2 : 1;
  uint32_t at;
  const uint4* mine;
  __device__ __forceinline__ Ahead(uint8_t* smem) {
    mine = reinterpret_cast<const uint4*>(smem) + threadIdx.x;
    at = smem_u32(mine);
  }
  static __host__ __device__ constexpr int bytes(int threads, int stages) { return stages * R * TENSORS * 2 * threads * 16; }
  __device__ __forceinline__ int slot(int stage, int r, int tensor) const {
    return ((stage * R + r) * TENSORS + tensor) * 2 * (int)blockDim.x;
  }
  __device__ __forceinline__ Item<T, V> get(int stage, int r, int tensor) const {
    const int i = slot(stage, r, tensor);
    return {mine[i], mine[i + blockDim.x]};
  }
  template <typename W>
  __device__ __forceinline__ void fetch(const W& w, int stage, const Token& x, const Token& d, bool there) const {
    if (there) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (!w.has(r)) continue;      // its slot stays zero
        const T* p = w.x[r] + x.of(w.is_k(r));
        const uint32_t to = at + slot(stage, r, 0) * 16;
        cp_async16(to, p);
        cp_async16(to + blockDim.x * 16, p + w.hi);
        if (GRAD) {
          const T* p = w.dy[GRAD ? r : 0] + d.of(w.is_k(r));
          const uint32_t to = at + slot(stage, r, 1) * 16;
          cp_async16(to, p);
          cp_async16(to + blockDim.x * 16, p + w.hi);
        }
      }
    }
    cp_async_commit();
  }
  __device__ __forceinline__ void clear(int stages) const {
    for (int i = 0; i < stages * R * TENSORS * 2; ++i) const_cast<uint4*>(mine)[i * blockDim.x] = make_uint4(0u, 0u, 0u, 0u);
  }
};

// Sums over the block of one value each for q and k (and a second pair for the gradient): one meeting, after which every thread
// has them.  `red` is not the one of the meeting before, which others may still read.
template <typename F>      // float2 or float4
__device__ __forceinline__ void meet(F& v, F* red) {
  constexpr int n = sizeof(F) / 4;
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  float* f = reinterpret_cast<float*>(&v);
  // the n values share the warp: each step hands half of them to the other half of the lanes until a lane has one
  float part[n];
#pragma unroll
  for (int i = 0; i < n; ++i) part[i] = f[i];
#pragma unroll
  for (int k = n / 2, d = 16; k; k >>= 1, d >>= 1) {
    const bool upper = lane & d;
#pragma unroll
    for (int i = 0; i < k; ++i)
      part[i] = (upper ? part[i + k] : part[i]) + __shfl_xor_sync(0xffffffffu, upper ? part[i] : part[i + k], d);
  }
#pragma unroll
  for (int d = 16 / n; d; d >>= 1) part[0] += __shfl_xor_sync(0xffffffffu, part[0], d);
  if (lane % (32 / n) == 0) reinterpret_cast<float*>(red + (threadIdx.x >> 5))[lane / (32 / n)] = part[0];
  __syncthreads();
  v = red[0];
  for (int w = 1; w < warps; ++w) {
    const F o = red[w];
#pragma unroll
    for (int i = 0; i < n; ++i) f[i] += reinterpret_cast<const float*>(&o)[i];
  }
}

// Blocks take tokens in turn, with x of the next two on its way.  One meeting of the block a token: behind it the sums of the norm and
// the angles of this token (computed one token ahead, in the third of three tables) are there.
// Bound by memory: q and k of 75,600 tokens of 40 heads of 128, 3.1 GB, take 600 us with the norm over all heads and 530
// without in a loop over the same tensors (5.2 and 5.8 TB/s), 617 to 639 with the norm where they change from call to call.
// One block a token with x loaded to registers took 715; the kernel below, which reads x twice and weights one by one, 1,690.
constexpr int ROT_AHEAD = 3;
constexpr int fwd_threads(int R) { return R == 4 ? 512 : 256; }
constexpr int fwd_regs(int R) { return R == 1 ? 104 : 128; }
template <typename T, int V, bool INTER, int R>
__global__ void __launch_bounds__(fwd_threads(R), R == 4 ? 1 : 2)
    rotary_items_kernel(const RotaryArgs a, int L) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ AngleTable tables[3];
  __shared__ float2 red[2][16];
  const Work<T, V, INTER, R, false> work(a, L);
  Place place[R];
#pragma unroll
  for (int r = 0; r < R; ++r) place[r] = place_of(a, work.group + r * work.groups, work.on_item);
  const Weights<T, V, INTER, R, (R < 4)> weights(a, place, work.lo, work.hi);
  const Ahead<T, V, R, false> ahead(smem_raw);
  ahead.clear(ROT_AHEAD);
#pragma unroll
  for (int s = 0; s < ROT_AHEAD; ++s) {
    const long long row = blockIdx.x + (long long)s * gridDim.x;
    ahead.fetch(work, s, token_at<TENSOR_X>(a, row), Token(), row < a.rows);
  }
  AngleMaker angles(a, blockIdx.x);
  angles.make(a, tables[0], blockIdx.x + gridDim.x);
  const float inv_q = 1.f / (float)(a.side[0].heads * a.D), inv_k = 1.f / (float)(a.side[1].heads * a.D), inv_d = 1.f / (float)a.D;
  int stage = 0, now = 0, flip = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int then = now == 2 ? 0 : now + 1;
    angles.make(a, tables[then], row + 2ll * gridDim.x);
    cp_async_wait<ROT_AHEAD - 1>();
    float2 sum = make_float2(0.f, 0.f);      // becomes the factors of q and k
    if (a.norm == T2T_NORM_ROW) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Pairs<V> y = unpack_item<T, V, INTER>(ahead.get(stage, r, 0));
        const float s = sum_products(y, y);
        if (work.is_k(r)) sum.y += s;
        else sum.x += s;
      }
      meet(sum, red[flip]);
      flip ^= 1;
      sum.x = rsqrtf(fmaf(sum.x, inv_q, a.eps));
      sum.y = rsqrtf(fmaf(sum.y, inv_k, a.eps));
    } else {
      __syncthreads();
    }
    const Angles<V> t = load_angles<V>(tables[now], work.j_lo, work.j_hi);
    const Token o = token_at<TENSOR_OUT>(a, row);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      Pairs<V> y = unpack_item<T, V, INTER>(ahead.get(stage, r, 0));
      if (a.norm) {
        float f = work.is_k(r) ? sum.y : sum.x;
        if (a.norm == T2T_NORM_HEAD) f = rsqrtf(fmaf(group_sum(sum_products(y, y), L), inv_d, a.eps));
        if (work.has(r)) {
          scale_pairs(y, weights.get(r, work.hi));
          scale_pairs(y, f);
        }
      }
      turn_pairs(y, t);
      if (work.has(r)) {
        const Item<T, V> v = pack_item<T, V, INTER>(y);
        T* p = work.out[r] + o.of(work.is_k(r));
        *reinterpret_cast<uint4*>(p) = v.lo;
        *reinterpret_cast<uint4*>(p + work.hi) = v.hi;
      }
    }
    const long long next = row + (long long)ROT_AHEAD * gridDim.x;
    ahead.fetch(work, stage, token_at<TENSOR_X>(a, next), Token(), next < a.rows);
    stage = stage + 1 == ROT_AHEAD ? 0 : stage + 1;
    now = then;
  }
}

// Gradient of norm and rotation (formulas below).  As above, with x and dy on their way; a thread keeps the sums of dw of its items
// in registers.
constexpr int ROT_GRAD_AHEAD = 2;
constexpr int grad_threads(int R, int V) { return R == 1 || (R == 4 && V == 8) ? 256 : 320; }
constexpr int grad_regs(int R, int V) { return R == 1 ? 128 : V == 4 || R == 2 ? 168 : 255; }
template <typename T, int V, bool INTER, int R>
__global__ void __launch_bounds__(grad_threads(R, V), R == 1 ? 2 : 1)
    rotary_items_grad_kernel(const RotaryArgs a, int L) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ AngleTable tables[3];
  __shared__ float4 red[2][16];
  const Work<T, V, INTER, R, true> work(a, L);
  Place place[R];
#pragma unroll
  for (int r = 0; r < R; ++r) place[r] = place_of(a, work.group + r * work.groups, work.on_item);
  const Weights<T, V, INTER, R, (R == 1)> weights(a, place, work.lo, work.hi);
  Pairs<V> dw[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < V / 2; ++e) dw[r].a[e] = dw[r].b[e] = 0;
  const Ahead<T, V, R, true> ahead(smem_raw);
  ahead.clear(ROT_GRAD_AHEAD);
#pragma unroll
  for (int s = 0; s < ROT_GRAD_AHEAD; ++s) {
    const long long row = blockIdx.x + (long long)s * gridDim.x;
    ahead.fetch(work, s, token_at<TENSOR_X>(a, row), token_at<TENSOR_DY>(a, row), row < a.rows);
  }
  AngleMaker angles(a, blockIdx.x);
  angles.make(a, tables[0], blockIdx.x + gridDim.x);
  __syncthreads();      // later tables are complete behind the meeting of the token before
  const float inv_q = 1.f / (float)(a.side[0].heads * a.D), inv_k = 1.f / (float)(a.side[1].heads * a.D), inv_d = 1.f / (float)a.D;
  int stage = 0, now = 0, flip = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int then = now == 2 ? 0 : now + 1;
    angles.make(a, tables[then], row + 2ll * gridDim.x);
    cp_async_wait<ROT_GRAD_AHEAD - 1>();
    const Angles<V> t = load_angles<V>(tables[now], work.j_lo, work.j_hi);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);      // x^2 and g w x of q, of k
    float own[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const Pairs<V> y = unpack_item<T, V, INTER>(ahead.get(stage, r, 0));
      Pairs<V> g = unpack_item<T, V, INTER>(ahead.get(stage, r, 1));
      turn_pairs(g, t);
      if (work.has(r)) scale_pairs(g, weights.get(r, work.hi));
      own[r][0] = sum_products(y, y);
      own[r][1] = sum_products(y, g);
      if (work.is_k(r)) sum.z += own[r][0], sum.w += own[r][1];
      else sum.x += own[r][0], sum.y += own[r][1];
    }
    if (a.norm == T2T_NORM_ROW) {
      meet(sum, red[flip]);
      flip ^= 1;
    } else {
      __syncthreads();
    }
    const Token o = token_at<TENSOR_OUT>(a, row);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float xx, gx;      // means
      if (a.norm == T2T_NORM_ROW) {
        const float inv = work.is_k(r) ? inv_k : inv_q;
        xx = (work.is_k(r) ? sum.z : sum.x) * inv;
        gx = (work.is_k(r) ? sum.w : sum.y) * inv;
      } else {
        xx = group_sum(own[r][0], L) * inv_d;
        gx = group_sum(own[r][1], L) * inv_d;
      }
      if (!work.has(r)) continue;
      const float f = rsqrtf(xx + a.eps), c = f * f * gx;
      Pairs<V> y = unpack_item<T, V, INTER>(ahead.get(stage, r, 0)), g = unpack_item<T, V, INTER>(ahead.get(stage, r, 1));
      turn_pairs(g, t);
      const uint64_t ff = pair_of(f, f), cc = pair_of(-c, -c);
      const Pairs<V> weight = weights.get(r, work.hi);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        dw[r].a[e] = fma2(g.a[e], mul2(y.a[e], ff), dw[r].a[e]);
        dw[r].b[e] = fma2(g.b[e], mul2(y.b[e], ff), dw[r].b[e]);
        y.a[e] = mul2(ff, fma2(y.a[e], cc, mul2(g.a[e], weight.a[e])));
        y.b[e] = mul2(ff, fma2(y.b[e], cc, mul2(g.b[e], weight.b[e])));
      }
      const Item<T, V> v = pack_item<T, V, INTER>(y);
      T* p = work.out[r] + o.of(work.is_k(r));
      *reinterpret_cast<uint4*>(p) = v.lo;
      *reinterpret_cast<uint4*>(p + work.hi) = v.hi;
    }
    const long long next = row + (long long)ROT_GRAD_AHEAD * gridDim.x;
    ahead.fetch(work, stage, token_at<TENSOR_X>(a, next), token_at<TENSOR_DY>(a, next), next < a.rows);
    stage = stage + 1 == ROT_GRAD_AHEAD ? 0 : stage + 1;
    now = then;
  }
  const int lo = work.lo, hi = work.lo + work.hi, group = work.group, groups = work.groups;
  cp_async_wait<0>();
  auto put = [&](const Pairs<V>& v, float* p) {
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
      const int pa = INTER ? (e < V / 4 ? lo + 4 * e : hi + 4 * (e - V / 4)) : lo + 2 * e, step = INTER ? 2 : 1;
      const int pb = INTER ? pa + 1 : hi + 2 * e;
      pair_to(v.a[e], p[pa], p[pa + step]);
      pair_to(v.b[e], p[pb], p[pb + step]);
    }
  };
  if (a.norm == T2T_NORM_ROW) {      // every element has one owner
    const long long total = (long long)(a.side[0].heads + a.side[1].heads) * a.D;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const Place w = place[r];
      if (w.on) put(dw[r], a.partial + blockIdx.x * total + (long long)((w.side ? a.side[0].heads : 0) + w.head) * a.D);
    }
    return;
  }
  // norm per head: the heads' sums meet, those of a thread first, then the groups' in their order
  float* sums = reinterpret_cast<float*>(smem_raw);      // [2][groups][D], where the tokens were
  __syncthreads();
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    Pairs<V> v;
#pragma unroll
    for (int e = 0; e < V / 2; ++e) v.a[e] = v.b[e] = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (place[r].side == s) {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          v.a[e] = add2(v.a[e], dw[r].a[e]);
          v.b[e] = add2(v.b[e], dw[r].b[e]);
        }
      }
    if (work.on_item) put(v, sums + (s * groups + group) * a.D);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * a.D; e += blockDim.x) {
    const int s = e / a.D;
    float v = 0.f;
    for (int q = 0; q < groups; ++q) v += sums[(s * groups + q) * a.D + e - s * a.D];
    a.partial[(long long)blockIdx.x * 2 * a.D + e] = v;
  }
}

// ---- any shape ------------------------------------------------------------------------
// One block per token.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a, int L) {
  __shared__ float2 table[ROT_MAX_PAIRS];
  __shared__ float red[64];
  const long long row = blockIdx.x, b = row / a.N, n = row - b * a.N;
  const int items = a.D / (2 * V), group = threadIdx.x / L, groups = blockDim.x / L, i0 = threadIdx.x % L;
  rotary_table(a, b, n, table);
  float inv[2] = {1.f, 1.f};
  if (a.norm == T2T_NORM_ROW) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const RotarySide& z = a.side[s];
      for (int h = group; h < z.heads; h += groups) {
        const T* x = static_cast<const T*>(z.x) + b * z.x_batch + n * z.x_token + h * z.x_head;
        for (int i = i0; i < items; i += L) {
          int lo, hi, j0;
          item_at<V, INTER>(i, a.rd, lo, hi, j0);
          float v[2 * V];
          load_item<T, V>(x, lo, hi, v);
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) sum[s] += v[e] * v[e];
        }
      }
    }
    block_sum<2>(sum, red);
#pragma unroll
    for (int s = 0; s < 2; ++s) inv[s] = rsqrtf(sum[s] / (float)(a.side[s].heads * a.D) + a.eps);
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const RotarySide& z = a.side[s];
    for (int h0 = 0; h0 < z.heads; h0 += groups) {      // every lane of a warp takes part in the group's sum
      const int h = h0 + group;
      const bool on = h < z.heads;
      const T* x = static_cast<const T*>(z.x) + b * z.x_batch + n * z.x_token + (on ? h : 0) * z.x_head;
      T* out = static_cast<T*>(z.out) + b * z.o_batch + n * z.o_token + (on ? h : 0) * z.o_head;
      float r = inv[s];
      if (a.norm == T2T_NORM_HEAD) {
        float sum = 0.f;
        for (int i = i0; on && i < items; i += L) {
          int lo, hi, j0;
          item_at<V, INTER>(i, a.rd, lo, hi, j0);
          float v[2 * V];
          load_item<T, V>(x, lo, hi, v);
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) sum += v[e] * v[e];
        }
        r = rsqrtf(group_sum(sum, L) / (float)a.D + a.eps);
      }
      for (int i = i0; on && i < items; i += L) {
        int lo, hi, j0;
        item_at<V, INTER>(i, a.rd, lo, hi, j0);
        float v[2 * V];
        load_item<T, V>(x, lo, hi, v);
        if (a.norm) {
          const long long w = a.norm == T2T_NORM_ROW ? (long long)h * a.D : 0;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            v[e] *= r * load_elem(z.weight, w + lo + e, a.weight_dtype);
            v[V + e] *= r * load_elem(z.weight, w + hi + e, a.weight_dtype);
          }
        }
        turn<V, INTER>(v, table, j0);
        store_item<T, V>(out, lo, hi, v);
      }
    }
  }
}

// Gradient of norm and rotation.  With g the gradient turned back, x-hat = r x the normalised input (r = rsqrt(mean x^2 + eps)):
//   dx = r (g w - x-hat mean(g w x-hat)),   dw = sum over tokens (and heads, for the norm per head) of g x-hat.
// A block takes every gridDim.x-th token; a thread meets the same elements of every token, so it adds their dw to sums that it
// alone owns, in shared memory; the blocks' sums are joined in a fixed order by a second kernel.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(256) rotary_grad_kernel(const RotaryArgs a, int L) {
  extern __shared__ float dw[];                  // [heads of q and k][D]
  __shared__ float2 table[ROT_MAX_PAIRS];
  __shared__ float red[128];
  const int items = a.D / (2 * V), group = threadIdx.x / L, groups = blockDim.x / L, i0 = threadIdx.x % L;
  const int total = (a.side[0].heads + a.side[1].heads) * a.D;
  for (int e = threadIdx.x; e < total; e += blockDim.x) dw[e] = 0.f;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const long long b = row / a.N, n = row - b * a.N;
    __syncthreads();
    rotary_table(a, b, n, table);
    __syncthreads();
    // the two sums of every row (or head): x^2 and g w x; then the second look writes
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int look = a.norm == T2T_NORM_ROW ? 0 : 1; look < 2; ++look) {
      float* dws = dw;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const RotarySide& z = a.side[s];
        for (int h0 = 0; h0 < z.heads; h0 += groups) {
          const int h = h0 + group;
          const bool on = h < z.heads;
          const T* x = static_cast<const T*>(z.x) + b * z.x_batch + n * z.x_token + (on ? h : 0) * z.x_head;
          const T* dy = static_cast<const T*>(z.dy) + b * z.d_batch + n * z.d_token + (on ? h : 0) * z.d_head;
          T* out = static_cast<T*>(z.out) + b * z.o_batch + n * z.o_token + (on ? h : 0) * z.o_head;
          const long long w = a.norm == T2T_NORM_ROW ? (long long)h * a.D : 0;
          float xx = 0.f, gx = 0.f;
          if (look == 0 || a.norm == T2T_NORM_HEAD) {
            for (int i = i0; on && i < items; i += L) {
              int lo, hi, j0;
              item_at<V, INTER>(i, a.rd, lo, hi, j0);
              float v[2 * V], g[2 * V];
              load_item<T, V>(x, lo, hi, v);
              load_item<T, V>(dy, lo, hi, g);
              turn<V, INTER>(g, table, j0);
#pragma unroll
              for (int e = 0; e < 2 * V; ++e) {
                xx += v[e] * v[e];
                gx += v[e] * g[e] * load_elem(z.weight, w + (e < V ? lo + e : hi + e - V), a.weight_dtype);
              }
            }
          }
          if (look == 0) {
            sum[2 * s] += xx;
            sum[2 * s + 1] += gx;
            continue;
          }
          float count = (float)a.D;
          if (a.norm == T2T_NORM_HEAD) {
            xx = group_sum(xx, L);
            gx = group_sum(gx, L);
          } else {
            xx = sum[2 * s];
            gx = sum[2 * s + 1];
            count *= z.heads;
          }
          const float r = rsqrtf(xx / count + a.eps), c = r * r * (gx / count);
          for (int i = i0; on && i < items; i += L) {
            int lo, hi, j0;
            item_at<V, INTER>(i, a.rd, lo, hi, j0);
            float v[2 * V], g[2 * V];
            load_item<T, V>(x, lo, hi, v);
            load_item<T, V>(dy, lo, hi, g);
            turn<V, INTER>(g, table, j0);
#pragma unroll
            for (int e = 0; e < 2 * V; ++e) {
              const int d = e < V ? lo + e : hi + e - V;
              dws[h * a.D + d] += g[e] * v[e] * r;
              v[e] = r * (g[e] * load_elem(z.weight, w + d, a.weight_dtype) - v[e] * c);
            }
            store_item<T, V>(out, lo, hi, v);
          }
        }
        dws += z.heads * a.D;
      }
      if (look == 0) block_sum<4>(sum, red);
    }
  }
  __syncthreads();
  if (a.norm == T2T_NORM_ROW) {
    for (int e = threadIdx.x; e < total; e += blockDim.x) a.partial[(long long)blockIdx.x * total + e] = dw[e];
  } else {
    for (int e = threadIdx.x; e < 2 * a.D; e += blockDim.x) {
      const int s = e / a.D, d = e - s * a.D;
      float v = 0.f;
      for (int h = 0; h < a.side[s].heads; ++h) v += dw[((s ? a.side[0].heads : 0) + h) * a.D + d];
      a.partial[(long long)blockIdx.x * 2 * a.D + e] = v;
    }
  }
}

// out[e] = sum over the blocks of partial[block][e]: eight threads an element, each adding every eighth block's, joined in order.
__global__ void __launch_bounds__(256) rotary_weight_grad_kernel(const float* __restrict__ partial, int blocks, int total,
                                                                 int first, int used, float* __restrict__ dq,
                                                                 float* __restrict__ dk) {
  __shared__ float part[8][33];
  const int e = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  float v = 0.f;
  if (e < used)
    for (int b = w; b < blocks; b += 8) v += partial[(long long)b * total + e];
  part[w][threadIdx.x & 31] = v;
  __syncthreads();
  if (w || e >= used) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += part[i][threadIdx.x & 31];
  if (e < first) dq[e] = v;
  else dk[e - first] = v;
}

constexpr int ROT_GRAD_BLOCKS = 148 * 4;

// Widest vector that the shapes, addresses and strides allow: 2 V divides the head and its rotated part.  Of the latter a whole
// interleaved 16-byte vector is enough: the kernels that keep items in registers look at each vector by itself.
static int rotary_width(const RotaryArgs& a, int bytes, bool inter, bool grad) {
  for (int v = 16 / bytes; v > 1; v >>= 1) {
    bool ok = a.D % (2 * v) == 0 && a.rd % (inter && v * bytes == 16 ? v : 2 * v) == 0;
    for (const RotarySide& z : a.side) {
      if (!z.heads) continue;
      const long long all = z.x_batch | z.x_token | z.x_head | z.o_batch | z.o_token | z.o_head |
                            (grad ? z.d_batch | z.d_token | z.d_head : 0);
      const uintptr_t at = (uintptr_t)z.x | (uintptr_t)z.out | (grad ? (uintptr_t)z.dy : 0);
      ok = ok && all % v == 0 && at % (uintptr_t)(v * bytes) == 0;
    }
    if (ok) return v;
  }
  return 1;
}

// Threads of a block whose threads hold at most R items each: the fewest idle groups, at least 64 threads and one a
// pair of the angles.  0: none.
static int items_threads(int heads, int L, int R, int pairs, int most) {
  int best = 0, waste = 0;
  for (int t = pairs > 64 ? cdiv(pairs, 32) * 32 : 64; t <= most; t += 32) {
    const int groups = t / L, rounds = cdiv(heads, groups);
    if (rounds > R) continue;
    const int w = rounds * groups - heads;
    if (!best || w < waste) best = t, waste = w;
  }
  return best;
}

// Blocks of a kernel that stay on the SMs: what the registers of an SM's four parts, shared memory and thread slots hold.
static int resident(int threads, int regs, int smem) {
  int n = 4 * (16384 / (32 * regs)) / (threads / 32);
  if (n > 2048 / threads) n = 2048 / threads;
  if (n > 226 * 1024 / (smem + 8 * 1024)) n = 226 * 1024 / (smem + 8 * 1024);
  return 148 * (n > 1 ? n : 1);
}

template <typename T, int V, int R>
static int rotary_launch_items(const RotaryArgs& a, bool inter, int threads, int L, cudaStream_t st) {
  auto* k = inter ? rotary_items_kernel<T, V, true, R> : rotary_items_kernel<T, V, false, R>;
  const int smem = Ahead<T, V, R, false>::bytes(threads, ROT_AHEAD), most = resident(threads, fwd_regs(R), smem);
  static std::atomic<unsigned long long> allowed[2];
  if (!allow_smem(k, ROT_SMEM, allowed[inter])) return T2T_ERR_CUDA;
  k<<<(unsigned)(a.rows < most ? a.rows : most), threads, smem, st>>>(a, L);
  return cudaGetLastError() == cudaSuccess ? T2T_OK : T2T_ERR_CUDA;
}
template <typename T, int V, int R>
static int rotary_launch_items_grad(const RotaryArgs& a, bool inter, int threads, int L, int& blocks, cudaStream_t st) {
  auto* k = inter ? rotary_items_grad_kernel<T, V, true, R> : rotary_items_grad_kernel<T, V, false, R>;
  int smem = Ahead<T, V, R, true>::bytes(threads, ROT_GRAD_AHEAD);
  const int join = 2 * (threads / L) * a.D * 4;
  if (a.norm == T2T_NORM_HEAD && smem < join) smem = join;
  static std::atomic<unsigned long long> allowed[2];
  if (!allow_smem(k, ROT_SMEM, allowed[inter])) return T2T_ERR_CUDA;
  const int most = resident(threads, grad_regs(R, V), smem);
  if (blocks > most) blocks = most;
  k<<<blocks, threads, smem, st>>>(a, L);
  return cudaGetLastError() == cudaSuccess ? T2T_OK : T2T_ERR_CUDA;
}

// blocks: of the gradient, at most on entry, used on return.
template <typename T, int V>
static int rotary_launch_v(const RotaryArgs& a, bool inter, bool grad, int& blocks, cudaStream_t st) {
  int L = 1;
  while (L < 32 && L < a.D / (2 * V)) L <<= 1;
  const int heads = a.side[0].heads + a.side[1].heads;
  if constexpr (V * sizeof(T) == 16) {
    const bool weights = (((uintptr_t)a.side[0].weight | (uintptr_t)a.side[1].weight) & 15u) == 0;
    if (L * 2 * V >= a.D && weights) {
      // Three warps a token where its heads allow it, else six, else a block: more tokens in flight, fewer threads at each meeting (12 +
      // 12 heads: 98 us with three warps and two items a thread, 142 with six and one).  The gradient takes four items a
      // thread last: they leave a block of five warps on an SM (40 + 40 heads: 1,850 us, 1,340 with two).  With few
      // tokens, as many threads as have work.
      int t = 0, R = 1;
      for (const int most : {a.rows > 148 ? 96 : 256, 192, 256, 320, 512})
        for (R = 1; R <= (grad ? 2 : 4); R *= 2)
          if (most <= (grad ? grad_threads(R, V) : fwd_threads(R)) && (t = items_threads(heads, L, R, a.rd / 2, most))) goto found;
      if (grad) t = items_threads(heads, L, R, a.rd / 2, grad_threads(R, V));
    found:
      if (t && !grad) {
        if (R == 1) return rotary_launch_items<T, V, 1>(a, inter, t, L, st);
        if (R == 2) return rotary_launch_items<T, V, 2>(a, inter, t, L, st);
        return rotary_launch_items<T, V, 4>(a, inter, t, L, st);
      }
      if (t) {
        if (R == 1) return rotary_launch_items_grad<T, V, 1>(a, inter, t, L, blocks, st);
        if (R == 2) return rotary_launch_items_grad<T, V, 2>(a, inter, t, L, blocks, st);
        return rotary_launch_items_grad<T, V, 4>(a, inter, t, L, blocks, st);
      }
    }
    if (a.rd % (2 * V)) return rotary_launch_v<T, V / 2>(a, inter, grad, blocks, st);
  }
  if (!grad) {
    auto* k = inter ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>;
    k<<<(unsigned)a.rows, 256, 0, st>>>(a, L);
  } else {
    auto* k = inter ? rotary_grad_kernel<T, V, true> : rotary_grad_kernel<T, V, false>;
    const int smem = heads * a.D * 4;
    static std::atomic<unsigned long long> allowed[2];
    if (!allow_smem(k, ROT_SMEM, allowed[inter])) return T2T_ERR_CUDA;
    k<<<blocks, 256, smem, st>>>(a, L);
  }
  return cudaGetLastError() == cudaSuccess ? T2T_OK : T2T_ERR_CUDA;
}

template <typename T>
static int rotary_launch_t(const RotaryArgs& a, bool inter, bool grad, int& blocks, cudaStream_t st) {
  switch (rotary_width(a, sizeof(T), inter, grad)) {
    case 8: if constexpr (sizeof(T) == 2) return rotary_launch_v<T, 8>(a, inter, grad, blocks, st);
    case 4: return rotary_launch_v<T, 4>(a, inter, grad, blocks, st);
    case 2: return rotary_launch_v<T, 2>(a, inter, grad, blocks, st);
    default: return rotary_launch_v<T, 1>(a, inter, grad, blocks, st);
  }
}

static int rotary_launch(const RotaryArgs& a, int dtype, bool inter, bool grad, int& blocks, cudaStream_t st) {
  if (dtype == T2T_BF16) return rotary_launch_t<__nv_bfloat16>(a, inter, grad, blocks, st);
  if (dtype == T2T_FP16) return rotary_launch_t<__half>(a, inter, grad, blocks, st);
  return rotary_launch_t<float>(a, inter, grad, blocks, st);
}

static bool rotary_args_ok(int batch, int N, int Hq, int Hk, int D, int rd, int norm, int dtype, int weight_dtype,
                           int pos_bytes) {
  return batch > 0 && N > 0 && Hq > 0 && Hk >= 0 && D > 0 && D % 2 == 0 && rd > 0 && rd % 2 == 0 && rd <= D &&
         rd / 2 <= ROT_MAX_PAIRS && norm >= T2T_NORM_NONE && norm <= T2T_NORM_ROW && elem_known(dtype) &&
         (weight_dtype == dtype || weight_dtype == T2T_FP32) && (pos_bytes == 4 || pos_bytes == 8) &&
         (long long)batch * N <= 0x7fffffffLL && (long long)(Hq + Hk) * D <= 0x7fffffffLL;
}

}  // namespace t2t

using namespace t2t;

extern "C" int t2t_rotary(const void* q, const void* k, void* q_out, void* k_out, const void* q_weight, const void* k_weight,
                          int weight_dtype, const void* positions, int pos_bytes, long long pos_axis_stride,
                          long long pos_batch_stride, const long long* turns, const int* axis, const long long* strides,
                          int batch, int N, int Hq, int Hk, int D, int rotary_dim, int interleaved, int inverse, int norm,
                          float mscale, float eps, int dtype, cudaStream_t stream) {
  if (!rotary_args_ok(batch, N, Hq, Hk, D, rotary_dim, norm, dtype, weight_dtype, pos_bytes)) return T2T_ERR_ARG;
  if (!q || !q_out || (Hk && (!k || !k_out)) || !positions || !turns || !axis || !strides) return T2T_ERR_ARG;
  if (norm && (!q_weight || (Hk && !k_weight) || inverse)) return T2T_ERR_ARG;
  RotaryArgs a = {};
  const long long* s = strides;
  a.side[0] = {q, nullptr, q_out, q_weight, Hq, s[0], s[1], s[2], 0, 0, 0, s[6], s[7], s[8]};
  a.side[1] = {k, nullptr, k_out, k_weight, Hk, s[3], s[4], s[5], 0, 0, 0, s[9], s[10], s[11]};
  a.pos = positions;
  a.turns = turns;
  a.axis = axis;
  a.pos_axis = pos_axis_stride;
  a.pos_batch = pos_batch_stride;
  a.pos_bytes = pos_bytes;
  a.N = N;
  a.D = D;
  a.rd = rotary_dim;
  a.inverse = inverse;
  a.norm = norm;
  a.weight_dtype = weight_dtype;
  a.rows = (long long)batch * N;
  a.mscale = mscale;
  a.eps = eps;
  int blocks = 0;
  return rotary_launch(a, dtype, interleaved != 0, false, blocks, stream);
}

extern "C" size_t t2t_rotary_grad_ws_bytes(int Hq, int Hk, int D, int norm) {
  if (Hq <= 0 || Hk < 0 || D <= 0) return 0;
  const size_t each = norm == T2T_NORM_ROW ? (size_t)(Hq + Hk) * D : (size_t)2 * D;
  return each * ROT_GRAD_BLOCKS * sizeof(float);
}

extern "C" int t2t_rotary_grad(const void* dq, const void* dk, const void* q, const void* k, void* dq_out, void* dk_out,
                               const void* q_weight, const void* k_weight, int weight_dtype, float* dq_weight,
                               float* dk_weight, const void* positions, int pos_bytes, long long pos_axis_stride,
                               long long pos_batch_stride, const long long* turns, const int* axis, const long long* strides,
                               int batch, int N, int Hq, int Hk, int D, int rotary_dim, int interleaved, int norm,
                               float mscale, float eps, int dtype, void* ws, size_t ws_bytes, cudaStream_t stream) {
  if (!rotary_args_ok(batch, N, Hq, Hk, D, rotary_dim, norm, dtype, weight_dtype, pos_bytes) || norm == T2T_NORM_NONE)
    return T2T_ERR_ARG;
  if (!dq || !q || !dq_out || !q_weight || !dq_weight || !positions || !turns || !axis || !strides || !ws) return T2T_ERR_ARG;
  if (Hk && (!dk || !k || !dk_out || !k_weight || !dk_weight)) return T2T_ERR_ARG;
  if (ws_bytes < t2t_rotary_grad_ws_bytes(Hq, Hk, D, norm)) return T2T_ERR_WORKSPACE;
  if ((long long)(Hq + Hk) * D * 4 > ROT_SMEM) return T2T_ERR_TOO_LARGE;      // the sums of dw in shared memory
  RotaryArgs a = {};
  const long long* s = strides;
  a.side[0] = {q, dq, dq_out, q_weight, Hq, s[0], s[1], s[2], s[6], s[7], s[8], s[12], s[13], s[14]};
  a.side[1] = {k, dk, dk_out, k_weight, Hk, s[3], s[4], s[5], s[9], s[10], s[11], s[15], s[16], s[17]};
  a.pos = positions;
  a.turns = turns;
  a.axis = axis;
  a.pos_axis = pos_axis_stride;
  a.pos_batch = pos_batch_stride;
  a.pos_bytes = pos_bytes;
  a.N = N;
  a.D = D;
  a.rd = rotary_dim;
  a.inverse = 1;
  a.norm = norm;
  a.weight_dtype = weight_dtype;
  a.rows = (long long)batch * N;
  a.mscale = mscale;
  a.eps = eps;
  a.partial = static_cast<float*>(ws);
  int blocks = a.rows < ROT_GRAD_BLOCKS ? (int)a.rows : ROT_GRAD_BLOCKS;
  const int rc = rotary_launch(a, dtype, interleaved != 0, true, blocks, stream);
  if (rc != T2T_OK) return rc;
  const int first = norm == T2T_NORM_ROW ? Hq * D : D, total = norm == T2T_NORM_ROW ? (Hq + Hk) * D : 2 * D;
  const int used = Hk ? total : first;
  rotary_weight_grad_kernel<<<cdiv(used, 32), 256, 0, stream>>>(a.partial, blocks, total, first, used, dq_weight, dk_weight);
  return cudaGetLastError() == cudaSuccess ? T2T_OK : T2T_ERR_CUDA;
}
