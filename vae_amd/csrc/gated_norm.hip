// The two norms around a residual block, its gate and its residual scale in one pass, and the backward pass (gfx950).
//
//   u = norm(b) * gp + bp   (or b)        y = r + s * act(gate) * u        h = norm(y) * gn + bn
//
// norm is (t - mean) / sqrt(var + eps) or t / sqrt(mean t^2 + eps); y is rounded to its type before h is formed, so that the
// backward pass, which reads y again, works on the values that the forward pass used.  With dt the gradient that reaches y,
//
//   dt = dy + N_y(dh * gn)     dr = dt     dgate = dt * s * u * act'     ds = sum dt * act * u
//   dgp = sum dt * act * s * nb    dbp = sum dt * act * s    db = N_b(dt * act * s * gp)    dgn = sum dh * ny    dbn = sum dh
//   N(d) = (d - n * mean(d * n) [- mean d]) / sigma
//
// HBM-bound: the forward pass reads r, b and the gate and writes y and h, the backward pass reads y, b, the gate, dy and dh and
// writes dr, db and dgate, each once: a row lives in registers from its loads to its stores, in 32 bits.  A wave takes a row of
// up to 64 16-byte pieces, a workgroup of up to 1024 threads a longer one, one to four pieces per thread.  A workgroup walks
// over rows; the gradients of the vectors over columns are summed in registers over its rows, written once per workgroup, and
// added up in a second launch in a fixed order (no atomics: same bits every time).  32768 x 4096 bf16 with a full gate: forward
// 269 us = 4.9 TB/s, backward 440 us = 4.8 TB/s (a large copy: 4.9); without the next row's loads ahead of this row's work
// some 60 and 260 us more.  Rows on 16 waves (16 bits or fp32 beyond 4096 or 2048 columns) have no room for those loads, and from
// 4097 columns on the backward pass keeps part of its column sums in scratch: 16384 x 8192 bf16 forward 361 us, both 1646; 8192 x
// 16384 293 and 2425.
#include "../../include/vae_amd.h"
#include "common.h"

namespace {

typedef vae_gated_norm Args;
constexpr int N_COL = 5;                 // column sums: d gn, d s, d gp, d bn, d bp
constexpr int FWD_WAVES = 4;
constexpr int bwd_waves(int nw) { return nw <= 8 ? 2 : 4; }

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
// rows of an odd width start at any element: the hardware takes 16-byte accesses at any address, only the type has to say so
typedef u4 u4_any __attribute__((aligned(2)));

template <typename T> constexpr int PIECE = 16 / (int)sizeof(T);

// One piece as it is in memory: four registers whatever the type (as an array of elements the compiler would spread 16-bit
// ones over eight).
template <typename T> struct Raw {
  u4 q;
  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(q[j]);
    } else {
      const uint32_t w = q[j >> 1];
      if constexpr (__is_same(T, __bf16)) return __uint_as_float((j & 1) ? w & 0xffff0000u : w << 16);
      else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> (16 * (j & 1))));
    }
  }
};
template <typename T> __device__ __forceinline__ Raw<T> pack(const float (&v)[PIECE<T>]) {
  Raw<T> w;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      w.q[k] = __float_as_uint(v[k]);
    } else {
      typedef T t2 __attribute__((ext_vector_type(2)));
      t2 p;
      p[0] = (T)v[2 * k];
      p[1] = (T)v[2 * k + 1];
      w.q[k] = __builtin_bit_cast(uint32_t, p);
    }
  }
  return w;
}
// Elements of a row from column c on, those past D as zeros.  The last piece of a row is read where it ends at column D and
// shifted down, so that every piece is one unconditional 16-byte load (element by element, the loads of all operands' tails
// together set the registers of the whole kernel).
template <typename T> __device__ __forceinline__ Raw<T> load(const T* __restrict__ row, uint32_t c, uint32_t D) {
  constexpr uint32_t P = PIECE<T>;
  Raw<T> w;
  if (D >= P) {
    const uint32_t at = min(c, D - P);
    w.q = *reinterpret_cast<const u4_any*>(row + at);
    if (c > at) {
      const uint32_t by = (c - at) * (uint32_t)sizeof(T);          // bytes to drop
      if (by & 8) w.q[0] = w.q[2], w.q[1] = w.q[3], w.q[2] = w.q[3] = 0;
      if (by & 4) w.q[0] = w.q[1], w.q[1] = w.q[2], w.q[2] = w.q[3], w.q[3] = 0;
      if (sizeof(T) == 2 && (by & 2)) {
        w.q[0] = w.q[0] >> 16 | w.q[1] << 16;
        w.q[1] = w.q[1] >> 16 | w.q[2] << 16;
        w.q[2] = w.q[2] >> 16 | w.q[3] << 16;
        w.q[3] >>= 16;
      }
      if (c >= D) w.q = (u4)0;
    }
  } else {                                                         // rows shorter than a piece
    w.q = (u4)0;
    if (c == 0)
#pragma unroll
      for (uint32_t j = 0; j < P; ++j) {
        if (j >= D) continue;
        if constexpr (sizeof(T) == 4) w.q[j] = __float_as_uint(row[j]);
        else w.q[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[j] << (16 * (j & 1));
      }
  }
  return w;
}
template <typename T> __device__ __forceinline__ void store(T* __restrict__ row, uint32_t c, uint32_t D, const Raw<T>& w) {
  if (c + PIECE<T> <= D) {
    *reinterpret_cast<u4_any*>(row + c) = w.q;
  } else {
#pragma unroll
    for (int j = 0; j < PIECE<T>; ++j) {
      if (c + j >= D) continue;
      if constexpr (sizeof(T) == 4) row[c + j] = w[j];
      else reinterpret_cast<uint16_t*>(row)[c + j] = (uint16_t)(w.q[j >> 1] >> (16 * (j & 1)));
    }
  }
}
// A piece of a vector over columns, of the rows' type or float, as it is in memory; absent: `none` throughout.
template <typename V, int P> struct Vec {
  static constexpr int Q = P * (int)sizeof(V) / 16;
  Raw<V> w[Q];
  __device__ __forceinline__ float operator[](int j) const { return w[j / PIECE<V>][j % PIECE<V>]; }
};
template <typename V, int P> __device__ __forceinline__ Vec<V, P> column(const void* p, uint32_t c, uint32_t D, float none) {
  Vec<V, P> o;
#pragma unroll
  for (int i = 0; i < Vec<V, P>::Q; ++i) {
    if (p) {
      o.w[i] = load(reinterpret_cast<const V*>(p), c + i * PIECE<V>, D);
    } else {
      float v[PIECE<V>];
#pragma unroll
      for (int j = 0; j < PIECE<V>; ++j) v[j] = none;
      o.w[i] = pack<V>(v);
    }
  }
  return o;
}

// sums of K values over the row's threads: a wave by DPP, a workgroup of NW waves through `red` (one barrier; the caller
// alternates between two buffers, so that a fast wave does not overwrite what a slow one still reads)
template <int NW, int K> __device__ __forceinline__ void row_sums(float (&v)[K], float* __restrict__ red) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum_dpp(v[k]);
  if (NW > 1) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[k * NW + w] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) s += red[k * NW + i];
      v[k] = s;
    }
  }
}

// Both within 3e-7 of themselves up to |v| = 4 (v * log2 e is rounded: |v| 2^-24 beyond): the hardware's exponential and
// reciprocal (an ulp each) leave the registers that the correctly rounded division and the library's functions take, times 8
// elements, to the loads.
__device__ __forceinline__ float sigmoid_f(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.44269504088896341f));
}
__device__ __forceinline__ float tanh_f(float v) {
  const float t = fabsf(v), e = __builtin_amdgcn_exp2f(t * -2.88539008177792681f), q = t * t;
  // near 0 the quotient would cancel: the Taylor series, whose next term is 1382 / 155925 t^11
  const float far = (1.f - e) * __builtin_amdgcn_rcpf(1.f + e);
  const float near = t * fmaf(q, fmaf(q, fmaf(q, fmaf(q, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  return copysignf(t < 0.3f ? near : far, v);
}
// act(gate) of one piece
template <typename T> __device__ __forceinline__ void act_of(int act, const Raw<T>& g, float (&a)[PIECE<T>]) {
  constexpr int P = PIECE<T>;
  if (act == VAE_GATE_SIGMOID) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      a[j] = sigmoid_f(g[j]);
      if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  } else if (act == VAE_GATE_TANH) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      a[j] = tanh_f(g[j]);
      if (j % 2 == 1) __builtin_amdgcn_sched_barrier(0);
    }
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j) a[j] = g[j];
  }
}
// act' as a polynomial of a = act(gate): a - a^2, 1 - a^2 or 1
struct Slope {
  float k0, k1, k2;
  __device__ __forceinline__ explicit Slope(int act)
      : k0(act == VAE_GATE_SIGMOID ? 0.f : 1.f), k1(act == VAE_GATE_SIGMOID ? 1.f : 0.f), k2(act == VAE_GATE_IDENTITY ? 0.f : -1.f) {}
  __device__ __forceinline__ float operator()(float a) const { return fmaf(a, fmaf(k2, a, k1), k0); }
};
template <typename T> __device__ __forceinline__ float row_gate(const Args& a, int64_t row) {
  const Raw<T> w = load(reinterpret_cast<const T*>(a.gate) + row * a.ld_gate, 0, 1);
  float v[PIECE<T>];
  act_of<T>(a.act, w, v);
  return v[0];
}
// Values behind this are formed again from their 16-bit originals instead of being kept in 32 bits across a reduction.
__device__ __forceinline__ void reread(u4& q) { asm volatile("" : "+v"(q)); }

// NW waves share a row (NW = 1: four rows to a workgroup), ITEMS pieces per thread
template <typename T, typename V, int NW, int ITEMS>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64, FWD_WAVES) void gated_norm_fwd_kernel(Args a) {
  constexpr int P = PIECE<T>, TPR = NW * 64, RPW = NW == 1 ? 4 : 1;
  __shared__ float red[2][2 * NW];
  const uint32_t D = (uint32_t)a.D, lane = NW == 1 ? (threadIdx.x & 63) : threadIdx.x;
  const int first = blockIdx.x * RPW + (NW == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);   // (rows are uniform: scalar bases)
  const float inv_d = 1.f / (float)D;
  const bool layer = a.kind == VAE_NORM_LAYER, post = a.post_weight != nullptr;
  constexpr bool AHEAD = NW <= 8;                                  // (16 waves have 128 registers each: no room)
  struct In {
    Raw<T> r[ITEMS], b[ITEMS], g[ITEMS];
    float act;
  };
  auto fetch = [&](In& in, int64_t row) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t c = (uint32_t)((i * TPR + lane) * P);
      in.b[i] = load(reinterpret_cast<const T*>(a.b) + row * a.ld_b, c, D);
      in.r[i] = load(reinterpret_cast<const T*>(a.r) + row * a.ld_r, c, D);
      if (a.gate_mode == VAE_GATE_FULL) in.g[i] = load(reinterpret_cast<const T*>(a.gate) + row * a.ld_gate, c, D);
    }
    in.act = a.gate_mode == VAE_GATE_ROW ? row_gate<T>(a, row) : 1.f;
  };
  Vec<V, P> gn[ITEMS], bn[ITEMS], sc[ITEMS], gp[ITEMS], bp[ITEMS];
  auto columns = [&]() {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t c = (uint32_t)((i * TPR + lane) * P);
      gp[i] = column<V, P>(a.post_weight, c, D, 1.f);
      bp[i] = column<V, P>(a.post_bias, c, D, 0.f);
      sc[i] = column<V, P>(a.scale, c, D, 1.f);
      gn[i] = column<V, P>(a.norm_weight, c, D, 1.f);
      bn[i] = column<V, P>(a.norm_bias, c, D, 0.f);
    }
  };
  const int64_t stride = (int64_t)gridDim.x * RPW;
  In in, next;
  if (AHEAD && first < a.N) fetch(next, first), columns();
  int flip = 0;
  for (int64_t row = first; row < a.N; row += stride) {
    if (AHEAD) {                                                   // the next row is on its way while this one is worked on
      in = next;
      if (row + stride < a.N) fetch(next, row + stride);
    } else {
      columns();
      fetch(in, row);
    }
    auto &wr = in.r, &wb = in.b, &wg = in.g;
    const float row_act = in.act;
    // mean and 1 / sigma of the block's output, from its deviations
    float x[ITEMS][P];
    auto moments = [&](float& mean, float& inv) {
      mean = 0.f;
      if (layer) {
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
          for (int j = 0; j < P; ++j) s[0] += x[i][j];             // columns past D hold 0
        row_sums<NW, 1>(s, red[flip]);
        flip ^= 1;
        mean = s[0] * inv_d;
      }
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const float d = (i * TPR + lane) * P + j < D ? x[i][j] - mean : 0.f;
          s[0] = fmaf(d, d, s[0]);
        }
      row_sums<NW, 1>(s, red[flip]);
      flip ^= 1;
      inv = 1.f / sqrtf(s[0] * inv_d + a.eps);
    };
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) x[i][j] = wb[i][j];
    float mean_b = 0.f, inv_b = 1.f, mean_y, inv_y;
    if (post) moments(mean_b, inv_b);
    T* ry = reinterpret_cast<T*>(a.y) + row * a.D;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t c = (uint32_t)((i * TPR + lane) * P);
      float act[P], out[P];
#pragma unroll
      for (int j = 0; j < P; ++j) act[j] = row_act;
      if (a.gate_mode == VAE_GATE_FULL) act_of<T>(a.act, wg[i], act);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        float u = x[i][j];
        if (post) u = fmaf((u - mean_b) * inv_b, gp[i][j], bp[i][j]);
        out[j] = fmaf(u * sc[i][j], act[j], wr[i][j]);
      }
      const Raw<T> wy = pack<T>(out);
      store(ry, c, D, wy);
#pragma unroll
      for (int j = 0; j < P; ++j) x[i][j] = c + j < D ? wy[j] : 0.f;
    }
    moments(mean_y, inv_y);
    T* rh = reinterpret_cast<T*>(a.h) + row * a.D;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t c = (uint32_t)((i * TPR + lane) * P);
      float out[P];
#pragma unroll
      for (int j = 0; j < P; ++j) out[j] = fmaf((x[i][j] - mean_y) * inv_y, gn[i][j], bn[i][j]);
      store(rh, c, D, pack<T>(out));
    }
    if (a.stats && lane == 0) *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(mean_b, inv_b, mean_y, inv_y);
  }
}

// BIAS: whether a gradient of either norm's bias is asked for; without, their column sums are not carried.
template <typename T, typename V, int NW, int ITEMS, bool BIAS>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64, bwd_waves(NW)) void gated_norm_bwd_kernel(Args a, float* __restrict__ partial) {
  constexpr int P = PIECE<T>, TPR = NW * 64, RPW = NW == 1 ? 4 : 1;
  __shared__ float red[2][3 * NW];
  const uint32_t D = (uint32_t)a.D, lane = NW == 1 ? (threadIdx.x & 63) : threadIdx.x;
  const int first = blockIdx.x * RPW + (NW == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);   // (rows are uniform: scalar bases)
  const float inv_d = 1.f / (float)D;
  const bool layer = a.kind == VAE_NORM_LAYER, post = a.post_weight != nullptr;
  constexpr int COLS = BIAS ? N_COL : 3;
  float acc[COLS][ITEMS][P];
#pragma unroll
  for (int k = 0; k < COLS; ++k)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) acc[k][i][j] = 0.f;
  const Slope slope(a.act);
  constexpr bool AHEAD = NW <= 8;                                  // (16 waves have 128 registers each: no room)
  struct In {
    Raw<T> y[ITEMS], dh[ITEMS], dy[ITEMS], b[ITEMS], g[ITEMS];
    float4 st;                                                     // mean_b, inv_b, mean_y, inv_y
    float act;
  };
  auto fetch = [&](In& in, int64_t row) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t c = (uint32_t)((i * TPR + lane) * P);
      in.y[i] = load(reinterpret_cast<const T*>(a.y) + row * a.D, c, D);
      in.dh[i].q = in.dy[i].q = (u4)0;
      if (a.dh) in.dh[i] = load(reinterpret_cast<const T*>(a.dh) + row * a.ld_dh, c, D);
      if (a.dy) in.dy[i] = load(reinterpret_cast<const T*>(a.dy) + row * a.ld_dy, c, D);
      in.b[i] = load(reinterpret_cast<const T*>(a.b) + row * a.ld_b, c, D);
      if (a.gate_mode == VAE_GATE_FULL) in.g[i] = load(reinterpret_cast<const T*>(a.gate) + row * a.ld_gate, c, D);
    }
    in.st = *reinterpret_cast<const float4*>(a.stats + row * 4);
    in.act = a.gate_mode == VAE_GATE_ROW ? row_gate<T>(a, row) : 1.f;
  };
  Vec<V, P> gn[ITEMS], sc[ITEMS], gp[ITEMS], bp[ITEMS];
  auto columns = [&]() {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t c = (uint32_t)((i * TPR + lane) * P);
      gn[i] = column<V, P>(a.norm_weight, c, D, 1.f);
      sc[i] = column<V, P>(a.scale, c, D, 1.f);
      gp[i] = column<V, P>(a.post_weight, c, D, 1.f);
      bp[i] = column<V, P>(a.post_bias, c, D, 0.f);
    }
  };
  const int64_t stride = (int64_t)gridDim.x * RPW;
  In in, next;
  if (AHEAD && first < a.N) columns(), fetch(next, first);
  int flip = 0;
  for (int64_t row = first; row < a.N; row += stride) {
    if (AHEAD) {                                                   // the next row is on its way while this one is worked on
      in = next;
      if (row + stride < a.N) fetch(next, row + stride);
    } else {
      columns();
      fetch(in, row);
    }
    auto &wy = in.y, &wb = in.b, &wg = in.g, &wdy = in.dy, &wdh = in.dh;
    const float4 st = in.st;
    const float row_act = in.act;
    float s1[2] = {0.f, 0.f};
    float t[ITEMS][P];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) {                               // past D: dh is 0, and with it every term
        const float dh = wdh[i][j], ny = (wy[i][j] - st.z) * st.w, dn = dh * gn[i][j];
        acc[0][i][j] = fmaf(dh, ny, acc[0][i][j]);
        if (BIAS) acc[COLS - 2][i][j] += dh;
        s1[0] = fmaf(dn, ny, s1[0]);
        s1[1] += dn;
        if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    row_sums<NW, 2>(s1, red[flip]);
    flip ^= 1;
    const float c1 = s1[0] * inv_d, c2 = layer ? s1[1] * inv_d : 0.f;
    float s2[3] = {0.f, 0.f, 0.f};
    T* rdr = reinterpret_cast<T*>(a.dr) + row * a.D;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t c = (uint32_t)((i * TPR + lane) * P);
      float act[P], dr[P], dg[P];
#pragma unroll
      for (int j = 0; j < P; ++j) act[j] = row_act;
      if (a.gate_mode == VAE_GATE_FULL) act_of<T>(a.act, wg[i], act);
      reread(wy[i].q);
      reread(wdh[i].q);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float ny = (wy[i][j] - st.z) * st.w, dn = wdh[i][j] * gn[i][j];
        const float dt = c + j < D ? wdy[i][j] + (dn - ny * c1 - c2) * st.w : 0.f;
        dr[j] = dt;
        const float nb = post ? (wb[i][j] - st.x) * st.y : wb[i][j];
        const float u = post ? fmaf(nb, gp[i][j], bp[i][j]) : nb;
        const float dk = dt * u * sc[i][j];
        dg[j] = dk * slope(act[j]);
        s2[2] += dk;
        const float e = dt * act[j];
        acc[1][i][j] = fmaf(e, u, acc[1][i][j]);
        const float es = e * sc[i][j], d = es * gp[i][j];
        acc[2][i][j] = fmaf(es, nb, acc[2][i][j]);
        if (BIAS) acc[COLS - 1][i][j] += es;
        t[i][j] = post ? d : es;
        s2[0] = fmaf(d, nb, s2[0]);
        s2[1] += d;
        if (j % 2 == 1) __builtin_amdgcn_sched_barrier(0);        // (all at once the temporaries of 8 elements cost a wave)
      }
      store(rdr, c, D, pack<T>(dr));
      if (a.gate_mode == VAE_GATE_FULL && a.dgate) store(reinterpret_cast<T*>(a.dgate) + row * a.D, c, D, pack<T>(dg));
    }
    float c3 = 0.f, c4 = 0.f;
    if (post || a.gate_mode == VAE_GATE_ROW) {
      row_sums<NW, 3>(s2, red[flip]);
      flip ^= 1;
      c3 = post ? s2[0] * inv_d : 0.f;
      c4 = post && layer ? s2[1] * inv_d : 0.f;
      if (a.gate_mode == VAE_GATE_ROW && a.dgate && lane == 0) reinterpret_cast<T*>(a.dgate)[row] = (T)(s2[2] * slope(row_act));
    }
    T* rdb = reinterpret_cast<T*>(a.db) + row * a.D;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      float db[P];
      reread(wb[i].q);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float nb = (wb[i][j] - st.x) * st.y;
        db[j] = post ? (t[i][j] - nb * c3 - c4) * st.y : t[i][j];
      }
      store(rdb, (uint32_t)((i * TPR + lane) * P), D, pack<T>(db));
    }
  }
  if (!partial) return;
  // this workgroup's sums: partial[column sum][workgroup][D]
  const bool want[N_COL] = {a.dnorm_weight != nullptr, a.dscale != nullptr, a.dpost_weight != nullptr, a.dnorm_bias != nullptr,
                            a.dpost_bias != nullptr};
  if (NW == 1) {                                                  // four waves hold the same columns: waves 1..3 hand theirs over
    __shared__ float part[3][64 * P];
    const int w = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
      if (!want[k]) continue;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        __syncthreads();
        if (w)
#pragma unroll
          for (int j = 0; j < P; ++j) part[w - 1][j * 64 + lane] = acc[k][i][j];
        __syncthreads();
        if (!w) {
          const uint32_t c = (uint32_t)((i * TPR + lane) * P);
#pragma unroll
          for (int j = 0; j < P; ++j) {
            const float s = ((acc[k][i][j] + part[0][j * 64 + lane]) + part[1][j * 64 + lane]) + part[2][j * 64 + lane];
            if (c + j < D) partial[((int64_t)k * gridDim.x + blockIdx.x) * D + c + j] = s;
          }
        }
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
      if (!want[k]) continue;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const uint32_t c = (uint32_t)((i * TPR + lane) * P);
#pragma unroll
        for (int j = 0; j < P; ++j)
          if (c + j < D) partial[((int64_t)k * gridDim.x + blockIdx.x) * D + c + j] = acc[k][i][j];
      }
    }
  }
}

// out[k][c] = sum over the workgroups' partials: 64 columns to a workgroup of 16 waves, each of which adds every 16th partial,
// eight loads in flight; the 16 sums are added in order
struct Outs {
  void* out[N_COL];
  int elem;                              // VAE_ADAMW_F32 / BF16 / F16
};
__global__ __launch_bounds__(1024) void gated_norm_cols_kernel(const float* __restrict__ partial, int groups, int D, Outs o) {
  __shared__ float red[16][64];
  const int k = blockIdx.y, c = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  if (!o.out[k]) return;
  float s = 0.f;
  if (c < D) {
    const float* p = partial + (int64_t)k * groups * D + c;
    int g = w;
    for (; g + 7 * 16 < groups; g += 8 * 16) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[(int64_t)(g + 16 * i) * D];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
    for (; g < groups; g += 16) s += p[(int64_t)g * D];
  }
  red[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && c < D) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x & 63];
    if (o.elem == VAE_ADAMW_F32) reinterpret_cast<float*>(o.out[k])[c] = s;
    else if (o.elem == VAE_ADAMW_BF16) reinterpret_cast<__bf16*>(o.out[k])[c] = (__bf16)s;
    else reinterpret_cast<_Float16*>(o.out[k])[c] = (_Float16)s;
  }
}

// waves per row and pieces per thread for a row of `pieces` 16-byte pieces: the fewest waves that hold one piece per thread,
// which keeps the backward pass's column sums at 5 * 8 registers; beyond 16 waves more pieces
struct Shape {
  int nw, items;
};
Shape shape_of(int64_t pieces) {
  if (pieces <= 64) return {1, 1};
  if (pieces <= 128) return {2, 1};
  if (pieces <= 256) return {4, 1};
  if (pieces <= 512) return {8, 1};
  if (pieces <= 1024) return {16, 1};
  if (pieces <= 2048) return {16, 2};
  return {16, 4};
}
// As many workgroups as are resident at once on 256 CUs: the forward pass leaves room for 4 waves per SIMD, the backward pass
// for bwd_waves(); at least one row each.
int groups_of(int64_t rows, const Shape& s, bool bwd) {
  const int waves = s.nw == 1 ? 4 : s.nw, per_cu = (bwd ? bwd_waves(s.nw) : FWD_WAVES) * 4 / waves;
  const int64_t need = s.nw == 1 ? (rows + 3) / 4 : rows, fit = 256 * (per_cu < 1 ? 1 : per_cu);
  return (int)(need < fit ? need : fit);
}
int64_t pieces_of(int64_t D, int dtype) {
  const int64_t p = dtype == VAE_ADAMW_F32 ? 4 : 8;
  return (D + p - 1) / p;
}

template <typename T, typename V> void launch(const Args& a, bool bwd, float* partial, const Shape& s, int groups, hipStream_t st) {
#define VAE_GN(NW, ITEMS)                                                                                    \
  if (s.nw == NW && s.items == ITEMS) {                                                                      \
    if (bwd && (a.dnorm_bias || a.dpost_bias))                                                               \
      gated_norm_bwd_kernel<T, V, NW, ITEMS, true><<<groups, NW == 1 ? 256 : NW * 64, 0, st>>>(a, partial);  \
    else if (bwd)                                                                                            \
      gated_norm_bwd_kernel<T, V, NW, ITEMS, false><<<groups, NW == 1 ? 256 : NW * 64, 0, st>>>(a, partial); \
    else                                                                                                     \
      gated_norm_fwd_kernel<T, V, NW, ITEMS><<<groups, NW == 1 ? 256 : NW * 64, 0, st>>>(a);                 \
    return;                                                                                                  \
  }
  VAE_GN(1, 1) VAE_GN(2, 1) VAE_GN(4, 1) VAE_GN(8, 1) VAE_GN(16, 1) VAE_GN(16, 2)
  if constexpr (sizeof(T) == 4) { VAE_GN(16, 4) }
#undef VAE_GN
}

void dispatch(const Args& a, bool bwd, float* partial, hipStream_t st) {
  const Shape s = shape_of(pieces_of(a.D, a.dtype));
  const int groups = groups_of(a.N, s, bwd);
  const bool f = a.vectors_f32;
  if (a.dtype == VAE_ADAMW_F32) launch<float, float>(a, bwd, partial, s, groups, st);
  else if (a.dtype == VAE_ADAMW_BF16) f ? launch<__bf16, float>(a, bwd, partial, s, groups, st) : launch<__bf16, __bf16>(a, bwd, partial, s, groups, st);
  else f ? launch<_Float16, float>(a, bwd, partial, s, groups, st) : launch<_Float16, _Float16>(a, bwd, partial, s, groups, st);
}

int check(const Args* a, const char* who) {
  VAE_REQUIRE(a, "%s: null arguments", who);
  VAE_REQUIRE(a->dtype >= 0 && a->dtype <= 2, "%s: unknown dtype %d", who, a->dtype);
  VAE_REQUIRE(a->N >= 0 && a->D >= 1 && a->D <= VAE_GATED_NORM_MAX_D, "%s: N >= 0 and 1 <= D <= %d needed", who, VAE_GATED_NORM_MAX_D);
  VAE_REQUIRE(a->kind == VAE_NORM_RMS || a->kind == VAE_NORM_LAYER, "%s: unknown norm %d", who, a->kind);
  VAE_REQUIRE(a->gate_mode >= VAE_GATE_NONE && a->gate_mode <= VAE_GATE_FULL, "%s: unknown gate mode %d", who, a->gate_mode);
  VAE_REQUIRE(a->act >= VAE_GATE_IDENTITY && a->act <= VAE_GATE_TANH, "%s: unknown gate activation %d", who, a->act);
  VAE_REQUIRE(a->eps >= 0, "%s: negative eps", who);
  VAE_REQUIRE(!a->post_bias || a->post_weight, "%s: post_bias needs post_weight", who);
  VAE_REQUIRE(a->N == 0 || (a->b && a->y && (a->gate_mode == VAE_GATE_NONE || a->gate)), "%s: null pointer", who);
  const uintptr_t bad = a->dtype == VAE_ADAMW_F32 ? 3 : 1;
  const void* rows[] = {a->r, a->b, a->gate, a->y, a->h, a->dy, a->dh, a->dr, a->db, a->dgate};
  for (const void* p : rows) VAE_REQUIRE((reinterpret_cast<uintptr_t>(p) & bad) == 0, "%s: a pointer is not aligned to its element", who);
  const void* vectors[] = {a->norm_weight, a->norm_bias, a->scale, a->post_weight, a->post_bias, a->dnorm_weight, a->dnorm_bias, a->dscale,
                           a->dpost_weight, a->dpost_bias};
  for (const void* p : vectors)
    VAE_REQUIRE((reinterpret_cast<uintptr_t>(p) & (a->vectors_f32 ? 3 : bad)) == 0, "%s: a vector is not aligned to its element", who);
  VAE_REQUIRE((reinterpret_cast<uintptr_t>(a->stats) & 15u) == 0, "%s: stats must be 16-byte aligned", who);
  return VAE_OK;
}

}  // namespace

extern "C" int64_t vae_gated_norm_workspace_bytes(int64_t N, int64_t D, int dtype) {
  if (N < 1 || D < 1 || D > VAE_GATED_NORM_MAX_D || dtype < 0 || dtype > 2) return 0;
  return (int64_t)N_COL * groups_of(N, shape_of(pieces_of(D, dtype)), true) * D * (int64_t)sizeof(float);
}

extern "C" int vae_gated_norm_fwd(const vae_gated_norm* a, void* stream) {
  if (int rc = check(a, "vae_gated_norm_fwd")) return rc;
  if (a->N == 0) return VAE_OK;
  VAE_REQUIRE(a->r && a->h, "vae_gated_norm_fwd: null pointer");
  dispatch(*a, false, nullptr, (hipStream_t)stream);
  VAE_CHECK_LAUNCH("vae_gated_norm_fwd");
  return VAE_OK;
}

extern "C" int vae_gated_norm_bwd(const vae_gated_norm* a, float* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check(a, "vae_gated_norm_bwd")) return rc;
  Outs o = {{a->dnorm_weight, a->dscale, a->dpost_weight, a->dnorm_bias, a->dpost_bias}, a->vectors_f32 ? VAE_ADAMW_F32 : a->dtype};
  bool cols = false;
  for (void* p : o.out) cols = cols || p;
  VAE_REQUIRE(a->N > 0, "vae_gated_norm_bwd: no rows");
  VAE_REQUIRE(a->stats && a->dr && a->db, "vae_gated_norm_bwd: null pointer");
  VAE_REQUIRE((!a->dpost_weight && !a->dpost_bias) || a->post_weight, "vae_gated_norm_bwd: gradients of a norm that is not there");
  VAE_REQUIRE(!cols || (workspace && workspace_bytes >= vae_gated_norm_workspace_bytes(a->N, a->D, a->dtype)),
              "vae_gated_norm_bwd: needs a workspace of vae_gated_norm_workspace_bytes()");
  hipStream_t st = (hipStream_t)stream;
  float* partial = cols ? workspace : nullptr;
  const int groups = groups_of(a->N, shape_of(pieces_of(a->D, a->dtype)), true);
  dispatch(*a, true, partial, st);
  VAE_CHECK_LAUNCH("vae_gated_norm_bwd");
  if (cols) {
    gated_norm_cols_kernel<<<dim3((unsigned)((a->D + 63) / 64), N_COL), 1024, 0, st>>>(partial, groups, (int)a->D, o);
    VAE_CHECK_LAUNCH("vae_gated_norm_bwd");
  }
  return VAE_OK;
}
