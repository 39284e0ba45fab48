// One AdamW step over many separate tensors (fp32, bf16 or fp16, mixed), moments in 32 or 8 bits (gfx950).
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// State is flat: tensor k owns the blocks of 256 elements from first_block[k] on; in 8 bits a block of the first moment is
// e4m3 codes times max|m| / 448 (nearest), and a block of u = sqrt(v) is e4m3 codes times max u / 448.  u is stored and not v
// because the 18 binades of e4m3 then span 36 binades of v, as many as the update can tell apart from the largest.  u is
// rounded up or down at random (an unbiased choice): one step decays it by (1 - b2) / 2, 0.1 % at b2 = 0.998, and rounding to
// nearest with steps of 6 to 12 % would never let it fall.  m moves by 1 - b1, 10 %, and is rounded to nearest.  A non-zero u
// never becomes 0, because it divides.  The update itself uses the unrounded moments of the step.
//
// HBM-bound: (p, g, m, v) are read and (p, m, v) written once, 28 bytes per fp32 parameter with 32-bit moments, 16 with
// 8-bit ones; gradient clipping reads g once more.  A wave takes 512 elements, 8 per lane: 16-byte accesses for 16-bit
// types and 32 lanes = one quantisation block, whose two maxima are five DPP / swizzle steps.  The tensors travel as kernel
// arguments, up to 96 and up to eight counts of steps to a launch: nothing has to be uploaded or kept between calls.  1e9 bf16
// parameters in 300 tensors with fp32 master weights and 8-bit moments: 3.22 ms = 5.0 TB/s; 18 M fp32 ones with 32-bit moments and
// clipping: 123 us, of which the norm 26 (a large copy: 4.9 TB/s).
#include "../../include/vae_amd.h"
#include "common.h"

#include <math.h>

#include <algorithm>
#include <new>

// Sums and products round one by one, as written: the 8-bit codes of two builds (and of a plain restatement) agree then.
#pragma clang fp contract(off)

namespace {

constexpr int BLK = VAE_ADAMW_BLOCK;
constexpr int PER_LAUNCH = 96;
constexpr int STEP_ELEMS = 2048;          // elements a workgroup of 256 threads takes at a time
constexpr int NORM_GROUPS = 512;          // norm partials per launch

struct Tensors {
  void* p[PER_LAUNCH];
  const void* g[PER_LAUNCH];
  int64_t n[PER_LAUNCH];
  uint32_t first_block[PER_LAUNCH];
  uint32_t chunk_end[PER_LAUNCH];         // running total of chunks, this tensor's included
  float keep[PER_LAUNCH];                 // 1 - lr * weight_decay
  uint8_t kind[PER_LAUNCH];               // dtype | 4: param and grad are 16-byte aligned | 8 * index of its count of steps
  int32_t count;
  int32_t steps;                          // a chunk is steps * STEP_ELEMS elements
};
// What follows from a tensor's count of steps.  Tensors of a launch share a few counts: one, where all have had every gradient.
constexpr int COUNTS = 8;
struct Count {
  float step_size, inv_bc2;
  uint32_t key;
};
struct Scalars {
  float b1, omb1, b2, omb2, eps, gscale;
  Count at[COUNTS];
};
static_assert(sizeof(Tensors) + sizeof(Scalars) + 48 <= 4096, "kernel arguments are limited to 4 KB");

// Austin Appleby's 32-bit finaliser (MurmurHash3, public domain)
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

// eight consecutive elements from `at`, those from n on read as 0
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ src, int64_t at, int64_t n, bool wide, float (&o)[8]) {
  if (wide && at + 8 <= n) {
    constexpr int Q = sizeof(T) / 2;      // 16-byte pieces
    union { u4 q[Q]; T t[8]; } w;
#pragma unroll
    for (int i = 0; i < Q; ++i) w.q[i] = reinterpret_cast<const u4*>(src + at)[i];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = to_f(w.t[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = at + j < n ? to_f(src[at + j]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ dst, int64_t at, int64_t n, bool wide, const float (&v)[8]) {
  if (wide && at + 8 <= n) {
    constexpr int Q = sizeof(T) / 2;
    union { u4 q[Q]; T t[8]; } w;
#pragma unroll
    for (int j = 0; j < 8; ++j) w.t[j] = (T)v[j];
#pragma unroll
    for (int i = 0; i < Q; ++i) reinterpret_cast<u4*>(dst + at)[i] = w.q[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + j < n) dst[at + j] = (T)v[j];
  }
}

// maximum over the 32 lanes of a half wave of non-negative floats as integers: a NaN is the largest and is kept
template <int CTRL> __device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t half_wave_max(uint32_t v) {
  v = max(v, dpp_u<0xB1>(v));                                          // quad_perm [1, 0, 3, 2]
  v = max(v, dpp_u<0x4E>(v));                                          // quad_perm [2, 3, 0, 1]
  v = max(v, dpp_u<0x124>(v));                                         // row_ror:4
  v = max(v, dpp_u<0x128>(v));                                         // row_ror:8
  return max(v, (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, 0x401F));   // lane ^ 16
}

// index of the tensor that chunk `b` belongs to: every lane compares two of the running totals
__device__ __forceinline__ int tensor_of(const Tensors& t, uint32_t b) {
  const int lane = threadIdx.x & 63;
  const uint32_t e0 = lane < t.count ? t.chunk_end[lane] : 0xffffffffu;
  const uint32_t e1 = lane + 64 < t.count && lane + 64 < PER_LAUNCH ? t.chunk_end[lane + 64] : 0xffffffffu;
  const int k = __popcll(__ballot(e0 <= b)) + __popcll(__ballot(e1 <= b));
  return __builtin_amdgcn_readfirstlane(k);
}

template <typename T, int BITS>
__device__ __forceinline__ void update(T* __restrict__ p, const T* __restrict__ g, int64_t n, bool wide, int64_t from, int64_t to,
                                       uint32_t first_block, float keep, float gs, const Scalars& s, const Count& c, void* __restrict__ em,
                                       void* __restrict__ ev, float* __restrict__ scales, int64_t n_blocks,
                                       float* __restrict__ master) {
  const int64_t flat0 = (int64_t)first_block * BLK;
  for (int64_t at = from + threadIdx.x * 8; at - threadIdx.x * 8 < to; at += STEP_ELEMS) {
    const bool live = at < n;                                          // a half wave's block is live as a whole or not at all,
    const int64_t f = flat0 + at;                                      // but for the padding of a tensor's last block
    const bool mine = at < (n + BLK - 1) / BLK * BLK;
    float pw[8], gw[8], m[8], v[8], u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) pw[j] = gw[j] = m[j] = v[j] = 0.f;
    float sm = 0.f, su = 0.f;
    const int64_t blk = f / BLK;
    if (live) {
      load8(g, at, n, wide, gw);
      if (master) load8(master + flat0, at, n, true, pw);
      else load8(p, at, n, wide, pw);
    }
    if (BITS == 8) {
      uint2 cm = make_uint2(0, 0), cv = make_uint2(0, 0);
      if (mine) {
        cm = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(em) + f);
        cv = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(ev) + f);
        sm = scales[blk];
        su = scales[n_blocks + blk];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int wm = q < 2 ? cm.x : cm.y, wv = q < 2 ? cv.x : cv.y;
        const auto a = (q & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8(wm, true) : __builtin_amdgcn_cvt_pk_f32_fp8(wm, false);
        const auto b = (q & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8(wv, true) : __builtin_amdgcn_cvt_pk_f32_fp8(wv, false);
        m[2 * q] = a[0] * sm;
        m[2 * q + 1] = a[1] * sm;
        const float u0 = b[0] * su, u1 = b[1] * su;
        v[2 * q] = u0 * u0;
        v[2 * q + 1] = u1 * u1;
      }
    } else if (mine) {
      load8(reinterpret_cast<const float*>(em), f, f + 8, true, m);
      load8(reinterpret_cast<const float*>(ev), f, f + 8, true, v);
    }
    uint32_t tm = 0, tu = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float gg = gw[j] * gs;
      m[j] = m[j] * s.b1 + gg * s.omb1;
      v[j] = v[j] * s.b2 + (gg * gg) * s.omb2;
      u[j] = sqrtf(v[j]);
      const float moved = (m[j] / (u[j] * c.inv_bc2 + s.eps)) * c.step_size;
      pw[j] = pw[j] * keep - moved;
      if (BITS == 8) {
        if (at + j >= n) m[j] = u[j] = 0.f;                            // padding holds zeros, whatever it held before
        tm = max(tm, __float_as_uint(m[j]) & 0x7fffffffu);
        tu = max(tu, __float_as_uint(u[j]) & 0x7fffffffu);
      }
    }
    if (live) {
      if (master) store8(master + flat0, at, n, true, pw);
      store8(p, at, n, wide, pw);
    }
    if (BITS == 8) {
      tm = half_wave_max(tm);
      tu = half_wave_max(tu);
      const float top_m = __uint_as_float(tm), top_u = __uint_as_float(tu);
      // below 1e-30 the reciprocal could overflow; such a block is held as zeros.  A NaN compares false: its scale says it
      const float im = top_m > 1e-30f ? (1.f / top_m) * 448.f : 0.f, iu = top_u > 1e-30f ? (1.f / top_u) * 448.f : 0.f;
      const uint32_t pair = (uint32_t)(f >> 1);                        // f is a multiple of 8: the four pairs share their upper half
      const uint32_t key = mix32((uint32_t)(f >> 33) + c.key);
      uint32_t wm[2], wv[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int code = 0;
        float q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = fminf(fmaxf(m[4 * h + j] * im, -448.f), 448.f);
        code = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], code, false);
        code = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], code, true);
        wm[h] = (uint32_t)code;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t hash = mix32((pair + 2 * h + j / 2) ^ key);
          const uint32_t r = (j & 1) ? hash >> 16 : hash & 0xffffu;
          // times 2^-120 the upper 12 bits of a float are the code (subnormals included): adding 20 random bits below
          // rounds up with the probability of the cut-off part, 16 of them random and the next the middle
          const uint32_t b = __float_as_uint((u[4 * h + j] * iu) * 0x1p-120f);
          uint32_t code = min((b + (r << 4) + 8u) >> 20, 126u);
          code = u[4 * h + j] > 0.f ? max(code, 1u) : code;
          w |= code << (8 * j);
        }
        wv[h] = w;
      }
      if (mine) {
        *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(em) + f) = make_uint2(wm[0], wm[1]);
        *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(ev) + f) = make_uint2(wv[0], wv[1]);
        if ((f & (BLK - 1)) == 0) {
          // (an infinity is passed on as NaN: beside a finite gradient's overflowing square the block would otherwise come back as
          // infinite roots, and weights that do not move any more)
          scales[blk] = top_m < INFINITY ? top_m * (float)(1.0 / 448.0) : NAN;
          scales[n_blocks + blk] = top_u < INFINITY ? top_u * (float)(1.0 / 448.0) : NAN;
        }
      }
    } else if (live) {
      // (the padding behind a tensor's last element is not written: n - at bounds the store)
      store8(reinterpret_cast<float*>(em), f, flat0 + n, true, m);
      store8(reinterpret_cast<float*>(ev), f, flat0 + n, true, v);
    }
  }
}

template <int BITS>
__global__ __launch_bounds__(256) void adamw_multi_kernel(Tensors t, Scalars s, void* __restrict__ em, void* __restrict__ ev,
                                                          float* __restrict__ scales, int64_t n_blocks, float* __restrict__ master,
                                                          const float* __restrict__ coef) {
  const int k = tensor_of(t, blockIdx.x);
  if (k >= t.count) return;
  const uint32_t first = k ? t.chunk_end[k - 1] : 0;
  const int64_t n = t.n[k], chunk = (int64_t)t.steps * STEP_ELEMS, from = (int64_t)(blockIdx.x - first) * chunk;
  const int64_t to = min(from + chunk, n);
  const float gs = coef ? s.gscale * coef[0] : s.gscale;
  const int kind = t.kind[k];
  const bool wide = kind & 4;
  const Count c = s.at[kind >> 3];
#define VAE_UPDATE(T) update<T, BITS>((T*)t.p[k], (const T*)t.g[k], n, wide, from, to, t.first_block[k], t.keep[k], gs, s, c, em, ev, scales, n_blocks, master)
  switch (kind & 3) {
    case 0: VAE_UPDATE(float); break;
    case 1: VAE_UPDATE(__bf16); break;
    default: VAE_UPDATE(_Float16); break;
  }
#undef VAE_UPDATE
}

// partial[block] = this workgroup's share of sum g^2, in 64 bits: the clip coefficient, and with it every code, is then the
// same however the sum is split
template <typename T>
__device__ __forceinline__ double sumsq(const T* __restrict__ g, int64_t n, bool wide, int64_t from, int64_t to) {
  double a = 0;
  for (int64_t at = from + threadIdx.x * 8; at < to; at += STEP_ELEMS) {
    float v[8];
    load8(g, at, n, wide, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) a = fma((double)v[j], (double)v[j], a);
  }
  return a;
}
__device__ __forceinline__ double block_sum64(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}
__global__ __launch_bounds__(256) void norm_partials_kernel(Tensors t, uint32_t chunks, double* __restrict__ partial) {
  __shared__ double red[4];
  double a = 0;
  for (uint32_t b = blockIdx.x; b < chunks; b += gridDim.x) {
    const int k = tensor_of(t, b);
    if (k >= t.count) break;
    const int64_t n = t.n[k], chunk = (int64_t)t.steps * STEP_ELEMS, from = (int64_t)(b - (k ? t.chunk_end[k - 1] : 0)) * chunk;
    const int64_t to = min(from + chunk, n);
    const int kind = t.kind[k];
    const bool wide = kind & 4;
    switch (kind & 3) {
      case 0: a += sumsq((const float*)t.g[k], n, wide, from, to); break;
      case 1: a += sumsq((const __bf16*)t.g[k], n, wide, from, to); break;
      default: a += sumsq((const _Float16*)t.g[k], n, wide, from, to); break;
    }
  }
  a = block_sum64(a, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = a;
}
// norm of grad_scale * g and min(1, max_norm / (norm + 1e-6)), as torch.nn.utils.clip_grad_norm_: a NaN norm is passed on, an
// infinite one gives 0
__global__ __launch_bounds__(256) void norm_finish_kernel(const double* __restrict__ partial, int n, double gscale, double max_norm,
                                                          float* __restrict__ coef, float* __restrict__ norm_out) {
  __shared__ double red[4];
  double a = 0;
  for (int i = threadIdx.x; i < n; i += 256) a += partial[i];
  a = block_sum64(a, red);
  if (threadIdx.x == 0) {
    const double norm = sqrt(a) * fabs(gscale);
    double c = max_norm / (norm + 1e-6);
    if (c > 1.0) c = 1.0;
    *coef = (float)c;
    if (norm_out) *norm_out = (float)norm;
  }
}

int64_t launches_of(int64_t n_tensors) { return (n_tensors + PER_LAUNCH - 1) / PER_LAUNCH; }

struct Span {
  uintptr_t b, e;
};

}  // namespace

extern "C" int64_t vae_adamw_multi_workspace_bytes(int64_t n_tensors) {
  return (launches_of(n_tensors < 1 ? 1 : n_tensors) * NORM_GROUPS + 1) * (int64_t)sizeof(double);
}

extern "C" int vae_adamw_multi(const vae_adamw_tensor* tensors, int64_t n_tensors, int state_bits, void* exp_avg, void* exp_avg_sq,
                               float* scales, int64_t n_blocks, float* master, double lr, double beta1, double beta2, double eps,
                               int64_t step, double max_grad_norm, double grad_scale, uint64_t seed, void* workspace,
                               int64_t workspace_bytes, float* grad_norm_out, void* stream) {
  VAE_REQUIRE(n_tensors >= 0 && n_tensors <= (1 << 20) && (tensors || n_tensors == 0), "vae_adamw_multi: null or too many tensors");
  VAE_REQUIRE(state_bits == 8 || state_bits == 32, "vae_adamw_multi: state_bits must be 8 or 32, got %d", state_bits);
  VAE_REQUIRE(step >= 1, "vae_adamw_multi: step counts from 1");
  VAE_REQUIRE(lr >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0, "vae_adamw_multi: bad hyper-parameter");
  VAE_REQUIRE(n_blocks >= 0 && n_blocks < (1ll << 31), "vae_adamw_multi: 0 <= n_blocks < 2^31");
  if (n_tensors == 0 || n_blocks == 0) {
    for (int64_t k = 0; k < n_tensors; ++k) VAE_REQUIRE(tensors[k].n == 0, "vae_adamw_multi: tensor %lld does not fit the state", (long long)k);
    VAE_REQUIRE(max_grad_norm <= 0 && !grad_norm_out, "vae_adamw_multi: no gradient to take a norm of");
    return VAE_OK;
  }
  VAE_REQUIRE(exp_avg && exp_avg_sq && vae_aligned16(exp_avg) && vae_aligned16(exp_avg_sq) && vae_aligned16(master),
              "vae_adamw_multi: the state is null or not 16-byte aligned");
  VAE_REQUIRE(state_bits == 32 || scales, "vae_adamw_multi: 8-bit moments need scales (2, n_blocks)");
  const bool clip = max_grad_norm > 0 || grad_norm_out;
  VAE_REQUIRE(!clip || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0 &&
                        workspace_bytes >= vae_adamw_multi_workspace_bytes(n_tensors)),
              "vae_adamw_multi: clipping needs an 8-byte aligned workspace of vae_adamw_multi_workspace_bytes()");
  // what is written must be disjoint, and no gradient may lie in it: two accesses to one element would race
  Span* spans = new (std::nothrow) Span[2 * n_tensors + 4];
  VAE_REQUIRE(spans, "vae_adamw_multi: out of host memory");
  Span* blocks = spans + n_tensors + 4;
  int64_t total = 0, n_spans = 0, n_live = 0;
  const char* bad = nullptr;
  long long bad_at = 0;
  const int64_t per = state_bits == 8 ? 1 : 4;
  for (int64_t k = 0; k < n_tensors && !bad; ++k) {
    const vae_adamw_tensor& t = tensors[k];
    const int esize = t.dtype == VAE_ADAMW_F32 ? 4 : 2;
    const uintptr_t pb = reinterpret_cast<uintptr_t>(t.param), gb = reinterpret_cast<uintptr_t>(t.grad);
    bad_at = (long long)k;
    if (t.n < 0 || t.n > (1ll << 40)) bad = "a size is negative or too large";
    else if (t.n && (!t.param || !t.grad)) bad = "a null param or grad";
    else if (t.dtype < 0 || t.dtype > 2) bad = "unknown dtype";
    else if (pb % esize || gb % esize) bad = "param or grad is not aligned to its element";
    else if (t.first_block < 0 || t.first_block > n_blocks || (t.n + BLK - 1) / BLK > n_blocks - t.first_block) bad = "does not fit the state";
    else if (!(t.weight_decay >= 0)) bad = "negative weight decay";
    else if (t.step < 0) bad = "step counts from 1";
    else if (t.n) {
      spans[n_spans++] = {pb, pb + (uintptr_t)(t.n * esize)};
      blocks[n_live++] = {(uintptr_t)t.first_block, (uintptr_t)(t.first_block + (t.n + BLK - 1) / BLK)};
      total += t.n;
    }
  }
  const auto disjoint = [](Span* s, int64_t n) {
    std::sort(s, s + n, [](const Span& a, const Span& b) { return a.b < b.b; });
    for (int64_t i = 1; i < n; ++i)
      if (s[i].b < s[i - 1].e) return false;
    return true;
  };
  if (!bad) {
    auto add = [&](const void* q, int64_t bytes) {
      if (q) spans[n_spans++] = {reinterpret_cast<uintptr_t>(q), reinterpret_cast<uintptr_t>(q) + (uintptr_t)bytes};
    };
    add(exp_avg, n_blocks * BLK * per);
    add(exp_avg_sq, n_blocks * BLK * per);
    if (state_bits == 8) add(scales, 2 * n_blocks * 4);
    add(master, n_blocks * BLK * 4);
    if (!disjoint(spans, n_spans)) bad = "params and state overlap in memory", bad_at = -1;
    else if (!disjoint(blocks, n_live)) bad = "two tensors share blocks of the state", bad_at = -1;
    else if (total > 1ll << 37) bad = "more than 2^37 elements", bad_at = -1;      // (a launch's grid holds what 96 of them need)
  }
  for (int64_t k = 0; k < n_tensors && !bad; ++k) {
    const vae_adamw_tensor& t = tensors[k];
    const uintptr_t b = reinterpret_cast<uintptr_t>(t.grad), e = b + (uintptr_t)(t.n * (t.dtype == VAE_ADAMW_F32 ? 4 : 2));
    const Span* after = std::lower_bound(spans, spans + n_spans, e, [](const Span& s, uintptr_t x) { return s.b < x; });
    if (t.n && after != spans && after[-1].e > b) bad = "the gradient overlaps what is written", bad_at = (long long)k;
  }
  delete[] spans;
  VAE_REQUIRE(!bad, "vae_adamw_multi: tensor %lld: %s", bad_at, bad);

  hipStream_t st = (hipStream_t)stream;
  // Chunks of 2048 elements until a launch has some 4096 of them (16 workgroups for every CU), then longer ones, which save
  // workgroup starts: up to 16384 elements.
  const int64_t want = total / ((int64_t)STEP_ELEMS * 4096);
  const int steps = (int)(want < 1 ? 1 : want > 8 ? 8 : want);
  const int64_t chunk = (int64_t)steps * STEP_ELEMS;
  Scalars s;
  s.b1 = (float)beta1;
  s.omb1 = (float)(1.0 - beta1);
  s.b2 = (float)beta2;
  s.omb2 = (float)(1.0 - beta2);
  s.eps = (float)eps;
  s.gscale = (float)grad_scale;
  const auto count_of = [&](int64_t n) -> Count {
    return {(float)(lr / (1.0 - pow(beta1, (double)n))), (float)(1.0 / sqrt(1.0 - pow(beta2, (double)n))),
            mix32(((uint32_t)seed ^ mix32((uint32_t)(seed >> 32))) ^ mix32((uint32_t)n * 0x9E3779B9u))};
  };
  double* partial = reinterpret_cast<double*>(workspace);
  float* coef = clip ? reinterpret_cast<float*>(partial + launches_of(n_tensors) * NORM_GROUPS) : nullptr;
  const float* use = max_grad_norm > 0 ? coef : nullptr;
  Tensors t;
  for (int pass = clip ? 0 : 1; pass < 2; ++pass) {
    int64_t n_partials = 0;
    for (int64_t k = 0; k < n_tensors;) {
      int64_t chunks = 0, counts[COUNTS];
      int n_counts = 0;
      t.count = 0;
      t.steps = steps;
      for (; k < n_tensors && t.count < PER_LAUNCH; ++k) {
        const vae_adamw_tensor& e = tensors[k];
        if (e.n == 0) continue;
        const int64_t own = e.step ? e.step : step;
        int at = 0;
        while (at < n_counts && counts[at] != own) ++at;
        if (pass == 0) at = 0;                                         // (the norm asks for none: its launches stay launches_of())
        else if (at == n_counts) {
          if (at == COUNTS) break;                                     // (one count more than a launch holds: the next launch's)
          counts[n_counts++] = own;
          s.at[at] = count_of(own);
        }
        const int i = t.count++;
        chunks += (e.n + chunk - 1) / chunk;
        t.p[i] = e.param;
        t.g[i] = e.grad;
        t.n[i] = e.n;
        t.first_block[i] = (uint32_t)e.first_block;
        t.chunk_end[i] = (uint32_t)chunks;
        t.keep[i] = (float)(1.0 - lr * (double)e.weight_decay);
        t.kind[i] = (uint8_t)(e.dtype | (vae_aligned16(e.param) && vae_aligned16(e.grad) ? 4 : 0) | at << 3);
      }
      if (!t.count) break;
      if (pass == 0) {
        const int grid = (int)(chunks < NORM_GROUPS ? chunks : NORM_GROUPS);
        norm_partials_kernel<<<grid, 256, 0, st>>>(t, (uint32_t)chunks, partial + n_partials);
        n_partials += grid;
      } else if (state_bits == 8) {
        adamw_multi_kernel<8><<<(uint32_t)chunks, 256, 0, st>>>(t, s, exp_avg, exp_avg_sq, scales, n_blocks, master, use);
      } else {
        adamw_multi_kernel<32><<<(uint32_t)chunks, 256, 0, st>>>(t, s, exp_avg, exp_avg_sq, nullptr, n_blocks, master, use);
      }
      VAE_CHECK_LAUNCH("vae_adamw_multi");
    }
    if (pass == 0) {
      norm_finish_kernel<<<1, 256, 0, st>>>(partial, (int)n_partials, grad_scale, max_grad_norm > 0 ? max_grad_norm : INFINITY, coef,
                                            grad_norm_out);
      VAE_CHECK_LAUNCH("vae_adamw_multi");
    }
  }
  return VAE_OK;
}
