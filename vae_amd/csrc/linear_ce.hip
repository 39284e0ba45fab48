// Softmax cross entropy of a linear head, z = x W^T + b over N rows and V classes, with its gradients, without the logits
// being in memory (gfx950).
//
//   lse_i = log sum_v exp z_iv        nll_i = c[t_i] (lse_i - z_{i, t_i})
//   d_iv  = g_i c[t_i] (exp(z_iv - lse_i) - [v = t_i])        dx = d W        dW = d^T x        db = sum_i d_i
//
// Rows with the ignored target are left out before anything else: the others are gathered, in order, into a packed copy of x
// (their number stays on the device; tiles and K loops behind it end at once), so that ignored rows cost nothing and what they
// hold, infinities and NaN included, reaches no gradient.
//
// Forward: a tile product of W with the packed x in which a lane owns a row of x and its accumulators run over classes.  The
// running maximum and sum of a tile are then taken inside a lane's registers, and only one pair per row and 256 classes is
// written.  Backward, for pieces of the classes whose d fits a fixed workspace: the same product again, whose epilogue turns
// the logits into d (16 bits) and sums it over its rows for db; then dx += d W and dW = d^T x, in one launch.  4 products of
// 2 N D V operations, of which one is the recompute that stands for keeping N V logits.  Bound by the matrix cores as soon as N
// and D are a few hundred: 8192 x 4096 x 131072 in bf16, loss 6.7 ms = 1.3 PFLOP/s, loss and gradients 26.9 ms = 1.3 PFLOP/s over
// all four products (a product of that shape by the library: 1.48).  Only where the tiles of the logits are too few to fill the
// chip is K split instead, and partial logits of at most 134 MB are written and read once (64 x 4000 x 900 bf16: both passes 70 us,
// 129 without; 901 x 3014 x 1683 fp32 326 and 527).
//
// Types: bf16 and fp16 multiply as they are, sums in 32 bits; d is rounded to the same type (by at most 2^-8 or 2^-11 of each
// element, independent of each other, so that a sum of them is off by no more than its own rounding).  d is divided by the
// largest factor g_i c[t_i] for that, and the products are multiplied by it in 32 bits: the term of the target, -1 in nearly
// every row of a large vocabulary, is then exact, where the rounding of 1 / N itself would shift every gradient by the same
// part, up to 2^-8 (error against 64 bits 3.7e-3 with it, 1.7e-3 without).  fp16 could not hold d, which goes down to 1e-12: it is
// multiplied by 2^14 as well, and where factors differ from row to row (see FACTOR_FREE) a row far below the largest one by a
// power of two of its own.  fp32 operands are split exactly into three bf16 terms, and for every 64 of K the six products
// that matter run one after the other: the error is that of 32-bit sums, at a sixth of the 16-bit rate (a 32-bit matrix
// instruction would give a sixteenth).
#include "../../include/vae_amd.h"
#include "common.h"

#include <math.h>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;
typedef __attribute__((address_space(3))) void* lds_void_ptr;
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef u4 u4_any __attribute__((aligned(2)));          // 16-byte accesses at any element

constexpr int ROW_PAD = 256;                            // packed rows and columns of d come in multiples of this
constexpr int K_PAD = 64;

// the state of a forward pass that the backward pass reads: int32 / float words
// kept rows, sum of c[t], finished workgroups; row index, class (-1: none) and lse, N each, of the kept rows
constexpr int S_KEPT = 0, S_TOTAL = 1, S_DONE = 2, S_ROWS = 4;

enum { EPI_STATS = 0, EPI_D = 1, EPI_STORE = 2 };

struct Gemm {
  const uint16_t *a, *b;        // A: [M][K] (KC) or [K][M] (RC); B: [N][K] or [K][N]; 16-bit elements
  int64_t lda, ldb;
  int64_t plane_a, plane_b;     // elements from one bf16 term to the next (fp32 operands)
  int M, N, K;
  int segs;                     // 1, or 6 products of bf16 terms
  const int* dyn;               // kept rows: bounds N, or K (dyn_k)
  int dyn_k;
  int split, tiles_m, tiles_n;
  // EPI_STATS, EPI_D
  int v0;                       // first class of this piece: class = v0 + m
  const void* bias;             // of the operands' outer type
  int bias_f32;
  const int* classes;           // by packed row
  float2* partial;              // (tile_m, N padded): running maximum and sum
  float* target_logit;          // by packed row
  const float* lse;             // by packed row
  const float* g;               // by packed row: upstream * class weight (0: an exactly zero row)
  const float* d_scale;         // what d is multiplied by, and its reciprocal
  const float* row_factor;      // fp16: null, or what row n of d has to be multiplied by besides (EPI_STORE: row n of the result)
  uint16_t* d;                  // [N padded][ldd], planes at plane_d
  int64_t ldd, plane_d;
  float* d_sums;                // null, or (tile_n, ldd): sums of d over a tile's rows
  // EPI_STORE: out[n][m], final type or float slabs (split, N, M) that are added to when `add`
  void* out;
  int64_t ldo;
  const int* rows;              // null, or where row n of the result belongs
  int out_kind;                 // 0 float slab, 1 the final 16-bit type, 2 final float
  int add;
};

__device__ __forceinline__ void split3(float v, __bf16& h, __bf16& m, __bf16& l) {
  h = (__bf16)v;
  const float r = v - (float)h;
  m = (__bf16)r;
  l = (__bf16)(r - (float)m);
}

// exp to an ulp or so for v <= 88, 0 far below: the rounding error of v * log2 e is fed back.  As vae_exp_acc, which takes a NaN for
// -inf, where this one passes it on (a NaN logit has to show in its row's loss)
__device__ __forceinline__ float exp_fine(float v) {
  v = v < -100.f ? -100.f : v;
  const float t = v * 1.44269504088896341f;
  float r = fmaf(v, 1.44269504088896341f, -t);
  r = fmaf(v, 1.925963033500011e-8f, r);
  const float e = __builtin_amdgcn_exp2f(t);
  return fmaf(e, r * 0.69314718055994531f, e);
}

// sum over 16 consecutive lanes, in all of them
template <int CTRL> __device__ __forceinline__ float dpp_f(float v) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row16_sum(float v) {
  v += dpp_f<0xB1>(v);                                        // quad_perm [1, 0, 3, 2]
  v += dpp_f<0x4E>(v);                                        // quad_perm [2, 3, 0, 1]
  v += dpp_f<0x124>(v);                                       // row_ror:4
  return v + dpp_f<0x128>(v);                                 // row_ror:8
}

// One wave instruction: lane i copies 16 bytes from base + off_i to LDS byte lds + 16 i.  In inline asm so that the compiler
// does not drain the counter ahead of the next LDS read; the kernel waits itself.
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(off), "s"(base), "s"(lds)
               : "memory");
}
template <int LEFT> __device__ __forceinline__ void wait_and_meet() {   // this wave's loads but LEFT have landed, its LDS reads are done
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// 16 x 16 x 32: with operands in registers alone this instruction sustains 1985 TFLOP/s in bf16 on random data where the
// 32 x 32 x 16 one, of the same peak, sustains 1264 (the clock gives way to its power).
template <bool F16> __device__ __forceinline__ f32x4 mma(u4 a, u4 b, f32x4 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <bool F16> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  union {
    __bf16 h[2];
    _Float16 f[2];
    uint32_t u;
  } w;
  if constexpr (F16) w.f[0] = (_Float16)a, w.f[1] = (_Float16)b;
  else w.h[0] = (__bf16)a, w.h[1] = (__bf16)b;
  return w.u;
}

__device__ __forceinline__ int rc_swizzle(int k) { return (k & 3) << 2 | (k >> 3 & 1) << 1; }

// Tile product.  BM x BN outputs, W_M x W_N waves, K in steps of BK through two images in LDS, filled by direct loads; one
// barrier per step.
//   KC image [rows][BK]: 16-byte chunk c of a row sits at chunk c ^ f(row), so that the 16 rows of a b128 read hit all banks.
//   RC image [BK][rows]: chunk c of k sits at c ^ f(k); fragments by the transposing read, whose 16 lanes take 4 k x 16 rows: f
//   spreads the 8 values of k that half a wave reads over the banks.
// The largest tile's step of 64 takes 1.4 us = 1.5 PFLOP/s over the chip (bf16, 8192 x 16384 from K 1024 to 4096; an image of
// 32 of K in four stages, a third image for B alone, two 256 x 128 workgroups to a CU and 128 x 128 in four waves were all
// slower), what a tile starts and ends with 8 to 12 us.
// Rows and columns of A past its end are clamped to the last one (their products are not stored, or meet zeros in B); B is a
// packed operand, padded with zeros to whole tiles.
constexpr int lds_elements(int bm, int bn, int w_m, int epi) { return 2 * 64 * (bm + bn) + (epi == EPI_STATS ? w_m * bn * 4 : 0); }
template <bool F16, bool A_KC, bool B_KC, int BM, int BN, int W_M, int W_N, int EPI, bool FINE>
__device__ __forceinline__ void head_gemm(Gemm g, uint16_t* smem, int block, int blocks) {
  constexpr int BK = 64, STAGES = 2;
  constexpr int NW = W_M * W_N, TM = BM / (16 * W_M), TN = BN / (16 * W_N);
  constexpr int IMG_A = BM * BK, IMG_B = BN * BK, STAGE = IMG_A + IMG_B;          // elements
  constexpr int PA = IMG_A * 2 / 1024 / NW, PB = IMG_B * 2 / 1024 / NW;           // 1 KB pieces per wave
  static_assert(PA >= 1 && PB >= 1, "tile too small for the workgroup");
  // Workgroups whose epilogue leaves the images alone stay for several tiles and send for the next one's first steps during the
  // last ones of the tile before: 250 -> 242 us for 4093 x 1000 x 30011, 473 -> 464 for 2048 x 2048 x 65536.
  constexpr bool STAY = EPI == EPI_STATS;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / W_N, wn = wave % W_N, l15 = lane & 15, lj = lane >> 4;

  int N = g.N, K = g.K, tiles_n = g.tiles_n;
  if (g.dyn) {
    const int kept = __builtin_amdgcn_readfirstlane(*g.dyn);
    if (g.dyn_k) K = min(K, kept);
    else N = min(N, kept), tiles_n = (N + BN - 1) / BN;
  }
  // Workgroups go round the 8 XCDs: give each XCD a run of consecutive tiles (all tiles of one part of K, where K is split),
  // which its workgroups take in turn, and order the tiles in bands of 4 along M, so that the 32 tiles an XCD works on at a time
  // share 4 blocks of A and 8 of B in its L2.
  const int total = g.tiles_m * tiles_n;
  int id, end, turn;
  {
    const int all = total * g.split, q8 = all >> 3, r8 = all & 7, xcd = block & 7, beg = xcd * q8 + min(xcd, r8);
    id = beg + (block >> 3);
    end = beg + q8 + (xcd < r8 ? 1 : 0);
    turn = (blocks + 7 - xcd) >> 3;
  }
  if (id >= end) return;
  const int part = id / total;                               // of K (which is split only where a workgroup has one tile)
  auto place = [&](int tile, int& m0, int& n0) {
    constexpr int BAND = 4;
    const int at = tile % total, band = at / (BAND * tiles_n), in = at - band * BAND * tiles_n;
    const int height = min(BAND, g.tiles_m - band * BAND);
    m0 = (band * BAND + in % height) * BM;
    n0 = in / height * BN;
  };

  const int kt1 = (K + BK - 1) / BK, all_k = kt1 * g.segs, per = (all_k + g.split - 1) / g.split;
  const int t_beg = min(part * per, all_k), steps = min(t_beg + per, all_k) - t_beg;

  // ---- loads: per-lane byte offsets from a base that moves with K; `k_left` elements of K remain from the step on ----
  int f_m0, f_n0;                                            // the tile that is being loaded: ahead of the one in work at its end
  auto chunk_a = [&](int i, int k_left) -> uint32_t {
    const int piece = wave * PA + i;
    if (A_KC) {
      constexpr int CPR = BK / 8;
      const int row = piece * (64 / CPR) + lane / CPR, swz = (row >> 1) & 7;
      const int c = min((lane % CPR) ^ swz, (k_left + 7) / 8 - 1);
      return (uint32_t)(((int64_t)(min(f_m0 + row, g.M - 1) - f_m0) * g.lda + 8 * c) * 2);
    }
    constexpr int CPR = BM / 8;
    const int k = piece * (64 / CPR) + lane / CPR, c = (lane % CPR) ^ rc_swizzle(k);
    return (uint32_t)(((int64_t)min(k, k_left - 1) * g.lda + min(8 * c, ((g.M + 7) & ~7) - 8 - f_m0)) * 2);
  };
  auto chunk_b = [&](int i) -> uint32_t {
    const int piece = wave * PB + i;
    if (B_KC) {
      constexpr int CPR = BK / 8;
      const int row = piece * (64 / CPR) + lane / CPR, swz = (row >> 1) & 7;
      return (uint32_t)(((int64_t)row * g.ldb + 8 * ((lane % CPR) ^ swz)) * 2);
    }
    constexpr int CPR = BN / 8;
    const int k = piece * (64 / CPR) + lane / CPR, c = (lane % CPR) ^ rc_swizzle(k);
    return (uint32_t)(((int64_t)k * g.ldb + 8 * c) * 2);
  };
  const int k_tail = K - (kt1 - 1) * BK;                     // of the last step: 1 .. BK
  uint32_t off_a[PA], off_t[PA], off_b[PB];
  auto offsets = [&]() {
#pragma unroll
    for (int i = 0; i < PA; ++i) off_a[i] = chunk_a(i, BK), off_t[i] = chunk_a(i, max(k_tail, 1));
#pragma unroll
    for (int i = 0; i < PB; ++i) off_b[i] = chunk_b(i);
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_ptr)smem;
  const uint16_t *base_a, *base_b;
  int kt, seg, f_id = id, f_steps = 0, fill = 0;             // of the next step to load; steps loaded of its tile; its image
  auto start = [&]() {
    place(f_id, f_m0, f_n0);
    base_a = A_KC ? g.a + (int64_t)f_m0 * g.lda : g.a + f_m0;
    base_b = B_KC ? g.b + (int64_t)f_n0 * g.ldb : g.b + f_n0;
    kt = t_beg / g.segs;
    seg = t_beg - kt * g.segs;
    f_steps = 0;
    offsets();
  };
  start();
  const uint16_t *sa, *sb;                                              // its base
  bool tail;
  auto more = [&]() { return f_steps < steps || (STAY && f_id + turn < end); };
  auto aim = [&]() {
    if (STAY && f_steps == steps) f_id += turn, start();    // on to the next tile
    ++f_steps;
    // terms (hi 0, mid 1, lo 2) of the product a * b that segment `seg` forms: mm, hl, lh, hm, mh, hh
    const int pa = g.segs == 1 ? 0 : (0x102010 >> (20 - 4 * seg)) & 15, pb = g.segs == 1 ? 0 : (0x120100 >> (20 - 4 * seg)) & 15;
    const int k0 = kt * BK;
    sa = base_a + pa * g.plane_a + (A_KC ? (int64_t)k0 : (int64_t)k0 * g.lda);
    sb = base_b + pb * g.plane_b + (B_KC ? (int64_t)k0 : (int64_t)k0 * g.ldb);
    tail = kt == kt1 - 1;
    if (++seg == g.segs) seg = 0, ++kt;                                 // (a block's terms stay in the L2 for all its products)
  };
  auto load = [&](int i) {                                              // piece i of the step aimed at
    const uint32_t st = lds0 + (uint32_t)fill * (STAGE * 2u);
    if (i < PA) dma16(sa, tail ? off_t[i] : off_a[i], st + (uint32_t)(wave * PA + i) * 1024u);
    else dma16(sb, off_b[i - PA], st + IMG_A * 2u + (uint32_t)(wave * PB + i - PA) * 1024u);
  };

  // ---- fragments: 16 rows, 32 of K, 8 consecutive ones to a lane ----
  const int swz = (l15 >> 1) & 7, lq = l15 >> 2, lp = l15 & 3;
  const int kc_a = (wm * 16 * TM + l15) * BK, kc_b = (wn * 16 * TN + l15) * BK;
  const int rc_k = 8 * lj + lq, rc_f = rc_swizzle(rc_k) << 3;
  const int rc_a = wm * 16 * TM + 4 * lp, rc_b = wn * 16 * TN + 4 * lp;
  auto frag_kc = [&](const uint16_t* img, int base, int t, int ks) -> u4 {
    return *reinterpret_cast<const u4*>(img + base + t * 16 * BK + (((4 * ks + lj) ^ swz) << 3));
  };
  auto frag_rc = [&](const uint16_t* img, int width, int col0, int t, int ks) -> u4 {
    const uint16_t* p = img + (ks * 32 + rc_k) * width + ((col0 + t * 16) ^ rc_f);
    union {
      s16x4 s[2];
      u4 v;
    } u;
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p);
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p + 4 * width));
    return u.v;
  };

  // Two images: while one is multiplied the other is filled.  In each half of a step (32 of K) the fragment of A is read again,
  // for the next half, as soon as its products are issued, and B's beside the one in use.  After the first products of the
  // second half a step's image has been read by everyone, and the step after next is sent into it, piece by piece between the
  // products of that half: all at once the pieces fill the queue of the vector memory unit and hold up what comes behind them,
  // and over three quarters or five of a half they took 2 and 5 % longer.
  // The steps run on from one tile to the next: the last two of a tile send for the first two of the next one, which are on
  // their way during its epilogue.
  u4 a[TM], b[2][TN];
  constexpr int LOADS = PA + PB;
  static_assert(TN <= TM, "a fragment of B for every block of products");
  auto read_a = [&](int image, int ks, int i) {
    const uint16_t* img = smem + image * STAGE;
    a[i] = A_KC ? frag_kc(img, kc_a, i, ks) : frag_rc(img, BM, rc_a, i, ks);
  };
  auto read_b = [&](int which, int image, int ks, int j) {
    const uint16_t* img = smem + image * STAGE + IMG_A;
    b[which][j] = B_KC ? frag_kc(img, kc_b, j, ks) : frag_rc(img, BN, rc_b, j, ks);
  };
  int fetched = 0;
  for (; fetched < STAGES && more(); ++fetched, ++fill) {
    aim();
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(i);
  }
  if (fetched == STAGES) wait_and_meet<LOADS>();
  else wait_and_meet<0>();
  int image = 0;
  for (; id < end; id += turn) {
    int m0, n0;
    place(id, m0, n0);
    // what the epilogue needs of this lane's rows, asked for now
    int cls[TN];
    float lse[TN], gn[TN];
    if constexpr (EPI != EPI_STORE) {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = n0 + (wn * TN + j) * 16 + l15;
        const bool real = n < N;
        cls[j] = real ? g.classes[n] : -1;
        lse[j] = EPI == EPI_D && real ? g.lse[n] : 0.f;
        gn[j] = EPI == EPI_D && real ? g.g[n] : 0.f;
      }
    }
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = (f32x4)0.f;

#pragma unroll
    for (int j = 0; j < TN; ++j) read_b(0, image, 0, j);
#pragma unroll
    for (int i = 0; i < TM; ++i) read_a(image, 0, i);
    bool send = false;
    for (int t = 0; t < steps; ++t) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = mma<F16>(a[i], b[ks][j], acc[i][j]);
          if (ks && i == 0) {
            wait_and_meet<0>();                                // the next step is here, and nobody reads this image any more
            send = more();
            fill = image;
            if (send) aim();
          }
          const int from = ks ? image ^ 1 : image;             // (behind the last step: old values)
          read_a(from, ks ^ 1, i);
#pragma unroll
          for (int j = 0; j < TN; ++j)
            if (j * TM / TN == i) read_b(ks ^ 1, from, ks ^ 1, j);
          if (ks && send) {
#pragma unroll
            for (int e = 0; e < LOADS; ++e)
              if (e * TM / LOADS == i) load(e);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      image ^= 1;
    }

    // acc[i][j][r]: m = m0 + 16 (wm TM + i) + 4 lj + r, n = n0 + 16 (wn TN + j) + l15
    const int mw = m0 + wm * 16 * TM + 4 * lj, nw = n0 + wn * 16 * TN + l15;
    // The waves' outputs go through LDS (the images are done with), where a row n of the tile is contiguous in m, and leave as
    // whole rows: straight from the registers every store would touch 16 rows.  16-byte chunk c of row n sits at c ^ 2 n (16-bit
    // elements) or c ^ 4 n (floats), so that neither the writes nor the reads meet in a bank.
    auto rows_out16 = [&](auto&& value, auto&& send_row) {         // value(i, j) -> 4 packed elements; send_row(row, chunk, 16 bytes)
      constexpr int CPR = BM / 8;
      wait_and_meet<0>();
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int row = wn * 16 * TN + 16 * j + l15, c = wm * 2 * TM + 2 * i + (lj >> 1);
          *reinterpret_cast<uint2*>(smem + row * BM + (((c ^ (2 * row)) % CPR) << 3) + 4 * (lj & 1)) = value(i, j);
        }
      __syncthreads();
      for (int x = threadIdx.x; x < BN * CPR; x += 64 * NW) {
        const int row = x / CPR, c = x % CPR;
        send_row(row, c, *reinterpret_cast<const u4*>(smem + row * BM + (((c ^ (2 * row)) % CPR) << 3)));
      }
    };
    if constexpr (EPI == EPI_STORE) {
      const float all = g.d_scale ? g.d_scale[1] : 1.f;
      float inv[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) inv[j] = F16 && g.row_factor && nw + 16 * j < N ? all * g.row_factor[nw + 16 * j] : all;
      if (g.out_kind == 1) {
        uint16_t* out = reinterpret_cast<uint16_t*>(g.out);
        rows_out16(
            [&](int i, int j) {
              const f32x4 v = acc[i][j] * inv[j];
              return make_uint2(pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]));
            },
            [&](int row, int c, u4 v) {
              const int n = n0 + row, m = m0 + 8 * c;
              if (n >= N || m >= g.M) return;
              uint16_t* o = out + (int64_t)(g.rows ? g.rows[n] : n) * g.ldo + m;
              if (m + 8 <= g.M) {
                *reinterpret_cast<u4_any*>(o) = v;
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (m + e < g.M) o[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
              }
            });
      } else {
        typedef float f4 __attribute__((ext_vector_type(4)));
        typedef f4 f4_any __attribute__((aligned(4)));
        float *lds = reinterpret_cast<float*>(smem), *out = reinterpret_cast<float*>(g.out) + (int64_t)(g.out_kind == 0 ? part : 0) * g.N * g.ldo;
        constexpr int CPR = BM / 4, ROWS = 32 * W_N;           // 32 rows of every wave at a time
        static_assert(ROWS * BM * 2 <= STAGES * STAGE && TN % 2 == 0, "a pass fits");
#pragma unroll
        for (int j0 = 0; j0 < TN; j0 += 2) {
          wait_and_meet<0>();
#pragma unroll
          for (int j = j0; j < j0 + 2; ++j)
#pragma unroll
            for (int i = 0; i < TM; ++i) {
              const int row = wn * 32 + 16 * (j - j0) + l15, c = wm * 4 * TM + 4 * i + lj;
              *reinterpret_cast<f4*>(lds + row * BM + (((c ^ (4 * row)) % CPR) << 2)) = acc[i][j] * inv[j];
            }
          __syncthreads();
          for (int x = threadIdx.x; x < ROWS * CPR; x += 64 * NW) {
            const int row = x / CPR, c = x % CPR;
            f4 v = *reinterpret_cast<const f4*>(lds + row * BM + (((c ^ (4 * row)) % CPR) << 2));
            const int n = n0 + (row >> 5) * 16 * TN + 16 * j0 + (row & 31), m = m0 + 4 * c;
            if (n >= N || m >= g.M) continue;
            float* o = out + (int64_t)(g.rows ? g.rows[n] : n) * g.ldo + m;
            if (m + 4 <= g.M) {
              if (g.add) v += *reinterpret_cast<const f4_any*>(o);
              *reinterpret_cast<f4_any*>(o) = v;
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (m + e < g.M) o[e] = g.add ? o[e] + v[e] : v[e];
            }
          }
        }
      }
    } else {
      if (g.bias) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int v = g.v0 + min(mw + 16 * i + r, g.M - 1);
            const float bv = g.bias_f32 ? reinterpret_cast<const float*>(g.bias)[v]
                             : F16      ? (float)reinterpret_cast<const _Float16*>(g.bias)[v]
                                        : (float)reinterpret_cast<const __bf16*>(g.bias)[v];
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j][r] += bv;
          }
      }
      constexpr float L2E = 1.44269504088896341f;                // (with |ref| below 1e37 a z of the type's lowest value gives 0)
      const bool edge = m0 + BM > g.M;                          // classes past the last one
      if constexpr (EPI == EPI_STATS) {
        float2* red = reinterpret_cast<float2*>(smem + STAGES * STAGE);          // [W_M][BN]
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int n = nw + 16 * j;
          const int at = cls[j] - g.v0 - mw;                    // 16 i + r where the target's logit is ours
          if (__any(at >= 0 && at < 16 * TM)) {
            float hit = 0.f;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) hit = at == 16 * i + r ? acc[i][j][r] : hit;
            if (at >= 0 && at < 16 * TM && !(at & 12)) g.target_logit[n] = hit;   // (at & 12: it is another lane's)
          }
          if (edge) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (mw + 16 * i + r >= g.M) acc[i][j][r] = -INFINITY;
          }
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[i][j][r]);
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float ref = top == -INFINITY ? 0.f : top;       // all of them -inf: the sum is 0, not NaN
          float sum = 0.f;
          if (!FINE && __all(fabsf(ref) < 1e37f)) {
            const float neg = -ref * L2E;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], L2E, neg));
          } else {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) sum += FINE ? exp_fine(acc[i][j][r] - ref) : __builtin_amdgcn_exp2f((acc[i][j][r] - ref) * L2E);
          }
          sum += __shfl_xor(sum, 16, 64);
          sum += __shfl_xor(sum, 32, 64);
          if (lj == 0) red[wm * BN + wn * 16 * TN + 16 * j + l15] = make_float2(top, sum);
        }
        wait_and_meet<63>();
        for (int c = threadIdx.x; c < BN; c += 64 * NW) {
          if (n0 + c >= N) continue;
          float2 p = red[c];
#pragma unroll
          for (int w = 1; w < W_M; ++w) {
            const float2 o = red[w * BN + c];
            const float top = fmaxf(p.x, o.x), ref = top == -INFINITY ? 0.f : top;
            p.y = p.y * exp_fine(p.x - ref) + o.y * exp_fine(o.x - ref);
            p.x = top;
          }
          g.partial[(int64_t)(m0 / BM) * ((g.N + ROW_PAD - 1) / ROW_PAD * ROW_PAD) + n0 + c] = p;
        }
      } else {
        const float scale = g.d_scale[0];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const float gs = gn[j] * scale, ref = lse[j];
          const int at = cls[j] - g.v0 - mw;
          if (!FINE && __all(fabsf(ref) < 1e37f)) {
            const float neg = -ref * L2E;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], L2E, neg));
          } else {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[i][j][r] = FINE ? exp_fine(acc[i][j][r] - ref) : __builtin_amdgcn_exp2f((acc[i][j][r] - ref) * L2E);
          }
          if (__any(at >= 0 && at < 16 * TM)) {                 // the target is among this wave's classes
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (at == 16 * i + r) acc[i][j][r] -= 1.f;
          }
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] *= gs;
          if (edge || __any(gs == 0.f)) {                       // rows without a gradient and classes past the end: exactly zero
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (gs == 0.f || mw + 16 * i + r >= g.M) acc[i][j][r] = 0.f;
          }
        }
      if (g.d_sums) {                                         // (of d as it is, before its rounding)
        float* red = reinterpret_cast<float*>(smem);          // [W_N][BM]
        // (factors are powers of two: taken off for the sums and put back without a rounding)
        auto times_factor = [&](bool back) {
          if (!F16 || !g.row_factor) return;
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const float f = nw + 16 * j < N ? g.row_factor[nw + 16 * j] : 1.f, by = back ? 1.f / f : f;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[i][j][r] *= by;
          }
        };
        times_factor(false);
        wait_and_meet<0>();
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < TN; ++j) s += acc[i][j][r];
            s = row16_sum(s);
            if (l15 == 0) red[wn * BM + wm * 16 * TM + 16 * i + 4 * lj + r] = s;
          }
        wait_and_meet<0>();
        for (int c = threadIdx.x; c < BM; c += 64 * NW) {
          float s = 0.f;
#pragma unroll
          for (int w = 0; w < W_N; ++w) s += red[w * BM + c];
          g.d_sums[(int64_t)(n0 / BN) * g.ldd + m0 + c] = s;
        }
        times_factor(true);
      }
#pragma unroll
      for (int plane = 0; plane < (FINE ? 3 : 1); ++plane)
          rows_out16(
              [&](int i, int j) {
                if constexpr (!FINE) return make_uint2(pack2<F16>(acc[i][j][0], acc[i][j][1]), pack2<F16>(acc[i][j][2], acc[i][j][3]));
                union {
                  __bf16 t[4];
                  uint2 u;
                } w;
#pragma unroll
                for (int e = 0; e < 4; ++e) {                   // the term, and what it leaves for the next
                  w.t[e] = (__bf16)acc[i][j][e];
                  acc[i][j][e] -= (float)w.t[e];
                }
                return w.u;
              },
              [&](int row, int c, u4 v) { *reinterpret_cast<u4*>(g.d + plane * g.plane_d + (int64_t)(n0 + row) * g.ldd + m0 + 8 * c) = v; });
      }
    }
    if (!STAY) return;
    offsets();                                                  // (formed again rather than held through the epilogue)
  }
}

template <bool F16, int BM, int BN, int W_M, int W_N, int EPI, bool FINE>
__global__ __launch_bounds__(64 * W_M * W_N, 2) void head_logits_kernel(Gemm g) {
  __shared__ __attribute__((aligned(16))) uint16_t smem[lds_elements(BM, BN, W_M, EPI)];
  head_gemm<F16, true, true, BM, BN, W_M, W_N, EPI, FINE>(g, smem, blockIdx.x, gridDim.x);
}
// dx and dW of a piece of classes, in one launch: neither fills the chip to its end.  `dx_blocks`: a multiple of 8
template <bool F16, int BM, int BN, int W_M, int W_N>
__global__ __launch_bounds__(64 * W_M * W_N, 2) void head_grads_kernel(Gemm dx, Gemm dw, int dx_blocks) {
  __shared__ __attribute__((aligned(16))) uint16_t smem[lds_elements(BM, BN, W_M, EPI_STORE)];
  const int block = blockIdx.x;
  if (block < dx_blocks) head_gemm<F16, false, true, BM, BN, W_M, W_N, EPI_STORE, false>(dx, smem, block, dx_blocks);
  else head_gemm<F16, false, false, BM, BN, W_M, W_N, EPI_STORE, false>(dw, smem, block - dx_blocks, (int)gridDim.x - dx_blocks);
}

// Rows that count, in order, and the sum of their class weights, by one workgroup (ROWS_AT_ONCE targets at a time: a wave takes
// 64 in a row, so that what it writes stands together) -> their number.  They go to `table`, or (`write`) to the state, and an ignored row's loss is written as 0 where losses are
// returned by row.
constexpr int ROWS_AT_ONCE = 8192, TABLE_ROWS = 4096;
struct Rows {
  const int64_t* target;
  int N, V;
  int64_t ignore;
  const float* cw;
  int* state;
  float *target_logit, *loss_rows;
};
__device__ __forceinline__ int find_rows(const Rows& r, bool write, int* table) {
  __shared__ int counts[129];                                 // of the waves' 64 targets, in order; then of those ahead of them
  __shared__ double wave_w[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, N = r.N, V = r.V;
  int before = 0;
  double weight = 0;
  for (int base = 0; base < N; base += ROWS_AT_ONCE) {
    int64_t t[8];
    uint64_t mask[8];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = base + j * 1024 + (int)threadIdx.x;
      t[j] = i < N ? r.target[i] : r.ignore;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mask[j] = __ballot(t[j] != r.ignore);
      if (lane == 0) counts[j * 16 + wave] = __popcll(mask[j]);
    }
    __syncthreads();
    if (wave == 0) {
      const int a = counts[2 * lane], b = counts[2 * lane + 1];
      int run = a + b;                                        // inclusive scan over the wave
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(run, o, 64);
        if (lane >= o) run += u;
      }
      counts[2 * lane] = run - a - b;
      counts[2 * lane + 1] = run - b;
      if (lane == 63) counts[128] = run;
    }
    __syncthreads();
    const int all = counts[128];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = base + j * 1024 + (int)threadIdx.x, at = before + counts[j * 16 + wave] + __popcll(mask[j] & ((1ull << lane) - 1));
      if (i >= N) continue;
      if (t[j] != r.ignore) {
        if (table) table[at] = i;
        if (write) {
          const bool real = t[j] >= 0 && t[j] < V;
          r.state[S_ROWS + at] = i;
          r.state[S_ROWS + N + at] = real ? (int)t[j] : -1;
          r.target_logit[at] = NAN;                           // stays so where the target is no class
          weight += !real ? 0.0 : r.cw ? (double)r.cw[t[j]] : 1.0;   // (no class has no weight: the divisor stays that of the others)
        }
      } else if (write && r.loss_rows) {
        r.loss_rows[i] = 0.f;
      }
    }
    before += all;
  }
  if (write) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) weight += __shfl_xor(weight, o, 64);
    if (lane == 0) wave_w[wave] = weight;
  }
  __syncthreads();
  if (write && threadIdx.x == 0) {
    double w = 0;
    for (int i = 0; i < 16; ++i) w += wave_w[i];
    r.state[S_KEPT] = before;
    r.state[S_DONE] = 0;
    reinterpret_cast<float*>(r.state)[S_TOTAL] = (float)w;
  }
  return before;
}
__global__ __launch_bounds__(1024) void ce_rows_kernel(Rows r) { find_rows(r, true, nullptr); }

// fp16: d of a row whose factor g is 2^-k of the largest would sink into the subnormals with it (at 1e-7 of the largest the
// gradient of a row of 30000 classes was off by 30 %).  Past FACTOR_FREE such a row's d is multiplied by 2^s, s up to FACTOR_MOST;
// dx is multiplied by 2^-s where it is stored, and dW takes the row of x times 2^-s, which is exact down to |x| = 2^-4 or so
// (s = 10) and off by 2^-25 below.  Rows down to 2^-16 of the largest so keep 11 bits of every probability from 2^-22 on, and a row
// at 2^-24 from 2^-14 on.  Nothing of this where all factors are equal (one upstream gradient, no class weights);
// elsewhere the copy of x times 2^-s takes 1 % (4093 x 1000 x 30011, reduction "none", 1074 and 1085 us).
constexpr int FACTOR_FREE = 6, FACTOR_MOST = 10;
// g[i] = upstream * class weight / total of the kept rows (times 2^s); d_scale: (to / max |g|, max |g| / to); factor: 2^-s by row;
// by one workgroup
struct Upstream {
  const float* up;                                            // null: nothing to do
  const int* state;
  int reduction, N;
  const float* cw;
  float to;
  float *g, *d_scale, *factor;                                // factor: null where it is 1 throughout
};
__device__ __forceinline__ void upstream(const Upstream& u) {
  __shared__ float red[16];
  const int kept = u.state[S_KEPT];
  const float total = reinterpret_cast<const float*>(u.state)[S_TOTAL];
  float top = 0.f;
  for (int i = threadIdx.x; i < kept; i += 1024) {
    const int orig = u.state[S_ROWS + i], t = u.state[S_ROWS + u.N + i];
    float v = u.reduction == VAE_CE_NONE ? u.up[orig] : u.up[0];
    if (t < 0) v = NAN;
    else if (u.cw) v *= u.cw[t];
    if (u.reduction == VAE_CE_MEAN) v /= total;
    u.g[i] = v;
    top = fmaxf(top, fabsf(v));
  }
  top = block_max<16>(top, red);
  const bool usable = top > 1e-30f && top < INFINITY;         // (nothing to do without a gradient; infinities reach the result)
  if (u.factor) {
    const auto exponent = [](float v) { return (int)(__float_as_uint(v) >> 23 & 255u); };
    for (int i = threadIdx.x; i < kept; i += 1024) {
      const float v = u.g[i];                                 // (this thread's own)
      const int s = usable && v != 0.f ? min(max(exponent(top) - exponent(v) - FACTOR_FREE, 0), FACTOR_MOST) : 0;
      u.g[i] = ldexpf(v, s);
      u.factor[i] = ldexpf(1.f, -s);
    }
  }
  if (threadIdx.x == 0) {
    u.d_scale[0] = usable ? u.to / top : 1.f;
    u.d_scale[1] = usable ? top / u.to : 1.f;
  }
}

// out[i][0 .. ldo) = src[rows[i]][0 .. D), zeros behind the last column and the last kept row (up to whole tiles): 8 elements
// per thread; T = float: three bf16 planes
struct Pack {
  const void* src;
  int64_t ld;
  const int* state;                                           // null: all rows as they are
  int rows, blocks;
  uint16_t* out;
  int64_t plane;
};
template <typename T, typename Index>
__device__ __forceinline__ void pack_rows(const Pack& p, int block, int D, int64_t ldo, int kept, int padded, Index&& index) {
  const int per = (int)(ldo / 8);
  const int64_t all = (int64_t)padded * per;
  for (int64_t i = (int64_t)block * 1024 + threadIdx.x; i < all; i += (int64_t)p.blocks * 1024) {
    const int row = (int)(i / per), c = (int)(i - (int64_t)row * per) * 8;
    constexpr int Q = sizeof(T) / 2;
    union {
      T t[8];
      u4 q[Q];
    } v;
#pragma unroll
    for (int q = 0; q < Q; ++q) v.q[q] = (u4)0;
    if (row < kept) {
      const T* from = reinterpret_cast<const T*>(p.src) + (int64_t)index(row) * p.ld + c;
      if (c + 8 <= D) {
#pragma unroll
        for (int q = 0; q < Q; ++q) v.q[q] = reinterpret_cast<const u4_any*>(from)[q];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < D) v.t[j] = from[j];
      }
    }
    uint16_t* o = p.out + (int64_t)row * ldo + c;
    if constexpr (sizeof(T) == 4) {
      union {
        __bf16 t[8];
        u4 q;
      } w[3];
#pragma unroll
      for (int j = 0; j < 8; ++j) split3(v.t[j], w[0].t[j], w[1].t[j], w[2].t[j]);
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<u4*>(o + k * p.plane) = w[k].q;
    } else {
      *reinterpret_cast<u4*>(o) = v.q[0];
    }
  }
}
// fp16: out = the packed rows of x (rows, ldo) times their factors, 8 elements per thread
__global__ __launch_bounds__(256) void ce_scale_rows_kernel(const _Float16* __restrict__ x, const float* __restrict__ factor,
                                                            const int* __restrict__ state, int64_t ldo, _Float16* __restrict__ out) {
  const int per = (int)(ldo / 8);
  const int64_t all = (int64_t)state[S_KEPT] * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const _Float16 f = (_Float16)factor[i / per];             // (a power of two from 2^-10 on: exact)
    reinterpret_cast<f16x8*>(out)[i] = reinterpret_cast<const f16x8*>(x)[i] * f;
  }
}
// All that comes ahead of the products, in one launch: the row factors, x, and w where it has to be packed.  Where the rows that
// count, of at most TABLE_ROWS, are to be found first, every workgroup of x does so for itself: a launch less (loss of 2000 x 300 x
// 50 19.5 us and 21.2, called eagerly 26 and 30; of 8192 x 1024 x 500 47.8 and 43.8).
template <typename T> __global__ __launch_bounds__(1024) void ce_pack_kernel(Rows r, Upstream u, Pack x, Pack w, int D, int64_t ldo) {
  __shared__ int table[TABLE_ROWS];
  int block = blockIdx.x;
  const auto padded = [](int kept) { return (kept + ROW_PAD - 1) / ROW_PAD * ROW_PAD; };
  if (u.up && block-- == 0) {
    upstream(u);
  } else if (block >= x.blocks) {
    pack_rows<T>(w, block - x.blocks, D, ldo, w.rows, w.rows, [](int row) { return row; });
  } else if (r.target) {
    const int kept = find_rows(r, block == 0, table);
    pack_rows<T>(x, block, D, ldo, kept, padded(kept), [&](int row) { return table[row]; });
  } else {
    const int kept = x.state[S_KEPT];
    pack_rows<T>(x, block, D, ldo, kept, padded(kept), [&](int row) { return x.state[S_ROWS + row]; });
  }
}

// Sum and mean of the losses: every workgroup leaves the sum of its rows' (`share`, over its threads), and the one that finishes
// last adds up what all of them left, in order (same bits every time).
__device__ __forceinline__ double block_sum64(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) v += red[i];
  return v;
}
__device__ __forceinline__ void sum_losses(double share, int blocks, int* state, int reduction, double* sums, float* loss) {
  __shared__ double red[16];
  __shared__ bool last;
  share = block_sum64(share, red);
  if (threadIdx.x == 0) {
    __hip_atomic_store(sums + blockIdx.x, share, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = __hip_atomic_fetch_add(state + S_DONE, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == blocks - 1;
  }
  __syncthreads();
  if (!last) return;
  share = 0;
  for (int i = threadIdx.x; i < blocks; i += blockDim.x) share += __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  share = block_sum64(share, red);
  if (threadIdx.x == 0) *loss = (float)(reduction == VAE_CE_MEAN ? share / (double)reinterpret_cast<const float*>(state)[S_TOTAL] : share);
}

// The partial maxima and sums of a row over the tiles -> lse and the row's loss: 32 rows to a workgroup, 8 threads to a row
__global__ __launch_bounds__(256) void ce_combine_kernel(const float2* __restrict__ partial, int tiles, int64_t ldp, int* __restrict__ state,
                                                         int N, const float* __restrict__ cw, const float* __restrict__ target_logit,
                                                         int reduction, double* __restrict__ sums, float* __restrict__ loss) {
  __shared__ float2 red[8][32];
  const int kept = state[S_KEPT], blocks = max((kept + 31) / 32, 1);
  const int row = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
  if ((int)blockIdx.x >= blocks) return;
  float top = -INFINITY, sum = 0.f;
  if (row < kept) {
    for (int t = part; t < tiles; t += 64) {                  // eight loads in flight
      float2 p[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) p[u] = t + 8 * u < tiles ? partial[(int64_t)(t + 8 * u) * ldp + row] : make_float2(-INFINITY, 0.f);
      float m = top;
#pragma unroll
      for (int u = 0; u < 8; ++u) m = fmaxf(m, p[u].x);
      const float ref = m == -INFINITY ? 0.f : m;
      sum *= exp_fine(top - ref);
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += p[u].y * exp_fine(p[u].x - ref);
      top = m;
    }
  }
  red[part][threadIdx.x & 31] = make_float2(top, sum);
  __syncthreads();
  double share = 0;
  if (part == 0 && row < kept) {
    float m = top;
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i][threadIdx.x].x);
    const float ref = m == -INFINITY ? 0.f : m;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += red[i][threadIdx.x].y * exp_fine(red[i][threadIdx.x].x - ref);
    const float lse = m + logf(sum);
    reinterpret_cast<float*>(state)[S_ROWS + 2 * N + row] = lse;
    const int orig = state[S_ROWS + row], t = state[S_ROWS + N + row];
    const float v = (lse - target_logit[row]) * (!cw || t < 0 ? 1.f : cw[t]);
    if (reduction == VAE_CE_NONE) loss[orig] = v;
    share = (double)v;
  }
  if (reduction != VAE_CE_NONE) sum_losses(share, blocks, state, reduction, sums, loss);
}

typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ f4_any slab_sum(const float* p, int S, int64_t slab) {
  f4_any s = {0.f, 0.f, 0.f, 0.f};
  int k = 0;
  for (; k + 4 <= S; k += 4) {
    f4_any v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const f4_any*>(p + (k + u) * slab);
#pragma unroll
    for (int u = 0; u < 4; ++u) s += v[u];
  }
  for (; k < S; ++k) s += *reinterpret_cast<const f4_any*>(p + k * slab);
  return s;
}
__device__ __forceinline__ float slab_sum1(const float* p, int S, int64_t slab) {
  float s = 0.f;
  for (int k = 0; k < S; ++k) s += p[k * slab];
  return s;
}

// ---- logits whose K was split: slabs (S, N, ldz) of partial logits, by packed row ----
template <typename T> __device__ __forceinline__ f4_any slab_logits(const float* p, int S, int64_t slab, const T* bias, int c, int V) {
  f4_any z = slab_sum(p + c, S, slab);                        // (ldz is V, up to whole groups of 4)
#pragma unroll
  for (int e = 0; e < 4; ++e) z[e] = c + e < V ? z[e] + (bias ? (float)bias[c + e] : 0.f) : -INFINITY;
  return z;
}
// lse and loss: TPR threads to a row, a wave up to 1024 classes and a workgroup beyond (loss of 600 x 2000 x 900 bf16 34 us by waves,
// 39 by workgroups; of 64 x 4000 x 4000 45 and 31)
template <typename T, int TPR>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void ce_slab_loss_kernel(const float* __restrict__ slabs, int S, int64_t ldz, const T* __restrict__ bias,
                                                                            int* __restrict__ state, int N, int V, const float* __restrict__ cw,
                                                                            int reduction, double* __restrict__ sums, float* __restrict__ loss) {
  constexpr int RPW = TPR < 256 ? 256 / TPR : 1, WAVES = TPR / 64;
  static_assert(TPR == 64 || RPW == 1, "a row to a wave or to a workgroup");
  __shared__ float2 red[WAVES];
  __shared__ float target_hit;
  const int kept = state[S_KEPT], blocks = min(max((kept + RPW - 1) / RPW, 1), (int)gridDim.x);
  if ((int)blockIdx.x >= blocks) return;
  const int sub = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  double share = 0;
  for (int base = blockIdx.x * RPW; base < kept; base += blocks * RPW) {
    const int row = base + sub, t = row < kept ? state[S_ROWS + N + row] : -1;
    float top = -INFINITY, sum = 0.f, hit = NAN;              // (stays so where the target is no class)
    if (row < kept) {
      const float* p = slabs + (int64_t)row * ldz;
      for (int c = lane * 4; c < V; c += TPR * 4) {
        const f4_any z = slab_logits(p, S, (int64_t)N * ldz, bias, c, V);
        const float m = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), top), ref = m == -INFINITY ? 0.f : m;
        sum *= exp_fine(top - ref);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (c + e < V) sum += exp_fine(z[e] - ref);
          hit = c + e == t ? z[e] : hit;
        }
        top = m;
      }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float ot = __shfl_xor(top, o, 64), os = __shfl_xor(sum, o, 64), m = fmaxf(top, ot), ref = m == -INFINITY ? 0.f : m;
      sum = sum * exp_fine(top - ref) + os * exp_fine(ot - ref);
      top = m;
    }
    const int owner = t < 0 ? 0 : (t >> 2) % TPR;             // (whose hit is NaN where t < 0)
    if (WAVES == 1) {
      hit = __shfl(hit, owner, 64);
    } else {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(top, sum);
      if (lane == owner) target_hit = hit;
      __syncthreads();
      if (lane == 0) {
        hit = target_hit;
        float m = top;
        for (int i = 1; i < WAVES; ++i) m = fmaxf(m, red[i].x);
        const float ref = m == -INFINITY ? 0.f : m;
        sum *= exp_fine(top - ref);
        for (int i = 1; i < WAVES; ++i) sum += red[i].y * exp_fine(red[i].x - ref);
        top = m;
      }
    }
    if (lane == 0 && row < kept) {
      const float lse = top + logf(sum);
      reinterpret_cast<float*>(state)[S_ROWS + 2 * N + row] = lse;
      const float v = (lse - hit) * (!cw || t < 0 ? 1.f : cw[t]);
      if (reduction == VAE_CE_NONE) loss[state[S_ROWS + row]] = v;
      share += (double)v;
    }
  }
  if (reduction != VAE_CE_NONE) sum_losses(share, blocks, state, reduction, sums, loss);
}
// d and the sums of SLAB_ROWS rows of it; zeros behind the last class and the last kept row, up to whole steps of K.  `keep`: d
// also takes the place of the first slab
constexpr int SLAB_ROWS = 8;
template <typename T>
__global__ __launch_bounds__(256) void ce_slab_d_kernel(float* slabs, bool keep, int S, int64_t ldz, const T* __restrict__ bias,
                                                        const int* __restrict__ state, int N, int V, const float* __restrict__ gs,
                                                        const float* __restrict__ d_scale, const float* __restrict__ factor,
                                                        uint16_t* __restrict__ d, int64_t ldd, int64_t plane, float* __restrict__ sums) {
  const int kept = state[S_KEPT], rows = (kept + 63) / 64 * 64, c = (blockIdx.x * 256 + threadIdx.x) * 4;
  const int first = blockIdx.y * SLAB_ROWS;
  if (first >= rows || c >= (V + 63) / 64 * 64) return;
  const float scale = d_scale[0];
  f4_any total = {0.f, 0.f, 0.f, 0.f};
  for (int row = first; row < first + SLAB_ROWS; ++row) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const float g = row < kept ? gs[row] * scale : 0.f;
    if (g != 0.f && c < V) {
      const f4_any z = slab_logits(slabs + (int64_t)row * ldz, S, (int64_t)N * ldz, bias, c, V);
      const float lse = reinterpret_cast<const float*>(state)[S_ROWS + 2 * N + row];
      const int at = state[S_ROWS + N + row] - c;
      const float of = factor ? factor[row] : 1.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = exp_fine(z[e] - lse);
        v[e] = c + e < V ? (at == e ? p - 1.f : p) * g : 0.f;
        total[e] = fmaf(v[e], of, total[e]);
      }
    }
    if (keep && row < kept && c < V) *reinterpret_cast<f4_any*>(slabs + (int64_t)row * ldz + c) = f4_any{v[0], v[1], v[2], v[3]};
    uint16_t* o = d + (int64_t)row * ldd + c;
    if constexpr (sizeof(T) == 4) {
      union {
        __bf16 t[4];
        uint2 u;
      } w[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) split3(v[e], w[0].t[e], w[1].t[e], w[2].t[e]);
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<uint2*>(o + k * plane) = w[k].u;
    } else {
      constexpr bool F16 = __is_same(T, _Float16);
      *reinterpret_cast<uint2*>(o) = make_uint2(pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]));
    }
  }
  if (sums) *reinterpret_cast<f4_any*>(sums + (int64_t)blockIdx.y * ldd + c) = total;
}

// ---- at most FEW_ROWS rows (fp32) or classes: the long operand goes from memory straight into matrix instructions ----
// The three terms of W would be written and read again for a handful of rows.  Both kernels are bound by their one read of W; a
// lane's four consecutive floats are four values of K (or four columns) whose order the other operand shares.  8 x 1024 x 40000:
// partial logits 38 us = 4.3 TB/s of W, dx 28 us (W partly in the caches), a loss 52 us against 197 with three terms, loss and
// gradients 211 against 530; 64 x 1024 x 40000 101 against 196 and 364 against 532 (the rows, read by every wave, are then half of
// the traffic).  Worth its two launches more from V D of some 2^15 N on: 16 x 512 x 2000 61 us against 72, 64 x 512 x 4000 92 and
// 91, 64 x 100 x 1000 68 and 57.
// The loss of a head of at most as many classes on many rows reads x in the same way, in every type, where its packed copy would take
// longer than the product: from 2^21 elements of x on (8192 x 4000 x 10 bf16 50 us and 70, 4096 x 3000 x 30 fp32 43 and 72, 8192 x 1024
// x 10 bf16 32 and 46; 1000 x 1000 x 40 fp32 30 and 29).
constexpr int FEW_ROWS = 64;
constexpr int64_t HEAD_WORK = 1 << 21;
__device__ __forceinline__ f4_any load4(const float* p, int c, int n) {                // p[c .. c + 4), those from n on as zeros
  if (c + 4 <= n) return *reinterpret_cast<const f4_any*>(p + c);
  f4_any v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < n) v[e] = p[c + e];
  return v;
}
// 16 bytes of a row from feature c on, those from n on as zeros
template <typename T> __device__ __forceinline__ u4 load16(const T* p, int c, int n) {
  constexpr int P = 16 / (int)sizeof(T);
  if (c + P <= n) return *reinterpret_cast<const u4_any*>(p + c);
  union {
    T t[P];
    u4 q;
  } v;
  v.q = (u4)0;
#pragma unroll
  for (int e = 0; e < P; ++e)
    if (c + e < n) v.t[e] = p[c + e];
  return v.q;
}
template <typename T> __device__ __forceinline__ f32x4 mma16(u4 a, u4 b, f32x4 c) {      // 16 bytes of K to a lane
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  } else {
    return mma<__is_same(T, _Float16)>(a, b, c);
  }
}
// Partial logits (part, N, ldz) straight from memory.  A wave takes 32 rows of the long operand and all of the short one, at most 64
// rows in tiles of 16, over `per` features (a multiple of 64).  HEAD: x is the long one and W the short, otherwise W is long.
template <typename T, int NB, bool HEAD>
__global__ __launch_bounds__(256) void ce_few_z_kernel(const T* __restrict__ w, int64_t ldw, const T* __restrict__ x, int64_t ldx,
                                                       const int* __restrict__ state, int N, int D, int V, int per, float* __restrict__ slabs,
                                                       int64_t ldz) {
  const int kept = state[S_KEPT], lane = threadIdx.x & 63, l15 = lane & 15, lj = lane >> 4;
  const int m0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 32, k0 = blockIdx.y * per, k1 = min(k0 + per, D);
  if (kept == 0 || m0 >= (HEAD ? kept : V)) return;
  const auto row_of_x = [&](int n) { return x + (int64_t)state[S_ROWS + min(n, kept - 1)] * ldx; };
  const auto row_of_w = [&](int v) { return w + (int64_t)min(v, V - 1) * ldw; };
  const T *ar[2], *br[NB];
#pragma unroll
  for (int t = 0; t < 2; ++t) ar[t] = HEAD ? row_of_x(m0 + 16 * t + l15) : row_of_w(m0 + 16 * t + l15);
#pragma unroll
  for (int j = 0; j < NB; ++j) br[j] = HEAD ? row_of_w(16 * j + l15) : row_of_x(16 * j + l15);
  constexpr int PIECE = 16 / (int)sizeof(T), GROUP = 4 * PIECE;
  constexpr int AHEAD = NB <= 2 ? 4 : 2;                      // groups of features at a time, the next ones on their way
  f32x4 acc[AHEAD][2][NB];                                    // (a sum for each: a 32-bit one rounds at every product)
#pragma unroll
  for (int u = 0; u < AHEAD; ++u)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[u][t][j] = (f32x4)0.f;
  struct In {
    u4 a[AHEAD][2], b[AHEAD][NB];
  } in, next;
  auto fetch = [&](In& to, int k) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int c = k + GROUP * u + PIECE * lj;
#pragma unroll
      for (int t = 0; t < 2; ++t) to.a[u][t] = load16(ar[t], c, k1);
#pragma unroll
      for (int j = 0; j < NB; ++j) to.b[u][j] = load16(br[j], c, k1);
    }
  };
  fetch(next, k0);
  for (int k = k0; k < k1; k += GROUP * AHEAD) {
    in = next;
    if (k + GROUP * AHEAD < k1) fetch(next, k + GROUP * AHEAD);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[u][t][j] = mma16<T>(in.a[u][t], in.b[u][j], acc[u][t][j]);
  }
#pragma unroll
  for (int h = AHEAD / 2; h > 0; h >>= 1)
#pragma unroll
    for (int u = 0; u < h; ++u)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[u][t][j] += acc[u + h][t][j];
  float* out = slabs + (int64_t)blockIdx.y * N * ldz;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int n = 16 * j + l15;                               // acc[0][t][j][r]: row m0 + 16 t + 4 lj + r of the long operand, n of the short
    if (n >= (HEAD ? V : kept)) continue;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int m = m0 + 16 * t + 4 * lj;
      if constexpr (HEAD) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m + r < kept) out[(int64_t)(m + r) * ldz + n] = acc[0][t][j][r];
      } else if (m < V) {
        *reinterpret_cast<f32x4*>(out + (int64_t)n * ldz + m) = acc[0][t][j];       // (ldz: V in whole fours)
      }
    }
  }
}
// dx slabs (part, N, D): a wave takes 64 columns and all rows over `per` classes (a multiple of 16); d (N, ldz) in 32 bits
template <int NB>
__global__ __launch_bounds__(256) void ce_few_dx_kernel(const float* __restrict__ w, int64_t ldw, const float* __restrict__ d, int64_t ldz,
                                                        const int* __restrict__ state, int N, int D, int V, int per,
                                                        const float* __restrict__ d_scale, float* __restrict__ slabs) {
  const int kept = state[S_KEPT], lane = threadIdx.x & 63, l15 = lane & 15, lj = lane >> 4;
  const int c = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 64 + 4 * l15, k0 = blockIdx.y * per, k1 = min(k0 + per, V);
  if (kept == 0 || c - 4 * l15 >= D) return;
  const float* dr[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) dr[j] = d + (int64_t)min(16 * j + l15, kept - 1) * ldz;
  f32x4 acc[4][NB];                                           // [column & 3]
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[t][j] = (f32x4)0.f;
  constexpr int AHEAD = NB <= 2 ? 2 : 1;                      // groups of 16 classes at a time, the next ones on their way
  struct In {
    f4_any a[AHEAD][4], b[AHEAD][NB];
  } in, next;
  auto fetch = [&](In& to, int k) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int v = k + 16 * u + 4 * lj;
#pragma unroll
      for (int e = 0; e < 4; ++e) to.a[u][e] = load4(w + (int64_t)min(v + e, V - 1) * ldw, c, D);
#pragma unroll
      for (int j = 0; j < NB; ++j) to.b[u][j] = load4(dr[j], v, k1);
    }
  };
  fetch(next, k0);
  for (int k = k0; k < k1; k += 16 * AHEAD) {
    in = next;
    if (k + 16 * AHEAD < k1) fetch(next, k + 16 * AHEAD);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(in.a[u][e][t], in.b[u][j][e], acc[t][j], 0, 0, 0);
  }
  const float inv = d_scale[1];
  const int c0 = c - 4 * l15 + 16 * lj;                       // acc[t][j][r]: column c0 + 4 r + t
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int n = 16 * j + l15;
    if (n >= kept) continue;
    float* o = slabs + ((int64_t)blockIdx.y * N + n) * D;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f4_any v = f4_any{acc[0][j][r], acc[1][j][r], acc[2][j][r], acc[3][j][r]} * inv;
      const int at = c0 + 4 * r;
      if (at + 4 <= D) {
        *reinterpret_cast<f4_any*>(o + at) = v;
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (at + t < D) o[at + t] = v[t];
      }
    }
  }
}

// What is left behind the products of a piece, in one launch:
//   db: the sums of d over the rows of every tile, added up.  64 classes to a workgroup of 4 waves, each of which adds every
//       4th tile, eight loads in flight; the 4 sums are added in order
//   dW: its slabs, where there are several, added in order
//   dx: behind the last piece, the slabs (S, N, D) of a packed row, where there are any, added in order and put at its original
//       row; ignored rows are zero.  A workgroup per row, four columns per thread
struct Finish {
  int db_blocks, dw_blocks, dx_blocks;
  const int* state;
  const float* d_scale;
  const float* sums;
  int64_t ld_sums;
  int sum_rows, V;
  void* db;
  const float* dw_slabs;
  int dw_split;
  int64_t dw_n;
  void* dw;
  const float* dx_slabs;
  int dx_split, N, D;
  const int64_t* target;
  int64_t ignore;
  void* dx;
};
template <typename T> __global__ __launch_bounds__(256) void ce_finish_kernel(Finish f) {
  __shared__ float red[4][64];
  int block = blockIdx.x;
  const int kept = f.state[S_KEPT];
  if (block < f.db_blocks) {
    const int c = block * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6, tiles = (kept + f.sum_rows - 1) / f.sum_rows;
    float s = 0.f;
    if (c < f.V) {
      const float* p = f.sums + c;
      int t = w;
      for (; t + 7 * 4 < tiles; t += 8 * 4) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[(int64_t)(t + 4 * i) * f.ld_sums];
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
      }
      for (; t < tiles; t += 4) s += p[(int64_t)t * f.ld_sums];
    }
    red[w][threadIdx.x & 63] = s;
    __syncthreads();
    if (w || c >= f.V) return;
#pragma unroll
    for (int i = 1; i < 4; ++i) s += red[i][threadIdx.x];
    reinterpret_cast<T*>(f.db)[c] = (T)(s * f.d_scale[1]);
    return;
  }
  block -= f.db_blocks;
  if (block < f.dw_blocks) {
    T* dw = reinterpret_cast<T*>(f.dw);
    for (int64_t i = ((int64_t)block * 256 + threadIdx.x) * 4; i < f.dw_n; i += (int64_t)f.dw_blocks * 1024) {
      if (i + 4 <= f.dw_n) {
        const f4_any s = slab_sum(f.dw_slabs + i, f.dw_split, f.dw_n);
#pragma unroll
        for (int e = 0; e < 4; ++e) dw[i + e] = (T)s[e];
      } else {
        for (int64_t e = i; e < f.dw_n; ++e) dw[e] = (T)slab_sum1(f.dw_slabs + e, f.dw_split, f.dw_n);
      }
    }
    return;
  }
  block -= f.dw_blocks;
  const int64_t slab = (int64_t)f.N * f.D;
  for (int row = block; f.dx_slabs && row < kept; row += f.dx_blocks) {
    T* o = reinterpret_cast<T*>(f.dx) + (int64_t)f.state[S_ROWS + row] * f.D;
    const float* p = f.dx_slabs + (int64_t)row * f.D;
    for (int c = threadIdx.x * 4; c < f.D; c += 1024) {
      if (c + 4 <= f.D) {
        const f4_any s = slab_sum(p + c, f.dx_split, slab);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c + e] = (T)s[e];
      } else {
        for (int e = c; e < f.D; ++e) o[e] = (T)slab_sum1(p + e, f.dx_split, slab);
      }
    }
  }
  for (int row = block; row < f.N; row += f.dx_blocks) {
    if (f.target[row] != f.ignore) continue;
    for (int c = threadIdx.x; c < f.D; c += 256) reinterpret_cast<T*>(f.dx)[(int64_t)row * f.D + c] = (T)0;
  }
}

// ---- heads of at most 64 classes on at most 64 columns, few rows: the whole pass in one workgroup ----
// The products are too small for tiles and the dozen launches of the way above would be all that is waited for.  256 rows at a
// time lie in LDS beside W, in 32 bits whatever the type; four lanes share a row, which they hold in registers, and take every
// fourth class.  D is padded with zeros to DM columns.
constexpr int SMALL_V = 64, SMALL_D = 64, SMALL_ROWS = 1024, SMALL_WORK = 1 << 18, CHUNK = 256;
struct Small {
  int N, D, V, reduction;
  int64_t ldx, ldw, ignore;
  const void *x, *w, *bias;
  const int64_t* target;
  const float *cw, *up;
  int* state;
  float* loss;
  void *dx, *dw, *db;
};
template <typename T, int DM> struct SmallLds {
  float w[SMALL_V][DM + 4], x[CHUNK][DM + 4], bias[SMALL_V];
};
template <typename T, int DM> __device__ __forceinline__ void small_weights(const Small& a, SmallLds<T, DM>& s) {
  for (int i = threadIdx.x; i < a.V * DM; i += 1024) {
    const int v = i / DM, c = i % DM;
    s.w[v][c] = c < a.D ? (float)reinterpret_cast<const T*>(a.w)[v * a.ldw + c] : 0.f;
  }
  if ((int)threadIdx.x < a.V) s.bias[threadIdx.x] = a.bias ? (float)reinterpret_cast<const T*>(a.bias)[threadIdx.x] : 0.f;
}
// rows base .. base + CHUNK, ignored ones and those past the end as zeros
template <typename T, int DM> __device__ __forceinline__ void small_rows(const Small& a, SmallLds<T, DM>& s, int base) {
  for (int i = threadIdx.x; i < CHUNK * DM; i += 1024) {
    const int r = i / DM, c = i % DM, row = base + r;
    const bool real = row < a.N && c < a.D && a.target[row] != a.ignore;
    s.x[r][c] = real ? (float)reinterpret_cast<const T*>(a.x)[row * a.ldx + c] : 0.f;
  }
}
template <int DM> __device__ __forceinline__ float small_dot(const float (&x)[DM], const float* w, float z) {
  float p[4] = {z, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < DM; c += 4) {
    const float4 v = *reinterpret_cast<const float4*>(w + c);
    p[0] = fmaf(x[c], v.x, p[0]);
    p[1] = fmaf(x[c + 1], v.y, p[1]);
    p[2] = fmaf(x[c + 2], v.z, p[2]);
    p[3] = fmaf(x[c + 3], v.w, p[3]);
  }
  return (p[0] + p[1]) + (p[2] + p[3]);
}
template <int DM> __device__ __forceinline__ void small_row(const float* src, float (&x)[DM]) {
#pragma unroll
  for (int c = 0; c < DM; c += 4) {
    const float4 v = *reinterpret_cast<const float4*>(src + c);
    x[c] = v.x;
    x[c + 1] = v.y;
    x[c + 2] = v.z;
    x[c + 3] = v.w;
  }
}

template <typename T, int DM> __global__ __launch_bounds__(1024) void ce_small_fwd_kernel(Small a) {
  __shared__ __attribute__((aligned(16))) SmallLds<T, DM> s;
  __shared__ double red[2][16];
  const int r = threadIdx.x >> 2, part = threadIdx.x & 3;
  double total = 0, weight = 0;
  small_weights(a, s);
  for (int base = 0; base < a.N; base += CHUNK) {
    __syncthreads();
    small_rows(a, s, base);
    __syncthreads();
    const int row = base + r;
    const int64_t t = row < a.N ? a.target[row] : a.ignore;
    const bool kept = row < a.N && t != a.ignore;
    float x[DM], top = -INFINITY, sum = 0.f, hit = 0.f;
    small_row(s.x[r], x);
    for (int v = part; v < a.V; v += 4) {
      const float z = small_dot(x, s.w[v], s.bias[v]);
      if (v == t) hit = z;
      if (z > top) {
        sum = sum * exp_fine(top - z) + 1.f;
        top = z;
      } else if (z != -INFINITY) {                            // (a NaN ends here and stays)
        sum += exp_fine(z - top);
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      const float ot = __shfl_xor(top, o, 64), os = __shfl_xor(sum, o, 64), m = fmaxf(top, ot), ref = m == -INFINITY ? 0.f : m;
      sum = sum * exp_fine(top - ref) + os * exp_fine(ot - ref);
      top = m;
      hit += __shfl_xor(hit, o, 64);
    }
    if (part || row >= a.N) continue;
    const bool real = kept && t >= 0 && t < a.V;
    const float lse = top + logf(sum), c = !real ? 0.f : a.cw ? a.cw[t] : 1.f;
    const float loss = real ? (lse - hit) * c : kept ? NAN : 0.f;
    reinterpret_cast<float*>(a.state)[S_ROWS + 2 * a.N + row] = lse;
    if (a.reduction == VAE_CE_NONE) a.loss[row] = loss;
    total += (double)loss;
    weight += (double)c;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64), weight += __shfl_xor(weight, o, 64);
  if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = total, red[1][threadIdx.x >> 6] = weight;
  __syncthreads();
  if (threadIdx.x) return;
  total = weight = 0;
  for (int i = 0; i < 16; ++i) total += red[0][i], weight += red[1][i];
  reinterpret_cast<float*>(a.state)[S_TOTAL] = (float)weight;
  if (a.reduction != VAE_CE_NONE) *a.loss = (float)(a.reduction == VAE_CE_MEAN ? total / weight : total);
}

template <typename T, int DM> __global__ __launch_bounds__(1024) void ce_small_bwd_kernel(Small a) {
  __shared__ __attribute__((aligned(16))) SmallLds<T, DM> s;
  __shared__ float d[CHUNK][SMALL_V + 1];
  const int r = threadIdx.x >> 2, part = threadIdx.x & 3;
  constexpr int QUADS = DM / 4, COLS = DM / 4;
  // dW: four columns of one class to a thread, the rows shared out among `ways` groups of threads
  const int outputs = a.V * QUADS;
  int span = 64;                                              // threads to a group: whole waves
  while (span < outputs) span <<= 1;
  const int ways = 1024 / span, way = threadIdx.x / span, o = threadIdx.x % span, ov = o / QUADS, oq = o % QUADS;
  const bool mine = o < outputs;
  float4 dw = make_float4(0.f, 0.f, 0.f, 0.f);
  float db = 0.f;
  const float total = reinterpret_cast<const float*>(a.state)[S_TOTAL];
  small_weights(a, s);
  for (int base = 0; base < a.N; base += CHUNK) {
    __syncthreads();
    small_rows(a, s, base);
    __syncthreads();
    const int row = base + r;
    const int64_t t = row < a.N ? a.target[row] : a.ignore;
    const bool kept = row < a.N && t != a.ignore;
    float g = 0.f, lse = 0.f;
    if (kept) {
      g = (a.reduction == VAE_CE_NONE ? a.up[row] : a.up[0]) * (t < 0 || t >= a.V ? NAN : a.cw ? a.cw[t] : 1.f);
      if (a.reduction == VAE_CE_MEAN) g /= total;
      lse = reinterpret_cast<const float*>(a.state)[S_ROWS + 2 * a.N + row];
    }
    {
      float x[DM];
      small_row(s.x[r], x);
      for (int v = part; v < a.V; v += 4) {
        const float p = exp_fine(small_dot(x, s.w[v], s.bias[v]) - lse);
        d[r][v] = g == 0.f ? 0.f : (v == t ? p - 1.f : p) * g;
      }
    }
    __syncthreads();
    if (a.dx && row < a.N) {
      float acc[COLS];
#pragma unroll
      for (int c = 0; c < COLS; ++c) acc[c] = 0.f;
      if (kept)
        for (int v = 0; v < a.V; ++v) {
          const float dv = d[r][v];
#pragma unroll
          for (int c = 0; c < COLS; ++c) acc[c] = fmaf(dv, s.w[v][part * COLS + c], acc[c]);
        }
      T* out = reinterpret_cast<T*>(a.dx) + (int64_t)row * a.D + part * COLS;
#pragma unroll
      for (int c = 0; c < COLS; ++c)
        if (part * COLS + c < a.D) out[c] = (T)acc[c];
    }
    if (mine) {
      const int rows = min(CHUNK, a.N - base);
      for (int i = way; i < rows; i += ways) {
        const float dv = d[i][ov];
        const float4 x = *reinterpret_cast<const float4*>(&s.x[i][4 * oq]);
        dw.x = fmaf(dv, x.x, dw.x);
        dw.y = fmaf(dv, x.y, dw.y);
        dw.z = fmaf(dv, x.z, dw.z);
        dw.w = fmaf(dv, x.w, dw.w);
        db += dv;
      }
    }
  }
  // the groups' sums, in order
  __syncthreads();
  float* part_w = &s.x[0][0];                                 // [1024][5]
  static_assert(sizeof(s.x) >= 1024 * 5 * 4, "the rows' place holds the groups' sums");
  {
    float* p = part_w + threadIdx.x * 5;
    p[0] = dw.x;
    p[1] = dw.y;
    p[2] = dw.z;
    p[3] = dw.w;
    p[4] = db;
  }
  __syncthreads();
  if (way || !mine) return;
  float sum[5] = {};
  for (int k = 0; k < ways; ++k)
#pragma unroll
    for (int e = 0; e < 5; ++e) sum[e] += part_w[(k * span + o) * 5 + e];
  if (a.dw)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (4 * oq + e < a.D) reinterpret_cast<T*>(a.dw)[ov * a.D + 4 * oq + e] = (T)sum[e];
  if (a.db && oq == 0) reinterpret_cast<T*>(a.db)[ov] = (T)sum[4];
}

// One workgroup is the faster way up to some 2^18 products (both passes on the GPU, fp32, against the way above: 64 x 32 x 32 16 us
// and 46, 512 x 30 x 17 35 and 50, 1024 x 30 x 17, 2^19 products, 64 and 51; 1024 x 16 x 16 takes 55 and 37, but 3 launches less a
// pass save their caller 24).
bool small_head(const vae_linear_ce* a) {
  return a->V <= SMALL_V && a->D <= SMALL_D && a->N <= SMALL_ROWS && a->N * a->V * a->D <= SMALL_WORK;
}
Small small_args(const vae_linear_ce* a, int reduction, void* state) {
  return {(int)a->N, (int)a->D, (int)a->V, reduction, a->ldx, a->ldw, a->ignore_index, a->x, a->w, a->bias, a->target, a->class_weight,
          nullptr, reinterpret_cast<int*>(state), nullptr, nullptr, nullptr, nullptr};
}
template <typename T> void launch_small(const Small& s, bool bwd, hipStream_t st) {
  if (s.D <= 32) {
    if (bwd) ce_small_bwd_kernel<T, 32><<<1, 1024, 0, st>>>(s);
    else ce_small_fwd_kernel<T, 32><<<1, 1024, 0, st>>>(s);
  } else {
    if (bwd) ce_small_bwd_kernel<T, 64><<<1, 1024, 0, st>>>(s);
    else ce_small_fwd_kernel<T, 64><<<1, 1024, 0, st>>>(s);
  }
}
void small(const Small& s, int dtype, bool bwd, hipStream_t st) {
  if (dtype == VAE_ADAMW_F32) launch_small<float>(s, bwd, st);
  else if (dtype == VAE_ADAMW_BF16) launch_small<__bf16>(s, bwd, st);
  else launch_small<_Float16>(s, bwd, st);
}

// ---- host ----
int64_t up_to(int64_t n, int64_t k) { return (n + k - 1) / k * k; }

// Tiles of 256 x 256 (one workgroup to a CU) or 128 x 128 (two), and into how many parts the sum over K is split where the
// tiles do not fill the chip: the least of rounds * (steps * c + f) + the slabs' traffic, with c and f as measured in bf16: a
// step of 64 of K takes 1.4 us in a large tile and 0.9 in each of two small ones; starting and ending a tile 8 and 6 us, 12
// where a large tile of logits is turned into d, and 55 where it is turned into three terms of d, for which its registers do
// not suffice.  Large against small, rows x D x classes: 8192 x 4096 x 16384 bf16 loss 0.84 and 1.05 ms, 8192 x 1024 x 16384
// 290 and 356 us; d of 2048 x 256 x 20000 bf16 57 and 50, fp32 264 and 190, of 512 x 256 x 20000 fp32 90 and 67; dx of 2048 x
// 1024 x 8192 fp32 171 and 213.
struct Tiles {
  bool big;
  int split;
  int64_t wgs;                                        // workgroups
  double each, slabs;                                 // us of each, us of the slabs' traffic
};
Tiles tiles_at(bool big, int split, int64_t m, int64_t n, int64_t steps, bool always_slabs, double end_big) {
  const int64_t b = big ? 256 : 128, tiles = ((m + b - 1) / b) * ((n + b - 1) / b), per = (steps + split - 1) / split;
  return {big, split, tiles * split, (double)per * (big ? 1.4 : 0.9) + (big ? end_big : 6.0),
          always_slabs || split > 1 ? 3.0 + (double)split * (double)m * (double)n * 8.0 / 4.5e6 : 0.0};
}
// Of the logits (m classes, n rows): tiles that fill the chip finish them in their epilogue; otherwise K is split, and a launch
// that reads the slabs stands for the epilogue (`launch` us, where it is one more).  Two rounds at most: 677 x 2636 x 13825 fp32,
// 165 large tiles, loss 380 us in three parts, 416 in one
Tiles tiles_for(int64_t m, int64_t n, int64_t k, bool f32, double end_big, double launch) {
  const int64_t steps = (k + 63) / 64 * (f32 ? 6 : 1);
  Tiles best = {};
  double least = 1e30;
  for (int big = 0; big < 2; ++big)
    for (int split = 1; split <= 32 && (split == 1 || steps / split >= 4); split += split < 4 ? 1 : split < 16 ? 4 : 8) {
      const Tiles t = tiles_at(big, split, m, n, steps, false, split == 1 ? end_big : 8.0);
      const int64_t slots = big ? 256 : 512;
      if (split > 1 && t.wgs > 2 * slots) break;
      const double us = (double)((t.wgs + slots - 1) / slots) * t.each + t.slabs + (split > 1 ? launch : 0.0);
      if (us < least) least = us, best = t;
    }
  return best;
}

struct Plan {
  bool f32, pack_w;
  int64_t n_pad, d_pad, ldw;                          // packed x: (n_pad, d_pad); W as it is, or packed to (V, d_pad)
  int64_t planes;
  int64_t piece;                                      // classes whose d is held at a time (a multiple of 256)
  bool few, head;                                     // fp32, few rows: W as it is; few classes (of a loss): x as it is
  Tiles z_tiles, d_tiles;                             // (of a pass)
  int z_parts;                                        // slabs of partial logits; 0: the product's epilogue finishes them
  int64_t ldz;                                        // of partial logits
  int sum_rows;                                       // rows to a sum in d_sums
  bool grads_big, dx_slabs;                           // (dx is written as it is where it takes one product with one part)
  int dx_split, dw_split;
  // byte offsets in the workspaces
  int64_t x, w, partial, tlogit, sums, g, scale, factor, scaled, z, d, d_sums, slabs, slabs_w, bytes;
};

constexpr int64_t D_BYTES = 512ll << 20;              // workspace for d, at most (but at least one tile of classes)

// dx and dW share a launch: tiles of one size, each product with its own split.  dx's workgroups come first; those of dW take the
// slots that are left over in dx's last round, and then all of them.  (512 x 256 x 20000 fp32: 192 workgroups of dx beside 314 of
// dW on 512 slots, 73 us; one after the other, dx on all slots, 98.)
void grads_for(const vae_linear_ce* a, Plan& p) {
  const int64_t kx = (p.piece + 63) / 64 * (p.f32 ? 6 : 1), kw = (a->N + 63) / 64 * (p.f32 ? 6 : 1);
  double least = 1e30;
  auto next = [](int s) { return s + (s < 4 ? 1 : s < 16 ? 4 : 8); };
  for (int big = 0; big < 2; ++big) {
    const int64_t slots = big ? 256 : 512;
    for (int sx = 1; sx <= 64 && (sx == 1 || kx / sx >= 4); sx = next(sx)) {
      const Tiles x = tiles_at(big, sx, a->D, a->N, kx, p.piece < a->V, 8.0);
      if (sx > 1 && x.wgs > 2 * slots) break;
      for (int sw = 1; sw <= 64 && (sw == 1 || kw / sw >= 4); sw = next(sw)) {
        const Tiles w = tiles_at(big, sw, a->D, p.piece, kw, false, 8.0);
        if (sw > 1 && w.wgs > 2 * slots) break;
        const int64_t over = x.wgs % slots, beside = over ? (slots - over) * (int64_t)(x.each / w.each) : 0;
        const int64_t left = w.wgs > beside ? w.wgs - beside : 0;
        const double t = (double)((x.wgs + slots - 1) / slots) * x.each + (double)((left + slots - 1) / slots) * w.each + x.slabs + w.slabs;
        if (t < least) least = t, p.grads_big = big, p.dx_split = sx, p.dw_split = sw;
      }
    }
  }
}

Plan plan_of(const vae_linear_ce* a, bool bwd) {
  Plan p;
  p.f32 = a->dtype == VAE_ADAMW_F32;
  p.planes = p.f32 ? 3 : 1;
  p.n_pad = up_to(a->N, ROW_PAD);
  p.d_pad = up_to(a->D, K_PAD);
  // waves enough to fill the chip, sums over at most 2048 features, partial logits of at most 64 MiB
  p.ldz = up_to(a->V, 4);
  const auto parts_for = [&](int64_t rows) {
    const int64_t waves = (rows + 31) / 32, want = (4095 + waves) / waves, most = (a->D + 255) / 256, least = (a->D + 2047) / 2048;
    const int64_t parts = want > most ? most : want < least ? least : want;
    return (int)(parts <= 64 && parts * a->N * p.ldz * 4 <= 64ll << 20 ? parts : 0);
  };
  const int few_parts = parts_for(a->V);
  p.few = p.f32 && a->N <= FEW_ROWS && a->V * a->D >= a->N << 15 && few_parts &&
          a->V <= D_BYTES / (p.planes * p.n_pad * 2) / 256 * 256;
  p.head = !p.few && !bwd && a->V <= FEW_ROWS && a->N * a->D >= HEAD_WORK && parts_for(a->N);
  p.pack_w = !p.few && !p.head && (p.f32 || a->D % 8 || a->ldw % 8 || !vae_aligned16(a->w));
  p.ldw = p.pack_w ? p.d_pad : a->ldw;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up_to(bytes, 256);
    return o;
  };
  p.x = take(p.planes * p.n_pad * p.d_pad * 2);
  p.w = take(p.pack_w ? p.planes * a->V * p.d_pad * 2 : 0);
  if (!bwd) {
    p.z_tiles = tiles_for(a->V, a->N, a->D, p.f32, 8.0, 0.0);
    p.z_parts = p.few ? few_parts : p.head ? parts_for(a->N) : p.z_tiles.split > 1 ? p.z_tiles.split : 0;
    p.partial = take(p.z_parts ? p.z_parts * a->N * p.ldz * 4 : up_to(a->V, 128) / 128 * p.n_pad * 8);
    p.tlogit = take(p.n_pad * 4);
    p.sums = take(p.n_pad * 8);
  } else {
    p.g = take(p.n_pad * 4);
    p.scale = take(8);
    const bool f16 = a->dtype == VAE_ADAMW_F16;       // (which of its calls have factors by row is not known here)
    p.factor = take(f16 ? p.n_pad * 4 : 0);
    p.scaled = take(f16 ? p.n_pad * p.d_pad * 2 : 0);
    const int64_t fit = D_BYTES / (p.planes * p.n_pad * 2) / 256 * 256, most = up_to(a->V, 256);
    p.piece = fit < 256 ? 256 : fit < most ? fit : most;
    // pieces of equal length
    const int64_t pieces = (most + p.piece - 1) / p.piece;
    p.piece = up_to((most + pieces - 1) / pieces, 256);
    p.d = take(p.planes * p.n_pad * p.piece * 2);
    p.d_tiles = tiles_for(p.piece, a->N, a->D, p.f32, p.f32 ? 55.0 : 12.0, 5.0);
    p.z_parts = p.few ? few_parts : p.d_tiles.split > 1 ? p.d_tiles.split : 0;
    p.sum_rows = p.z_parts ? SLAB_ROWS : p.d_tiles.big ? 256 : 128;
    p.z = take((int64_t)p.z_parts * a->N * p.ldz * 4);
    grads_for(a, p);
    if (p.few) {                                      // (as above: waves of 64 columns)
      const int64_t cols = (a->D + 63) / 64, fill = (4095 + cols) / cols, most_x = (a->V + 63) / 64, cap = most_x < 128 ? most_x : 128;
      p.dx_split = (int)(fill < cap ? fill : cap);
    }
    p.dx_slabs = p.few || p.dx_split > 1 || p.piece < a->V;
    p.slabs = take(p.dx_slabs ? (int64_t)p.dx_split * a->N * a->D * 4 : 0);
    p.slabs_w = take(p.dw_split > 1 ? (int64_t)p.dw_split * p.piece * a->D * 4 : 0);
    p.d_sums = take(a->bias ? p.n_pad / p.sum_rows * p.piece * 4 : 0);
  }
  p.bytes = at;
  return p;
}

uint32_t tiles_of(Gemm& g, bool big) {
  const int b = big ? 256 : 128;
  g.tiles_m = (g.M + b - 1) / b;
  g.tiles_n = (g.N + b - 1) / b;
  return (uint32_t)g.tiles_m * (uint32_t)g.tiles_n * (uint32_t)g.split;
}
template <int EPI> void logits(Gemm g, int dtype, bool big, hipStream_t st) {
  uint32_t grid = tiles_of(g, big);
  const uint32_t resident = big ? 256 : 512;
  if (EPI == EPI_STATS && grid > resident) grid = resident;             // workgroups that stay, as many as are resident
#define VAE_CE(F16, FINE)                                                                           \
  if (big) head_logits_kernel<F16, 256, 256, 2, 4, EPI, FINE><<<grid, 512, 0, st>>>(g);             \
  else head_logits_kernel<F16, 128, 128, 2, 2, EPI, FINE><<<grid, 256, 0, st>>>(g)
  if (dtype == VAE_ADAMW_F32) { VAE_CE(false, EPI != EPI_STORE); }
  else if (dtype == VAE_ADAMW_BF16) { VAE_CE(false, false); }
  else { VAE_CE(true, false); }
#undef VAE_CE
}
// partial logits, float slabs (split, N, ldz)
void store_logits(Gemm g, const Tiles& t, int64_t ldz, void* slabs, int dtype, hipStream_t st) {
  g.split = t.split;
  g.d_scale = g.row_factor = nullptr;
  g.out = slabs;
  g.ldo = ldz;
  logits<EPI_STORE>(g, dtype, t.big, st);
}
void gradients(Gemm dx, Gemm dw, bool want_dx, bool want_dw, int dtype, bool big, hipStream_t st) {
  const uint32_t nx = want_dx ? (tiles_of(dx, big) + 7) / 8 * 8 : 0, grid = nx + (want_dw ? tiles_of(dw, big) : 0);
#define VAE_CE(F16)                                                                                 \
  if (big) head_grads_kernel<F16, 256, 256, 2, 4><<<grid, 512, 0, st>>>(dx, dw, (int)nx);           \
  else head_grads_kernel<F16, 128, 128, 2, 2><<<grid, 256, 0, st>>>(dx, dw, (int)nx)
  if (dtype == VAE_ADAMW_F16) { VAE_CE(true); }
  else { VAE_CE(false); }
#undef VAE_CE
}
void finish(const Finish& f, int dtype, hipStream_t st) {
  const unsigned grid = (unsigned)(f.db_blocks + f.dw_blocks + f.dx_blocks);
  if (!grid) return;
  if (dtype == VAE_ADAMW_F32) ce_finish_kernel<float><<<grid, 256, 0, st>>>(f);
  else if (dtype == VAE_ADAMW_BF16) ce_finish_kernel<__bf16><<<grid, 256, 0, st>>>(f);
  else ce_finish_kernel<_Float16><<<grid, 256, 0, st>>>(f);
}

void pack(const vae_linear_ce* a, const Plan& p, uint8_t* ws, const int* state, const Rows& r, const Upstream& u, hipStream_t st) {
  auto blocks = [&](int64_t rows) {
    const int64_t b = (rows * (p.d_pad / 8) + 1023) / 1024;
    return (int)(b < 1024 ? b : 1024);
  };
  const Pack x = {a->x, a->ldx, state, (int)a->N, blocks(p.n_pad), reinterpret_cast<uint16_t*>(ws + p.x), p.n_pad * p.d_pad};
  const Pack w = {a->w, a->ldw, nullptr, (int)a->V, p.pack_w ? blocks(a->V) : 0, reinterpret_cast<uint16_t*>(ws + p.w), a->V * p.d_pad};
  const int grid = (u.up ? 1 : 0) + x.blocks + w.blocks;
  if (p.f32) ce_pack_kernel<float><<<grid, 1024, 0, st>>>(r, u, x, w, (int)a->D, p.d_pad);
  else ce_pack_kernel<uint16_t><<<grid, 1024, 0, st>>>(r, u, x, w, (int)a->D, p.d_pad);
}

template <typename T, bool HEAD> void few_logits(const vae_linear_ce* a, const Plan& p, const int* state, float* slabs, hipStream_t st) {
  const int per = (int)up_to((a->D + p.z_parts - 1) / p.z_parts, 64), N = (int)a->N, D = (int)a->D, V = (int)a->V, few = HEAD ? V : N;
  const dim3 grid((unsigned)(((HEAD ? a->N : a->V) + 127) / 128), (unsigned)p.z_parts);
  const T *w = reinterpret_cast<const T*>(a->w), *x = reinterpret_cast<const T*>(a->x);
  if (few <= 16) ce_few_z_kernel<T, 1, HEAD><<<grid, 256, 0, st>>>(w, a->ldw, x, a->ldx, state, N, D, V, per, slabs, p.ldz);
  else if (few <= 32) ce_few_z_kernel<T, 2, HEAD><<<grid, 256, 0, st>>>(w, a->ldw, x, a->ldx, state, N, D, V, per, slabs, p.ldz);
  else ce_few_z_kernel<T, 4, HEAD><<<grid, 256, 0, st>>>(w, a->ldw, x, a->ldx, state, N, D, V, per, slabs, p.ldz);
}
void few_dx(const vae_linear_ce* a, const Plan& p, const int* state, const float* d, const float* d_scale, float* slabs, hipStream_t st) {
  const int per = (int)up_to((a->V + p.dx_split - 1) / p.dx_split, 16), N = (int)a->N, D = (int)a->D, V = (int)a->V;
  const dim3 grid((unsigned)((a->D + 255) / 256), (unsigned)p.dx_split);
  const float* w = reinterpret_cast<const float*>(a->w);
  if (N <= 16) ce_few_dx_kernel<1><<<grid, 256, 0, st>>>(w, a->ldw, d, p.ldz, state, N, D, V, per, d_scale, slabs);
  else if (N <= 32) ce_few_dx_kernel<2><<<grid, 256, 0, st>>>(w, a->ldw, d, p.ldz, state, N, D, V, per, d_scale, slabs);
  else ce_few_dx_kernel<4><<<grid, 256, 0, st>>>(w, a->ldw, d, p.ldz, state, N, D, V, per, d_scale, slabs);
}

int check(const vae_linear_ce* a, const char* who) {
  VAE_REQUIRE(a, "%s: null arguments", who);
  VAE_REQUIRE(a->dtype >= 0 && a->dtype <= 2, "%s: unknown dtype %d", who, a->dtype);
  VAE_REQUIRE(a->N >= 1 && a->D >= 1 && a->V >= 1, "%s: N, D and V must be at least 1", who);
  VAE_REQUIRE(a->N <= (1ll << 24) && a->D <= (1ll << 20) && a->V <= (1ll << 24), "%s: at most 2^24 rows, 2^20 columns and 2^24 classes", who);
  // (a launch holds 2^32 threads: 2^24 tiles of 256)
  VAE_REQUIRE((a->N + 127) / 128 * ((a->V + 127) / 128) < (1ll << 24), "%s: more than 2^24 tiles of 128 rows and 128 classes", who);
  VAE_REQUIRE((a->N + 127) / 128 * ((a->D + 127) / 128) < (1ll << 24), "%s: more than 2^24 tiles of 128 rows and 128 columns", who);
  VAE_REQUIRE((a->V + 127) / 128 * ((a->D + 127) / 128) < (1ll << 24), "%s: more than 2^24 tiles of 128 classes and 128 columns", who);
  VAE_REQUIRE(a->x && a->w && a->target, "%s: null pointer", who);
  VAE_REQUIRE((a->N == 1 || a->ldx >= 0) && (a->V == 1 || a->ldw >= a->D), "%s: bad row stride", who);
  VAE_REQUIRE(a->ldw < (1ll << 22) && a->ldx < (1ll << 40), "%s: a row stride is too large", who);
  const uintptr_t bad = a->dtype == VAE_ADAMW_F32 ? 3 : 1;
  VAE_REQUIRE(((reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->w) | reinterpret_cast<uintptr_t>(a->bias)) & bad) == 0,
              "%s: a pointer is not aligned to its element", who);
  return VAE_OK;
}

Gemm logits_gemm(const vae_linear_ce* a, const Plan& p, uint8_t* ws, const int* state) {
  Gemm g = {};
  g.a = p.pack_w ? reinterpret_cast<const uint16_t*>(ws + p.w) : reinterpret_cast<const uint16_t*>(a->w);
  g.lda = p.ldw;
  g.plane_a = a->V * p.d_pad;
  g.b = reinterpret_cast<const uint16_t*>(ws + p.x);
  g.ldb = p.d_pad;
  g.plane_b = p.n_pad * p.d_pad;
  g.M = (int)a->V;
  g.N = (int)a->N;
  g.K = (int)(p.pack_w ? p.d_pad : a->D);
  g.segs = p.f32 ? 6 : 1;
  g.split = 1;
  g.dyn = state + S_KEPT;
  g.bias = a->bias;
  g.bias_f32 = p.f32;
  g.classes = state + S_ROWS + a->N;
  return g;
}

}  // namespace

extern "C" int64_t vae_linear_ce_state_bytes(int64_t N) { return (S_ROWS + 3 * N) * 4; }

extern "C" int64_t vae_linear_ce_workspace_bytes(const vae_linear_ce* a, int backward) {
  if (check(a, "vae_linear_ce_workspace_bytes")) return -1;
  if (small_head(a)) return 0;
  return plan_of(a, backward != 0).bytes;
}

extern "C" int vae_linear_ce_fwd(const vae_linear_ce* a, int reduction, float* loss, void* state, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  if (int rc = check(a, "vae_linear_ce_fwd")) return rc;
  VAE_REQUIRE(reduction >= VAE_CE_NONE && reduction <= VAE_CE_MEAN, "vae_linear_ce_fwd: unknown reduction %d", reduction);
  VAE_REQUIRE(loss && state, "vae_linear_ce_fwd: null pointer");
  if (small_head(a)) {
    Small m = small_args(a, reduction, state);
    m.loss = loss;
    small(m, a->dtype, false, (hipStream_t)stream);
    VAE_CHECK_LAUNCH("vae_linear_ce_fwd");
    return VAE_OK;
  }
  const Plan p = plan_of(a, false);
  VAE_REQUIRE(workspace && vae_aligned16(workspace) && workspace_bytes >= p.bytes,
              "vae_linear_ce_fwd: needs a 16-byte aligned workspace of vae_linear_ce_workspace_bytes()");
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  int* s = reinterpret_cast<int*>(state);
  hipStream_t st = (hipStream_t)stream;
  float* tl = reinterpret_cast<float*>(ws + p.tlogit);
  const Rows rows = {a->target, (int)a->N, (int)a->V, a->ignore_index, a->class_weight, s, tl, reduction == VAE_CE_NONE ? loss : nullptr};
  const bool unpacked = p.few || p.head, apart = unpacked || a->N > TABLE_ROWS;
  if (apart) ce_rows_kernel<<<1, 1024, 0, st>>>(rows);
  VAE_CHECK_LAUNCH("vae_linear_ce_fwd");
  if (!unpacked) pack(a, p, ws, s, apart ? Rows{} : rows, Upstream{}, st);
  VAE_CHECK_LAUNCH("vae_linear_ce_fwd");
  Gemm g = logits_gemm(a, p, ws, s);
  g.partial = reinterpret_cast<float2*>(ws + p.partial);
  g.target_logit = tl;
  const bool big = p.z_tiles.big;
  double* sums = reinterpret_cast<double*>(ws + p.sums);
  if (p.z_parts) {
    float* z = reinterpret_cast<float*>(ws + p.partial);
    if (p.few) few_logits<float, false>(a, p, s, z, st);
    else if (p.head && p.f32) few_logits<float, true>(a, p, s, z, st);
    else if (p.head && a->dtype == VAE_ADAMW_BF16) few_logits<__bf16, true>(a, p, s, z, st);
    else if (p.head) few_logits<_Float16, true>(a, p, s, z, st);
    else store_logits(g, p.z_tiles, p.ldz, ws + p.partial, a->dtype, st);
    VAE_CHECK_LAUNCH("vae_linear_ce_fwd");
    const float* slabs = reinterpret_cast<const float*>(ws + p.partial);
    const int S = p.z_parts, N = (int)a->N, V = (int)a->V;
    const unsigned narrow = N < 1024 ? (N + 3) / 4 : 256, wide = N < 512 ? N : 512;
#define VAE_CE(T)                                                                                                                  \
  const T* bias = reinterpret_cast<const T*>(a->bias);                                                                             \
  if (V <= 1024)                                                                                                                   \
    ce_slab_loss_kernel<T, 64><<<narrow, 256, 0, st>>>(slabs, S, p.ldz, bias, s, N, V, a->class_weight, reduction, sums, loss);     \
  else                                                                                                                             \
    ce_slab_loss_kernel<T, 1024><<<wide, 1024, 0, st>>>(slabs, S, p.ldz, bias, s, N, V, a->class_weight, reduction, sums, loss)
    if (p.f32) { VAE_CE(float); }
    else if (a->dtype == VAE_ADAMW_BF16) { VAE_CE(__bf16); }
    else { VAE_CE(_Float16); }
#undef VAE_CE
  } else {
    logits<EPI_STATS>(g, a->dtype, big, st);
    VAE_CHECK_LAUNCH("vae_linear_ce_fwd");
    const int b = big ? 256 : 128;
    ce_combine_kernel<<<(unsigned)((a->N + 31) / 32), 256, 0, st>>>(g.partial, (int)((a->V + b - 1) / b), p.n_pad, s, (int)a->N, a->class_weight, tl,
                                                                    reduction, sums, loss);
  }
  VAE_CHECK_LAUNCH("vae_linear_ce_fwd");
  return VAE_OK;
}

extern "C" int vae_linear_ce_bwd(const vae_linear_ce* a, int reduction, const float* grad, const void* state, void* dx, void* dw, void* dbias,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check(a, "vae_linear_ce_bwd")) return rc;
  VAE_REQUIRE(reduction >= VAE_CE_NONE && reduction <= VAE_CE_MEAN, "vae_linear_ce_bwd: unknown reduction %d", reduction);
  VAE_REQUIRE(grad && state && (dx || dw || dbias), "vae_linear_ce_bwd: null pointer");
  VAE_REQUIRE(!dbias || a->bias, "vae_linear_ce_bwd: a gradient of a bias that is not there");
  if (small_head(a)) {
    Small m = small_args(a, reduction, const_cast<void*>(state));
    m.up = grad;
    m.dx = dx;
    m.dw = dw;
    m.db = dbias;
    small(m, a->dtype, true, (hipStream_t)stream);
    VAE_CHECK_LAUNCH("vae_linear_ce_bwd");
    return VAE_OK;
  }
  const Plan p = plan_of(a, true);
  VAE_REQUIRE(workspace && vae_aligned16(workspace) && workspace_bytes >= p.bytes,
              "vae_linear_ce_bwd: needs a 16-byte aligned workspace of vae_linear_ce_workspace_bytes()");
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  const int* s = reinterpret_cast<const int*>(state);
  hipStream_t st = (hipStream_t)stream;
  float *gr = reinterpret_cast<float*>(ws + p.g), *scale = reinterpret_cast<float*>(ws + p.scale);
  float *slabs = reinterpret_cast<float*>(ws + p.slabs), *sums = reinterpret_cast<float*>(ws + p.d_sums);
  uint16_t *xp = reinterpret_cast<uint16_t*>(ws + p.x), *d = reinterpret_cast<uint16_t*>(ws + p.d);
  const int64_t plane_d = p.n_pad * p.piece, esize = p.f32 ? 4 : 2;
  const bool f16 = a->dtype == VAE_ADAMW_F16;
  float* factor = f16 && (reduction == VAE_CE_NONE || a->class_weight) ? reinterpret_cast<float*>(ws + p.factor) : nullptr;
  pack(a, p, ws, s, Rows{}, {grad, s, reduction, (int)a->N, a->class_weight, f16 ? 16384.f : 1.f, gr, scale, factor}, st);
  VAE_CHECK_LAUNCH("vae_linear_ce_bwd");
  if (factor && dw) {
    const int64_t blocks = (a->N * (p.d_pad / 8) + 255) / 256;
    ce_scale_rows_kernel<<<(unsigned)(blocks < 2048 ? blocks : 2048), 256, 0, st>>>(reinterpret_cast<const _Float16*>(xp), factor, s, p.d_pad,
                                                                                   reinterpret_cast<_Float16*>(ws + p.scaled));
    VAE_CHECK_LAUNCH("vae_linear_ce_bwd");
    xp = reinterpret_cast<uint16_t*>(ws + p.scaled);
  }
  for (int64_t v0 = 0; v0 < a->V; v0 += p.piece) {
    const int64_t n_v = a->V - v0 < p.piece ? a->V - v0 : p.piece;
    Gemm z = logits_gemm(a, p, ws, s);
    const uint16_t* w0 = z.a + v0 * z.lda;
    z.a = w0;
    z.M = (int)n_v;
    z.v0 = (int)v0;
    z.lse = reinterpret_cast<const float*>(s) + S_ROWS + 2 * a->N;
    z.g = gr;
    z.d_scale = scale;
    z.row_factor = factor;
    z.d = d;
    z.ldd = p.piece;
    z.plane_d = plane_d;
    z.d_sums = dbias ? sums : nullptr;
    if (p.z_parts) {                                    // (one piece: few rows, or classes that do not fill the chip)
      if (p.few) few_logits<float, false>(a, p, s, reinterpret_cast<float*>(ws + p.z), st);
      else store_logits(z, p.d_tiles, p.ldz, ws + p.z, a->dtype, st);
      VAE_CHECK_LAUNCH("vae_linear_ce_bwd");
      const dim3 grid((unsigned)((up_to(n_v, 64) + 1023) / 1024), (unsigned)(up_to(a->N, 64) / SLAB_ROWS));
      float* zs = reinterpret_cast<float*>(ws + p.z);
      float* to = dbias ? sums : nullptr;
#define VAE_CE(T)                                                                                                               \
  ce_slab_d_kernel<T><<<grid, 256, 0, st>>>(zs, p.few, p.z_parts, p.ldz, (const T*)a->bias, s, (int)a->N, (int)n_v, gr, scale, factor, d, \
                                            p.piece, plane_d, to)
      if (p.f32) VAE_CE(float);
      else if (a->dtype == VAE_ADAMW_BF16) VAE_CE(__bf16);
      else VAE_CE(_Float16);
#undef VAE_CE
    } else {
      logits<EPI_D>(z, a->dtype, p.d_tiles.big, st);
    }
    VAE_CHECK_LAUNCH("vae_linear_ce_bwd");
    Gemm gx = {}, gw = {};
    // dx (N, D) += d (N, n_v) W (n_v, D)
    gx.a = w0;
    gx.lda = z.lda;
    gx.plane_a = z.plane_a;
    gx.b = d;
    gx.ldb = p.piece;
    gx.plane_b = plane_d;
    gx.M = (int)a->D;
    gx.N = (int)a->N;
    gx.K = (int)n_v;
    gx.segs = z.segs;
    gx.dyn = s + S_KEPT;
    gx.d_scale = scale;
    gx.row_factor = factor;
    gx.out = p.dx_slabs ? (void*)slabs : dx;
    gx.out_kind = p.dx_slabs ? 0 : p.f32 ? 2 : 1;
    gx.rows = p.dx_slabs ? nullptr : s + S_ROWS;
    gx.ldo = a->D;
    gx.add = v0 > 0;
    gx.split = p.dx_split;
    // dW (n_v, D) = d^T (n_v, N) x (N, D)
    gw.a = xp;
    gw.lda = p.d_pad;
    gw.plane_a = p.n_pad * p.d_pad;
    gw.b = d;
    gw.ldb = p.piece;
    gw.plane_b = plane_d;
    gw.M = (int)a->D;
    gw.N = (int)n_v;
    gw.K = (int)a->N;
    gw.segs = z.segs;
    gw.split = p.dw_split;
    gw.dyn = s + S_KEPT;
    gw.dyn_k = 1;
    gw.d_scale = scale;
    gw.ldo = a->D;
    uint8_t* o = dw ? reinterpret_cast<uint8_t*>(dw) + v0 * a->D * esize : nullptr;
    gw.out = gw.split > 1 ? ws + p.slabs_w : o;
    gw.out_kind = gw.split > 1 ? 0 : p.f32 ? 2 : 1;
    const bool tiled_dx = dx && !p.few;
    if (dx && p.few) few_dx(a, p, s, reinterpret_cast<const float*>(ws + p.z), scale, slabs, st);
    if (tiled_dx || dw) gradients(gx, gw, tiled_dx, dw, a->dtype, p.grads_big, st);
    VAE_CHECK_LAUNCH("vae_linear_ce_bwd");
    Finish f = {};
    f.state = s;
    f.d_scale = scale;
    if (dbias) {
      f.db_blocks = (int)((n_v + 63) / 64);
      f.sums = sums;
      f.ld_sums = p.piece;
      f.sum_rows = p.sum_rows;
      f.V = (int)n_v;
      f.db = reinterpret_cast<uint8_t*>(dbias) + v0 * esize;
    }
    if (dw && gw.split > 1) {
      const int64_t work = (n_v * a->D + 1023) / 1024;
      f.dw_blocks = (int)(work < 4096 ? work : 4096);
      f.dw_slabs = reinterpret_cast<const float*>(ws + p.slabs_w);
      f.dw_split = gw.split;
      f.dw_n = n_v * a->D;
      f.dw = o;
    }
    if (dx && v0 + n_v == a->V) {
      f.dx_blocks = (int)(a->N < 4096 ? a->N : 4096);
      f.dx_slabs = p.dx_slabs ? slabs : nullptr;
      f.dx_split = p.dx_split;
      f.N = (int)a->N;
      f.D = (int)a->D;
      f.target = a->target;
      f.ignore = a->ignore_index;
      f.dx = dx;
    }
    finish(f, a->dtype, st);
    VAE_CHECK_LAUNCH("vae_linear_ce_bwd");
  }
  return VAE_OK;
}
