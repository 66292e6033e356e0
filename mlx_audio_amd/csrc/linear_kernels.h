// The linear layer behind the encoder stem: y = act(x W^T + b) + residual, and its backward pass
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
// as one matrix product kernel on the matrix cores, C[m][n] = sum_k A[n][k] B[m][k]:
//
//   forward   A = W  (n, k)  k contiguous      B = x  (m, k)  k contiguous
//   dx        A = W  (k, n)  n contiguous      B = dz (m, k)  k contiguous
//   dW        A = x  (k, n)  n contiguous      B = dz (k, m)  m contiguous
//
// (k is what is summed over, n the result's contiguous index.)  An operand whose k is contiguous
// lies in LDS as rows of 128 bytes of k and a lane's 16-byte fragment is one ds_read_b128; the other
// kind lies as rows of n (or m) and fragments are taken down the columns: ds_read_b64_tr_b16 for
// two-byte types, four ds_read_b32 for float.  Nothing is transposed in memory.
#pragma once
#include "nn_common.h"


namespace mia {
namespace lin {
using namespace nn;

struct Epilogue {
  const void* bias;      // (n) of the operands' type, or float (bias_f32), or null
  int bias_f32;
  int act;               // MIA_ACT_*
  const void* residual;  // rows of residual_stride elements, or null
  long long residual_stride;
  void* z;               // (m, n) contiguous: the value before the activation, or null
  void* out;             // (m, n) contiguous
};

struct Gemm {
  const void* a;
  const void* b;
  long long lda, ldb;  // elements between rows in memory
  int n, m, k;
  int n_tiles, m_tiles;
  int splits;          // parts of k, each with a plane of `partial`; 1: the epilogue runs at once
  int k_per_split;     // a multiple of the k of a step
  float* partial;      // (splits, m, n)
  Epilogue e;
};

// 0.5 erfc(-x / sqrt 2) from erfc(z) = t (a1 + t (a2 + ... t a7)) exp(-z^2), t = 1 / (1 + 0.51 z): the
// coefficients are the least relative error (7.2e-7) over 0 <= z <= 9.4, behind which the result is below
// 1e-38, found by reweighted least squares against erfc(z) exp(z^2).  So x Phi(x) keeps its digits in the
// negative tail; the exponent's argument, rounded three times, adds at most 1.5e-5 there (x = -12.9).
// `e` receives exp(-x^2 / 2).
__device__ __forceinline__ float normal_cdf_fast(float x, float& e) {
  const float z = __builtin_fabsf(x) * 0.70710678118654752440f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.51f, z, 1.0f));
  float q = fmaf(t, 0.09548515f, -0.3624904f);
  q = fmaf(t, q, 0.36299136f);
  q = fmaf(t, q, 0.05193581f);
  q = fmaf(t, q, 0.28020033f);
  q = fmaf(t, q, 0.28394583f);
  q = fmaf(t, q, 0.28793213f);
  e = __builtin_amdgcn_exp2f(-1.44269504088896340736f * z * z);
  const float half_erfc = 0.5f * t * q * e;
  return x < 0.0f ? half_erfc : 1.0f - half_erfc;
}
// Two-byte results: 1.5e-5 of a value and less is far below their rounding (2^-12 of it at the least).  float: the
// library's erfc.
template <bool PRECISE>
__device__ __forceinline__ float activate(float z, int act) {
  if (act == MIA_ACT_GELU) {
    if constexpr (PRECISE) return 0.5f * z * erfcf(-0.70710678118654752440f * z);
    float e;
    return z * normal_cdf_fast(z, e);
  }
  if (act == MIA_ACT_GELU_TANH) {  // z (1 + tanh u) / 2 = z / (1 + exp(-2 u))
    const float u2 = 1.5957691216057308f * fmaf(0.044715f * z * z, z, z);
    if constexpr (PRECISE) return z / (1.0f + expf(-u2));
    return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * u2));
  }
  if (act == MIA_ACT_RELU) return z < 0.0f ? 0.0f : z;  // keeps a NaN
  return z;
}
template <bool PRECISE>
__device__ __forceinline__ float derivative(float z, int act) {
  // at +-20 either GELU's slope is 0 or 1 exactly; the limit keeps z exp(-z^2 / 2) and z^3 from infinities (a
  // float16 preactivation is one beyond 65504) and a NaN a NaN
  if (act == MIA_ACT_GELU || act == MIA_ACT_GELU_TANH) z = z > 20.0f ? 20.0f : (z < -20.0f ? -20.0f : z);
  if (act == MIA_ACT_GELU) {
    float e, cdf;
    if constexpr (PRECISE) {
      cdf = 0.5f * erfcf(-0.70710678118654752440f * z);
      e = expf(-0.5f * z * z);
    } else {
      cdf = normal_cdf_fast(z, e);
    }
    return fmaf(z * 0.39894228040143267794f, e, cdf);
  }
  if (act == MIA_ACT_GELU_TANH) {
    const float u2 = 1.5957691216057308f * fmaf(0.044715f * z * z, z, z);
    const float s = 1.0f / (1.0f + expf(-u2));
    return fmaf(z * s * (1.0f - s), 1.5957691216057308f * fmaf(0.134145f * z, z, 1.0f), s);
  }
  if (act == MIA_ACT_RELU) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
  return 1.0f;
}

template <class T>
__device__ __forceinline__ float bias_at(const Epilogue& e, int n) {
  return e.bias_f32 ? static_cast<const float*>(e.bias)[n] : (float)static_cast<const T*>(e.bias)[n];
}

// One 16-byte piece of results: V columns of a row from `out` and `z` on, `left` of them inside the row
// (>= V: all); b: the bias, r: the residual's piece (zeros where there is none).
template <class T, int ACT, bool PLUS>
__device__ __forceinline__ void finish(T* out, T* z, int left, const float* b, u4 r, float* v) {
  constexpr int V = kPer16<T>;
  constexpr bool PRECISE = sizeof(T) == 4;
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] += b[j];
  // z is read by a backward pass, long after: past the caches.  (24000 x 1280 -> 5120, bfloat16, GELU: 412 ->
  // 399 us.  The result itself stays in them, though 386 us would do without: what follows reads it, and
  // a block of the encoder on 8 - 16 clips took 2 - 3 % longer then.)
  if (z) store_piece<T, true>(z, pack<T>(v), left);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = activate<PRECISE>(v[j], ACT);
  if constexpr (PLUS) {
    float x[V];
    unpack<T>(r, x);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += x[j];
  }
  store_piece(out, pack<T>(v), left);
}
// Calls f(activation, with or without residual) with what the epilogue asks for as constants: one
// branch before the results instead of several at each of them.
template <class F>
__device__ __forceinline__ void with_epilogue(const Epilogue& e, F f) {
  auto plus = [&](auto act) {
    if (e.residual) f(act, std::true_type());
    else f(act, std::false_type());
  };
  if (e.act == MIA_ACT_GELU) plus(std::integral_constant<int, MIA_ACT_GELU>());
  else if (e.act == MIA_ACT_GELU_TANH) plus(std::integral_constant<int, MIA_ACT_GELU_TANH>());
  else if (e.act == MIA_ACT_RELU) plus(std::integral_constant<int, MIA_ACT_RELU>());
  else plus(std::integral_constant<int, MIA_ACT_NONE>());
}
// the bias of V columns from n on, zeros where there is none
template <class T>
__device__ __forceinline__ void load_bias(const Epilogue& e, int n, int left, float* b) {
  constexpr int V = kPer16<T>;
#pragma unroll
  for (int j = 0; j < V; ++j) b[j] = 0.0f;
  if (!e.bias) return;
  if (e.bias_f32) {
#pragma unroll
    for (int j = 0; j < V; j += 4) unpack<float>(load_piece(static_cast<const float*>(e.bias) + n + j, left - j), b + j);
  } else {
    unpack<T>(load_piece(static_cast<const T*>(e.bias) + n, left), b);
  }
}
template <class T>
__device__ __forceinline__ u4 load_residual(const Epilogue& e, long long m, int n, int left) {
  return load_piece(static_cast<const T*>(e.residual) + m * e.residual_stride + n, left);
}

// reads as zero: the source of every piece that lies outside its operand
__device__ const u4 kZeros[1] = {};
}  // namespace lin

// Tile of BN x BM results, WN x WM waves.  An LDS stage holds 128 bytes of k (two matrix steps) of both
// operands: whole cache lines of an operand whose k is contiguous; two stages.
template <int BN_, int BM_, int WN_, int WM_, int OCC_>
struct LinTile {
  static constexpr int BN = BN_, BM = BM_, WN = WN_, WM = WM_, OCC = OCC_;
  static constexpr int NW = WN * WM, WG = 64 * NW;
  static constexpr int TN = BN / WN, TM = BM / WM;  // a wave's part
  static constexpr int RN = TN / 16, RM = TM / 16;  // ... in accumulators of 16 x 16
  static constexpr int A_BYTES = BN * 128, B_BYTES = BM * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int PA = BN / (8 * NW), PB = BM / (8 * NW);  // 1 KiB pieces per wave and stage
  static constexpr int LDS = 2 * STAGE;
  static_assert(TN % 32 == 0 && TM % 16 == 0 && BN % (8 * NW) == 0 && BM % (8 * NW) == 0, "whole pieces");
  static_assert(LDS <= 160 * 1024 && (STAGE & (STAGE - 1)) == 0, "LDS budget");
};
using LinTile256 = LinTile<256, 256, 2, 4, 1>;
using LinTile128 = LinTile<128, 128, 2, 2, 2>;
using LinTile64 = LinTile<64, 64, 1, 4, 4>;

namespace lin {
// One operand's tile in LDS and its fragments.  KC: k contiguous, LDS rows are `ROWS` operand rows
// of eight 16-byte pieces of k; otherwise LDS rows are the stage's k, ROWS elements each.  Piece c of
// LDS row r sits at piece position c ^ swizzle(r), so that the lanes served together by an LDS read fall on
// different banks (the counter of the forward product says no conflicts), but for column reads with Q = 8,
// below; with LDS-DMA the same permutation is applied to the source addresses.
template <class T, bool KC, int ROWS, int Q>
struct Operand {
  static constexpr int ES = (int)sizeof(T), V = 16 / ES;
  static constexpr int KSTEP = 128 / ES;                          // k of a stage
  static constexpr int PITCH = KC ? 128 : ROWS * ES;              // bytes of an LDS row
  static constexpr int PIECES = PITCH / 16;                       // pieces of an LDS row
  static __device__ __forceinline__ int swizzle(int r) {
    // a fragment read takes one piece of rows r .. r + 15 (Q = 4) or of 8 q + (0 .. 3) (Q = 8): two
    // rows lie in one span of all banks, the other three bits of the row choose the position
    if constexpr (KC) return Q == 4 ? (r >> 1) & 7 : ((r >> 1) & 1) | ((r >> 2) & 6);
    // column reads touch rows r .. r + 3 (two-byte: of 8 groups of rows) at one column range
    return ES == 2 ? (((r & 3) | ((r >> 1) & 4)) << 1) & (PIECES - 1) : ((r & 15) << 1) & (PIECES - 1);
  }
  // piece s of the stage: LDS byte s * 16; operand row / k of its first element
  static __device__ __forceinline__ void where(int s, int& row, int& k) {
    const int r = s / PIECES, c = (s % PIECES) ^ swizzle(r);
    if constexpr (KC) {
      row = r, k = c * V;
    } else {
      row = c * V, k = r;
    }
  }
  // The 16-byte fragment of tile row row0 + Q (r >> 2) + (r & 3), r = lane & 15, k piece 4 sub + (lane >> 4).
  // Q = 4: rows in order.  Q = 8 (two-byte types, first operand): the accumulators at row0 = base and
  // base + 4 together give lane group g of the result the rows base + 8 g ... + 7, so that a store of
  // 16 bytes a lane writes 64 consecutive bytes of 16 rows.  (Down the columns Q = 8 takes 8 of
  // every 16 bytes, half of the LDS banks, and each read twice its cycles: 40 % of the LDS cycles in dx, 33 % in
  // dW are such conflicts; with Q = 4 and stores of 8 bytes the gradients took 2 - 9 % longer.)
  static __device__ __forceinline__ u4 fragment(const unsigned char* tile, int row0, int sub, int lane) {
    const int r15 = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      const int row = row0 + Q * (r15 >> 2) + (r15 & 3);
      return *reinterpret_cast<const u4*>(tile + row * 128 + (((4 * sub + g) ^ swizzle(row)) << 4));
    } else if constexpr (ES == 2) {
      const int col = row0 + Q * (r15 & 3);  // this lane's quad of columns
      const int k0 = 32 * sub + 8 * g + (r15 >> 2);
      const unsigned base = (unsigned)(unsigned long long)tile;
      const int c = (col * 2) >> 4, in = (col * 2) & 15;
      const s4 lo = lds_read_column4(base + k0 * PITCH + ((c ^ swizzle(k0)) << 4) + in);
      const s4 hi = lds_read_column4(base + (k0 + 4) * PITCH + ((c ^ swizzle(k0 + 4)) << 4) + in);
      union {
        s4 h[2];
        u4 u;
      } x;
      x.h[0] = lo, x.h[1] = hi;
      return x.u;
    } else {
      const int col = row0 + r15;
      const int c = col >> 2, in = (col & 3) * 4;
      u4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = 16 * sub + 4 * g + j;
        x[j] = *reinterpret_cast<const unsigned*>(tile + k * PITCH + ((c ^ swizzle(k)) << 4) + in);
      }
      return x;
    }
  }
};
}  // namespace lin

namespace lin {
// One workgroup's piece of the product: a tile of the result and a range of k.
struct Place {
  int n0, m0, k_begin, k_end, split;
};
// `logical` counts tiles so that neighbours share rows of both operands: columns of four tiles along m.
template <class TL>
__device__ __forceinline__ Place place(const Gemm& p, unsigned logical) {
  Place w;
  const unsigned tiles = (unsigned)p.n_tiles * (unsigned)p.m_tiles;
  w.split = (int)(logical / tiles);
  logical -= (unsigned)w.split * tiles;
  constexpr unsigned GM = 4;
  const unsigned group = logical / (GM * (unsigned)p.n_tiles);
  const unsigned in_group = logical - group * GM * (unsigned)p.n_tiles;
  const unsigned gm = min(GM, (unsigned)p.m_tiles - group * GM);
  w.n0 = (int)(in_group / gm) * TL::BN;
  w.m0 = (int)(group * GM + in_group % gm) * TL::BM;
  w.k_begin = w.split * p.k_per_split;
  w.k_end = min(p.k, w.k_begin + p.k_per_split);
  return w;
}
// Workgroups go to the eight XCDs in turn: XCD x gets a contiguous share [first, first + count) of
// `total` tiles, so that one L2 serves neighbours.
__device__ __forceinline__ void xcd_share(unsigned total, unsigned xcd, unsigned& first, unsigned& count) {
  const unsigned q = total / 8, r = total % 8;
  first = xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q;
  count = q + (xcd < r ? 1 : 0);
}

// The stream of LDS-DMA loads of one wave.  A piece's place is a uniform base that moves with k and a
// fixed offset per lane.  Rows outside the operand repeat the last one (their results are never
// stored); the last stage of a k that is not a whole number of stages takes zeros behind it.
template <class TL, class T, bool AKC, bool BKC>
struct Stream {
  using OA = Operand<T, AKC, TL::BN, kPer16<T>>;
  using OB = Operand<T, BKC, TL::BM, 4>;
  static constexpr int ES = (int)sizeof(T), KSTEP = OA::KSTEP, P = TL::PA + TL::PB;
  unsigned offset[P];
  const char *base_a, *base_b;
  int left_k;              // behind the next stage's first k
  unsigned lds_a, lds_b, slot;  // slot: the next stage's buffer, byte 0 or byte STAGE

  __device__ __forceinline__ static void where(int i, int wv, int lane, int& row, int& k) {
    if (i < TL::PA) OA::where((TL::PA * wv + i) * 64 + lane, row, k);
    else OB::where((TL::PB * wv + i - TL::PA) * 64 + lane, row, k);
  }
  __device__ __forceinline__ void init(const unsigned char* smem, int wv) {
    const unsigned lds0 = (unsigned)(unsigned long long)smem;
    lds_a = (unsigned)__builtin_amdgcn_readfirstlane((int)(lds0 + (unsigned)(TL::PA * wv) * 1024u));
    lds_b = (unsigned)__builtin_amdgcn_readfirstlane((int)(lds0 + TL::A_BYTES + (unsigned)(TL::PB * wv) * 1024u));
    slot = 0;
  }
  // start and the rare part of issue work places out anew: without that the compiler would keep them in
  // registers that the matrix loop needs.
  static __device__ __forceinline__ int anew(int lane) {
    asm volatile("" : "+v"(lane));
    return lane;
  }
  __device__ __forceinline__ void start(const Gemm& p, const Place& w, int wv, int lane) {
    lane = anew(lane);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const bool isa = i < TL::PA, kc = isa ? AKC : BKC;
      int row, k;
      where(i, wv, lane, row, k);
      row = min(row, (isa ? p.n - w.n0 : p.m - w.m0) - (kc ? 1 : OA::V));
      const long long ld = isa ? p.lda : p.ldb;
      offset[i] = (unsigned)((kc ? row * ld + k : k * ld + row) * ES);
    }
    base_a = static_cast<const char*>(p.a) + (AKC ? w.n0 * p.lda + w.k_begin : w.k_begin * p.lda + w.n0) * ES;
    base_b = static_cast<const char*>(p.b) + (BKC ? w.m0 * p.ldb + w.k_begin : w.k_begin * p.ldb + w.m0) * ES;
    left_k = w.k_end - w.k_begin;
  }
  __device__ __forceinline__ void issue(const Gemm& p, int wv, int lane) {
    const unsigned to_a = (unsigned)__builtin_amdgcn_readfirstlane((int)(slot + lds_a));
    const unsigned to_b = (unsigned)__builtin_amdgcn_readfirstlane((int)(slot + lds_b));
    if (left_k >= KSTEP) {
#pragma unroll
      for (int i = 0; i < P; ++i)
        dma16(i < TL::PA ? base_a : base_b, offset[i], i < TL::PA ? to_a + 1024u * i : to_b + 1024u * (i - TL::PA));
    } else {
      lane = anew(lane);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        int row, k;
        where(i, wv, lane, row, k);
        const char* base = i < TL::PA ? base_a : base_b;
        dma16(k < left_k ? base + offset[i] : reinterpret_cast<const char*>(kZeros),
              i < TL::PA ? to_a + 1024u * i : to_b + 1024u * (i - TL::PA));
      }
    }
    base_a += (AKC ? (long long)KSTEP : KSTEP * p.lda) * ES;
    base_b += (BKC ? (long long)KSTEP : KSTEP * p.ldb) * ES;
    left_k -= KSTEP;
    slot ^= TL::STAGE;
  }
};

// A wave's part of the tile: its accumulators, and the two halves of a matrix step.
template <class TL, class T, bool AKC, bool BKC>
struct Part {
  static constexpr int HALF = kPer16<T> / 4;  // accumulators that make up 16 bytes of a lane
  using OA = Operand<T, AKC, TL::BN, 4 * HALF>;
  using OB = Operand<T, BKC, TL::BM, 4>;
  f4 acc[TL::RN][TL::RM];
  // fragments of one matrix step: the second operand's (two steps' worth: the next step's arrive while
  // this one's are used) and one half of the first operand's at a time, likewise twice
  static constexpr int RH = TL::RN / 2;
  u4 fa[2][RH], fb[2][TL::RM];
  int wn, wm, lane;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < TL::RN; ++i)
#pragma unroll
      for (int j = 0; j < TL::RM; ++j) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  __device__ __forceinline__ void init(int wv, int lane_) {
    wn = (wv % TL::WN) * TL::TN, wm = (wv / TL::WN) * TL::TM, lane = lane_;
    clear();
  }
  __device__ __forceinline__ void read_b(const unsigned char* stage, int sub) {
#pragma unroll
    for (int j = 0; j < TL::RM; ++j) fb[sub & 1][j] = OB::fragment(stage + TL::A_BYTES, wm + 16 * j, sub, lane);
  }
  __device__ __forceinline__ void read_a(const unsigned char* stage, int sub, int half) {
#pragma unroll
    for (int h = 0; h < RH; ++h) {
      const int i = half * RH + h;
      fa[half][h] = OA::fragment(stage, wn + 16 * HALF * (i / HALF) + 4 * (i % HALF), sub, lane);
    }
  }
  __device__ __forceinline__ void multiply(int sub, int half) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int h = 0; h < RH; ++h)
#pragma unroll
      for (int j = 0; j < TL::RM; ++j)
        acc[half * RH + h][j] = Mma<T>::step(fa[half][h], fb[sub & 1][j], acc[half * RH + h][j]);
    __builtin_amdgcn_s_setprio(0);
  }
  // One stage, beginning with read_b(stage, 0) and read_a(stage, 0, 0) done: every read goes out half
  // a step (RH x RM matrix instructions) before its use.  `turn` is called once all reads of the stage
  // have arrived; it may start the next stage's.
  template <class F>
  __device__ __forceinline__ void run_stage(const unsigned char* stage, F turn) {
    read_a(stage, 0, 1);
    multiply(0, 0);
    read_b(stage, 1);
    read_a(stage, 1, 0);
    multiply(0, 1);
    read_a(stage, 1, 1);
    multiply(1, 0);
    turn();
    multiply(1, 1);
  }
  __device__ __forceinline__ void begin_stage(const unsigned char* stage) {
    read_b(stage, 0);
    read_a(stage, 0, 0);
  }

  // accumulators HALF i ...: columns n0 + wn + 16 HALF i + V g ... of row m0 + wm + 16 j + (lane & 15)
  static constexpr int V = kPer16<T>, NP = TL::RN / HALF;
  // the vector stores of a tile without edges are at least this many
  static constexpr int STORES = TL::RM * NP;
  template <bool WHOLE, int ACT, bool PLUS>  // WHOLE: no edge of the result inside this tile
  __device__ __forceinline__ void finish_tile(const Gemm& p, const Place& w) {
    const int n_first = w.n0 + wn + V * (lane >> 4);
    const int m_first = w.m0 + wm + (lane & 15);
    auto left_of = [&](int i) { return WHOLE ? V : p.n - (n_first + 16 * HALF * i); };
    auto residual = [&](int i, int j) {
      if constexpr (PLUS) {
        const int m = m_first + 16 * j;
        return load_residual<T>(p.e, m, n_first + 16 * HALF * i, WHOLE || m < p.m ? left_of(i) : 0);
      }
      return u4{0, 0, 0, 0};
    };
    T* const out = static_cast<T*>(p.e.out) + (long long)m_first * p.n + n_first;
    T* const z = p.e.z ? static_cast<T*>(p.e.z) + (long long)m_first * p.n + n_first : nullptr;
    const long long step = 16LL * p.n;
    // bias and residual are loaded one piece ahead of the stores
    float next_bias[V];
    u4 next = residual(0, 0);
    load_bias<T>(p.e, n_first, left_of(0), next_bias);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      float bias[V];
#pragma unroll
      for (int t = 0; t < V; ++t) bias[t] = next_bias[t];
      if (i + 1 < NP) load_bias<T>(p.e, n_first + 16 * HALF * (i + 1), left_of(i + 1), next_bias);
#pragma unroll
      for (int j = 0; j < TL::RM; ++j) {
        const u4 now = next;
        if (j + 1 < TL::RM) next = residual(i, j + 1);
        else if (i + 1 < NP) next = residual(i + 1, 0);
        if (!WHOLE && (m_first + 16 * j >= p.m || left_of(i) <= 0)) continue;
        float v[V];
#pragma unroll
        for (int t = 0; t < V; ++t) v[t] = acc[HALF * i + t / 4][j][t % 4];
        const long long at = j * step + 16 * HALF * i;
        finish<T, ACT, PLUS>(out + at, z ? z + at : nullptr, left_of(i), bias, now, v);
      }
    }
  }
  __device__ __forceinline__ void store_part(const Gemm& p, const Place& w) {
    const int n_first = w.n0 + wn + V * (lane >> 4);
#pragma unroll
    for (int j = 0; j < TL::RM; ++j) {
      const long long m = w.m0 + wm + 16 * j + (lane & 15);
      if (m >= p.m) continue;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int n = n_first + 16 * HALF * i, left = p.n - n;
        if (left <= 0) continue;
        float v[V];
#pragma unroll
        for (int t = 0; t < V; ++t) v[t] = acc[HALF * i + t / 4][j][t % 4];
        float* out = p.partial + ((long long)w.split * p.m + m) * p.n + n;
#pragma unroll
        for (int t = 0; t < V; t += 4) store_piece(out + t, pack<float>(v + t), left - t);
      }
    }
  }
  static __device__ __forceinline__ bool whole(const Gemm& p, const Place& w) {
    return w.n0 + TL::BN <= p.n && w.m0 + TL::BM <= p.m;
  }
  __device__ __forceinline__ void store(const Gemm& p, const Place& w) {
    if (p.splits > 1) {
      store_part(p, w);
    } else if constexpr (!AKC) {  // a gradient
      if (whole(p, w)) finish_tile<true, MIA_ACT_NONE, false>(p, w);
      else finish_tile<false, MIA_ACT_NONE, false>(p, w);
    } else if (whole(p, w)) {
      with_epilogue(p.e, [&](auto act, auto plus) { finish_tile<true, decltype(act)::value, decltype(plus)::value>(p, w); });
    } else {
      with_epilogue(p.e, [&](auto act, auto plus) { finish_tile<false, decltype(act)::value, decltype(plus)::value>(p, w); });
    }
    if (!whole(p, w)) __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): pieces outside were loaded and not used
  }
};
}  // namespace lin

// Four waves, one tile per workgroup; several workgroups share a compute unit and fill each other's
// gaps (dW of 24000 x 1280 -> 5120, bfloat16: 334 us here, 352 with the 256 tile in two parts; float32,
// 6000 x 5120 -> 1280: 600 us, 131 TFLOP/s).
// DMA: every 16-byte piece of both operands is aligned (bases, row strides) and lies either
// wholly inside its operand or wholly outside; otherwise pieces go through registers, element by
// element at the edges.
template <class TL, class T, bool AKC, bool BKC, bool DMA>
__global__ __launch_bounds__(TL::WG, TL::OCC) void lin_gemm_kernel(lin::Gemm p) {
  using namespace lin;
  using ST = Stream<TL, T, AKC, BKC>;
  constexpr int KSTEP = ST::KSTEP, P = ST::P;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  unsigned first, count;
  xcd_share(gridDim.x, blockIdx.x & 7, first, count);
  const Place w = place<TL>(p, first + (blockIdx.x >> 3));
  const int steps = (w.k_end - w.k_begin + KSTEP - 1) / KSTEP;
  Part<TL, T, AKC, BKC> part;
  part.init(wv, lane);

  if constexpr (DMA) {
    ST st;
    st.init(smem, wv);
    st.start(p, w, wv, lane);
    if (steps > 0) st.issue(p, wv, lane);
    if (steps > 1) st.issue(p, wv, lane);
    if (steps > 1) wait_loads<P>();
    else wait_loads<0>();
    barrier_keep_loads();
    if (steps > 0) part.begin_stage(smem);
    for (int s = 0; s < steps; ++s) {
      part.run_stage(smem + (s & 1) * TL::STAGE, [&] {
        if (s + 1 == steps) return;
        // stage s + 1 has landed for this wave, and its reads of stage s have arrived; the barrier makes
        // that all waves: stage s + 2 may go where stage s was
        wait_loads<0>();
        barrier_keep_loads();
        if (s + 2 < steps) st.issue(p, wv, lane);
        part.begin_stage(smem + ((s + 1) & 1) * TL::STAGE);
      });
    }
  } else {
    // two stages ahead in registers: a stage is a fraction of memory's latency
    u4 held[2][P];
    auto fetch = [&](int step, u4(&to)[P]) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const bool isa = i < TL::PA, kc = isa ? AKC : BKC;
        int row, k;
        ST::where(i, wv, lane, row, k);
        row += isa ? w.n0 : w.m0;
        k += w.k_begin + step * KSTEP;
        const int rows = isa ? p.n : p.m;
        const long long ld = isa ? p.lda : p.ldb;
        const T* base = static_cast<const T*>(isa ? p.a : p.b);
        to[i] = u4{0, 0, 0, 0};
        if (row < rows && k < w.k_end)
          to[i] = kc ? load_piece(base + row * ld + k, w.k_end - k, (rows - 1 - row) * ld + p.k - k)
                     : load_piece(base + k * ld + row, rows - row, (p.k - 1 - k) * ld + rows - row);
      }
    };
    auto stage_step = [&](int s, u4(&now)[P]) {
      unsigned char* stage = smem + (s & 1) * TL::STAGE;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int at = i < TL::PA ? (TL::PA * wv + i) * 1024 : TL::A_BYTES + (TL::PB * wv + i - TL::PA) * 1024;
        *reinterpret_cast<u4*>(stage + at + lane * 16) = now[i];
      }
      __syncthreads();  // this stage is written; every wave is done with the other one
      if (s + 2 < steps) fetch(s + 2, now);
      part.begin_stage(stage);
      part.run_stage(stage, [] {});
    };
    if (steps > 0) fetch(0, held[0]);
    if (steps > 1) fetch(1, held[1]);
    for (int s = 0; s < steps; s += 2) {
      stage_step(s, held[0]);
      if (s + 1 < steps) stage_step(s + 1, held[1]);
    }
  }
  part.store(p, w);
}

// Eight waves, one workgroup per compute unit, which walks tiles (of one XCD's share) without a break
// in its stream of loads: stage g + 2 of the stream, which may be the next tile's, is loaded into the
// buffer of stage g as soon as all waves have read that, one stage before its use.  So at the end of
// a tile the results are stored while the next tile's first stages arrive; a wave waits for its loads,
// never for the stores behind them (loads and stores are counted in order: "all but the newest STORES").
// Measured, bfloat16: 8192^3 802 us (1 372 TFLOP/s); 24000 x 1280 -> 5120 351 us (897; with GELU and the
// preactivation 389 - 396), 24000 x 5120 -> 1280 259 (1 214).  A stage takes 1.57 us, of which the matrix instructions
// need 0.85 at 2.4 GHz; reading fragments and multiplying share the rest.  Short k is bound by the tile's end.
template <class TL, class T, bool AKC, bool BKC>
__global__ __launch_bounds__(TL::WG, 1) void lin_gemm8_kernel(lin::Gemm p) {
  using namespace lin;
  using ST = Stream<TL, T, AKC, BKC>;
  using PT = Part<TL, T, AKC, BKC>;
  constexpr int KSTEP = ST::KSTEP;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  unsigned first, count;
  xcd_share((unsigned)p.n_tiles * p.m_tiles * p.splits, blockIdx.x & 7, first, count);
  const unsigned stride = (gridDim.x + 7 - (blockIdx.x & 7)) / 8;  // workgroups on this XCD
  unsigned at = blockIdx.x >> 3;                                   // index in the XCD's share
  if (at >= count) return;

  Place w = place<TL>(p, first + at);
  PT part;
  part.init(wv, lane);
  ST st;
  st.init(smem, wv);
  // the stream's own position: it is up to two stages, possibly a tile, ahead
  unsigned load_at = at;
  st.start(p, w, wv, lane);
  bool more = true;
  auto issue = [&] {
    if (!more) return;
    st.issue(p, wv, lane);
    if (st.left_k <= 0) {
      load_at += stride;
      more = load_at < count;
      if (more) st.start(p, place<TL>(p, first + load_at), wv, lane);
    }
  };
  issue();
  issue();
  wait_loads<0>();
  barrier_keep_loads();
  unsigned buffer = 0;
  bool stored = false;  // stores of a whole tile are behind this wave's newest loads
  for (;;) {
    const int steps = (w.k_end - w.k_begin + KSTEP - 1) / KSTEP;
    part.begin_stage(smem + buffer);
    for (int s = 0; s < steps; ++s) {
      part.run_stage(smem + buffer, [&] {
        // this wave's reads of the stage and its loads of the next one have arrived; then all waves'
        if (stored) wait_loads<PT::STORES>();
        else wait_loads<0>();
        stored = false;
        barrier_keep_loads();
        issue();
        buffer ^= TL::STAGE;
        if (s + 1 < steps) part.begin_stage(smem + buffer);
      });
    }
    part.store(p, w);
    stored = PT::whole(p, w);
    at += stride;
    if (at >= count) break;
    w = place<TL>(p, first + at);
    part.clear();
  }
}

// The parts of a product that was split along k, added in order, and the epilogue.
template <class T>
__global__ __launch_bounds__(256) void lin_join_kernel(lin::Gemm p) {
  using namespace lin;
  constexpr int V = kPer16<T>;
  const int per_row = (p.n + V - 1) / V;
  const long long total = (long long)p.m * per_row;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long m = i / per_row;
    const int n = (int)(i - m * per_row) * V;
    const int left = p.n - n;
    float b[V], v[V] = {};
    load_bias<T>(p.e, n, left, b);
    const u4 r = p.e.residual ? load_residual<T>(p.e, m, n, left) : u4{0, 0, 0, 0};
    for (int s = 0; s < p.splits; ++s) {
      const float* src = p.partial + ((long long)s * p.m + m) * p.n + n;
#pragma unroll
      for (int t = 0; t < V; t += 4) {
        float x[4];
        unpack<float>(load_piece(src + t, left - t), x);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[t + j] += x[j];
      }
    }
    T* out = static_cast<T*>(p.e.out) + m * p.n + n;
    T* z = p.e.z ? static_cast<T*>(p.e.z) + m * p.n + n : nullptr;
    with_epilogue(p.e, [&](auto act, auto plus) {
      finish<T, decltype(act)::value, decltype(plus)::value>(out, z, left, b, r, v);
    });
  }
}

// Few rows of x (MT groups of 16): a stream through the weights.  A workgroup owns 16 columns of
// the result, its waves take 64-byte steps of k in turn and their sums meet in LDS.  Fragments come
// straight from memory: 16 bytes a lane, 64 bytes of each of 16 weight rows per load.
// 8 x 1280 -> 5120, bfloat16, GELU: 8 us for 13 MB of weights; a call takes 12, bound by the host.
template <class T, int MT, int NW>
__global__ __launch_bounds__(64 * NW) void lin_few_kernel(lin::Gemm p) {
  using namespace lin;
  constexpr int ES = (int)sizeof(T), V = 16 / ES, KSTEP = 64 / ES;
  constexpr int UNROLL = MT == 1 ? 4 : 2;
  __shared__ f4 part[NW][MT][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int r15 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const bool n_in = n0 + r15 < p.n;
  const T* __restrict__ a = static_cast<const T*>(p.a) + (long long)(n_in ? n0 + r15 : 0) * p.lda;
  const T* __restrict__ b[MT];
  bool m_in[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    m_in[j] = 16 * j + r15 < p.m;
    b[j] = static_cast<const T*>(p.b) + (long long)(m_in[j] ? 16 * j + r15 : 0) * p.ldb;
  }
  f4 acc[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) acc[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int k0 = wv * KSTEP; k0 < p.k; k0 += UNROLL * NW * KSTEP) {
    u4 fa[UNROLL], fb[UNROLL][MT];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int k = k0 + u * NW * KSTEP + g * V;
      fa[u] = load_piece(a + k, n_in ? p.k - k : 0, (p.n - 1 - n0 - r15) * p.lda + p.k - k);
#pragma unroll
      for (int j = 0; j < MT; ++j) fb[u][j] = load_piece(b[j] + k, m_in[j] ? p.k - k : 0, (p.m - 1 - 16 * j - r15) * p.ldb + p.k - k);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[j] = Mma<T>::step(fa[u], fb[u][j], acc[j]);
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) part[wv][j][lane] = acc[j];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 64; i += 64 * NW) {
    const int j = i / 64, l = i % 64;
    f4 s = part[0][j][l];
    for (int w = 1; w < NW; ++w) s += part[w][j][l];
    const long long m = 16 * j + (l & 15);
    const int n = n0 + 4 * (l >> 4);
    const int left = p.n - n;
    if (m >= p.m || left <= 0) continue;
    // four results: half a piece of a two-byte type, so element by element
    for (int t = 0; t < 4 && t < left; ++t) {
      float v = s[t];
      if (p.e.bias) v += bias_at<T>(p.e, n + t);
      const long long at = m * p.n + n + t;
      if (p.e.z) static_cast<T*>(p.e.z)[at] = (T)v;
      v = activate<sizeof(T) == 4>(v, p.e.act);
      if (p.e.residual) v += (float)static_cast<const T*>(p.e.residual)[m * p.e.residual_stride + n + t];
      static_cast<T*>(p.e.out)[at] = (T)v;
    }
  }
}

// dz = dy act'(z), rounded to the operands' type for the two products that read it, and the column
// sums of the unrounded values (float16: dz is a multiple of 2^-24, as dy is): workgroup (x, y) takes rows y, y + gridDim.y ... of 64 pieces of 16
// bytes, four rows at a time (one per wave).  24000 x 5120, bfloat16: 150 us, 4.9 TB/s.
// z null: no activation, sums only (dz null too).
template <class T>
__global__ __launch_bounds__(256) void lin_dz_kernel(const T* __restrict__ dy, long long dy_stride,
                                                     const T* __restrict__ z, long long z_stride, int act, int m,
                                                     int n, T* __restrict__ dz, float* __restrict__ partial) {
  using namespace lin;
  constexpr int V = kPer16<T>;
  __shared__ float cols[4][64 * V];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int c0 = (blockIdx.x * 64 + lane) * V;
  const int left = n - c0;
  float sum[V] = {};
  if (left > 0) {
    for (long long row = (long long)blockIdx.y * 4 + wv; row < m; row += (long long)gridDim.y * 4) {
      float g[V];
      unpack<T>(load_piece(dy + row * dy_stride + c0, left, (m - 1 - row) * dy_stride + left), g);
      if (z) {
        float zz[V];
        unpack<T>(load_piece(z + row * z_stride + c0, left, (m - 1 - row) * z_stride + left), zz);
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] *= derivative<sizeof(T) == 4>(zz[j], act);
        store_piece(dz + row * n + c0, pack<T>(g), left);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += g[j];
    }
  }
  if (!partial) return;
#pragma unroll
  for (int j = 0; j < V; ++j) cols[wv][lane * V + j] = sum[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * V; i += 256) {
    const int c = blockIdx.x * 64 * V + i;
    if (c < n) partial[(long long)blockIdx.y * n + c] = (cols[0][i] + cols[1][i]) + (cols[2][i] + cols[3][i]);
  }
}
namespace lin {
constexpr int kCus = 256;  // compute units of an MI355X
constexpr int kFewRows = 64;

struct Operands {
  const void* a;
  long long lda;
  const void* b;
  long long ldb;
  long long n, m, k;
};

struct Choice {
  int tile;    // 256, 128, 64
  int splits;
  int k_per_split;
};

static long long tiles_of(long long n, long long m, int tile) {
  return ((n + tile - 1) / tile) * ((m + tile - 1) / tile);
}

// The tile and the number of parts of k: the pair with the least estimated time, from the sizes alone
// (the workspace size follows from it).  The estimate is rounds of workgroups x (stages x time of a
// stage + start and end), and the join of the parts; its constants, in us, were measured with every
// tile forced in turn (bfloat16 / float32, all compute units busy):
//   256 x 256, one workgroup per compute unit:  1.6 / 7.2 a stage (1.8 / 11 with both operands by columns)
//   128 x 128, two:                             0.88 / 3.6
//   64 x 64, four:                              0.83 / 1.8
// e.g. 24000 x 1280 -> 1280: 256 75 us, 128 87, 64 121;  6000 x 1280 -> 1280: 36, 25, 36;
// 1500 x 1280 -> 1280: 128 18.5, 64 14.0;  1500 x 5120 -> 1280: 128 in 4 parts 34.8, in 2 38.0.
static Choice choose(long long n, long long m, long long k, size_t es, bool dma, bool columns) {
  struct Kind {
    int tile, per_cu;
    double stage2, stage4, ends;
  };
  static const Kind kinds[3] = {{256, 1, 1.6, 7.2, 6.0}, {128, 2, 0.88, 3.6, 4.0}, {64, 4, 0.83, 1.8, 3.0}};
  const int kstep = (int)(128 / es);
  const long long steps = (k + kstep - 1) / kstep;
  Choice best{128, 1, 0};  // (too large for any: refused when launched)
  double least = 0.0;
  for (const Kind& kd : kinds) {
    if (kd.tile == 256 && !dma) continue;
    const long long tiles = tiles_of(n, m, kd.tile);
    for (int splits = 1; splits <= 32 && (splits == 1 || steps / splits >= 4); ++splits) {
      const long long groups = tiles * splits, per_cu = (groups + kCus - 1) / kCus;
      if (kd.tile != 256 && groups >= (1LL << 24)) break;  // more threads than a launch counts
      const double load = per_cu < kd.per_cu ? (double)per_cu / kd.per_cu : 1.0;  // a stage is faster alone
      double stage = (es == 4 ? kd.stage4 : kd.stage2) * (0.45 + 0.55 * load);
      if (!dma) stage *= kd.tile == 64 ? 1.6 : columns ? 3.4 : 1.9;  // pieces through registers
      if (kd.tile == 256) stage = es == 4 ? (columns ? 11.0 : kd.stage4) : (columns ? 1.8 : kd.stage2);
      const long long rounds = (groups + (long long)kCus * kd.per_cu - 1) / ((long long)kCus * kd.per_cu);
      double t = (double)rounds * ((double)((steps + splits - 1) / splits) * stage + kd.ends);
      if (splits > 1) {  // parts written and read: 8 TB/s while the caches hold them, half of that beyond
        const double mb = 8e-6 * (double)splits * (double)m * (double)n;
        t += 6.0 + mb / 8.0 + (mb > 64.0 ? (mb - 64.0) / 8.0 : 0.0);
      }
      if (least == 0.0 || t < least) {
        least = t;
        best.tile = kd.tile, best.splits = splits;
      }
    }
  }
  const long long per = steps ? (steps + best.splits - 1) / best.splits : 1;
  best.splits = steps ? (int)((steps + per - 1) / per) : 1;
  best.k_per_split = (int)(per * kstep);
  return best;
}

template <class TL, class T, bool AKC, bool BKC, bool DMA>
static int launch(Gemm g, hipStream_t s) {
  g.n_tiles = (g.n + TL::BN - 1) / TL::BN;
  g.m_tiles = (g.m + TL::BM - 1) / TL::BM;
  const long long blocks = (long long)g.n_tiles * g.m_tiles * g.splits;
  // a launch counts its threads in 32 bits (the kernel of eight waves walks its tiles: 31 bits of them)
  if (blocks >= (TL::NW == 8 ? 1LL << 31 : (1LL << 32) / TL::WG)) {
    set_error("product too large for one launch");
    return MIA_ERR_UNSUPPORTED;
  }
  auto run = [&](auto kern, unsigned grid) {
    if constexpr (TL::LDS > 64 * 1024) {
      MIA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, TL::LDS));
    }
    hipLaunchKernelGGL(kern, dim3(grid), dim3(TL::WG), TL::LDS, s, g);
    return MIA_OK;
  };
  if constexpr (TL::NW == 8) return run(lin_gemm8_kernel<TL, T, AKC, BKC>, (unsigned)(blocks < kCus ? blocks : kCus));
  else return run(lin_gemm_kernel<TL, T, AKC, BKC, DMA>, (unsigned)blocks);
}

template <class T, bool AKC, bool BKC>
static int gemm(const Operands& o, const Epilogue& e, void* workspace, bool dma, hipStream_t s) {
  const Choice c = choose(o.n, o.m, o.k, sizeof(T), dma, !AKC && !BKC);
  Gemm g{o.a, o.b, o.lda, o.ldb, (int)o.n, (int)o.m, (int)o.k, 0, 0, c.splits, c.k_per_split,
         static_cast<float*>(workspace), e};
  int rc;
  if (dma) {
    rc = c.tile == 256   ? launch<LinTile256, T, AKC, BKC, true>(g, s)
         : c.tile == 128 ? launch<LinTile128, T, AKC, BKC, true>(g, s)
                         : launch<LinTile64, T, AKC, BKC, true>(g, s);
  } else {
    rc = c.tile == 128 ? launch<LinTile128, T, AKC, BKC, false>(g, s) : launch<LinTile64, T, AKC, BKC, false>(g, s);
  }
  if (rc != MIA_OK) return rc;
  if (c.splits > 1) {
    const long long work = o.m * ((o.n + kPer16<T> - 1) / kPer16<T>);
    const long long blocks = (work + 255) / 256;
    hipLaunchKernelGGL(lin_join_kernel<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, g);
  }
  return MIA_OK;
}

// 16-byte pieces that are aligned and never cross the operand's edge, 256 rows within 32 bits of offset
static bool pieces_ok(const void* p, long long ld, long long contiguous, size_t es) {
  const long long v = (long long)(16 / es);
  return aligned16(p) && ld % v == 0 && contiguous % v == 0 && ld * (long long)es < (1LL << 24);
}

static size_t split_bytes(long long n, long long m, long long k, size_t es, bool columns) {
  // both ways of loading may be taken (alignment is not known here): the larger of the two
  size_t most = 0;
  for (int dma = 0; dma < 2; ++dma) {
    const Choice c = choose(n, m, k, es, dma != 0, columns);
    const size_t need = c.splits > 1 ? (size_t)c.splits * m * n * sizeof(float) : 0;
    most = need > most ? need : most;
  }
  return most;
}

template <class T, int MT>
static void launch_few(const Gemm& g, hipStream_t s) {
  const unsigned blocks = (unsigned)((g.n + 15) / 16);
  hipLaunchKernelGGL((lin_few_kernel<T, MT, 8>), dim3(blocks), dim3(512), 0, s, g);
}
template <class T>
struct Ops {
  static int forward(const Operands& o, const Epilogue& e, void* workspace, hipStream_t s);
  static int input_gradient(const Operands& o, const Epilogue& e, void* workspace, hipStream_t s);
  static int weight_gradient(const Operands& o, const Epilogue& e, void* workspace, hipStream_t s);
  static void dz(const void* dy, long long dy_stride, const void* z, long long z_stride, int act, long long m,
                 long long n, void* dz, float* partial, int groups, hipStream_t s);
};
#ifdef MIA_LINEAR_TYPE
template <class T>
int Ops<T>::forward(const Operands& o, const Epilogue& e, void* workspace, hipStream_t s) {
  if (o.m <= kFewRows) {
    const Gemm g{o.a, o.b, o.lda, o.ldb, (int)o.n, (int)o.m, (int)o.k, 0, 0, 1, 0, nullptr, e};
    if (o.m <= 16) launch_few<T, 1>(g, s);
    else if (o.m <= 32) launch_few<T, 2>(g, s);
    else launch_few<T, 4>(g, s);
    return MIA_OK;
  }
  const bool dma = pieces_ok(o.a, o.lda, o.k, sizeof(T)) && pieces_ok(o.b, o.ldb, o.k, sizeof(T));
  return gemm<T, true, true>(o, e, workspace, dma, s);
}
template <class T>
int Ops<T>::input_gradient(const Operands& o, const Epilogue& e, void* workspace, hipStream_t s) {
  const bool dma = pieces_ok(o.a, o.lda, o.n, sizeof(T)) && pieces_ok(o.b, o.ldb, o.k, sizeof(T));
  return gemm<T, false, true>(o, e, workspace, dma, s);
}
template <class T>
int Ops<T>::weight_gradient(const Operands& o, const Epilogue& e, void* workspace, hipStream_t s) {
  const bool dma = pieces_ok(o.a, o.lda, o.n, sizeof(T)) && pieces_ok(o.b, o.ldb, o.m, sizeof(T));
  return gemm<T, false, false>(o, e, workspace, dma, s);
}
template <class T>
void Ops<T>::dz(const void* dy, long long dy_stride, const void* z, long long z_stride, int act, long long m,
                long long n, void* dz, float* partial, int groups, hipStream_t s) {
  constexpr long long cols = 64 * kPer16<T>;
  hipLaunchKernelGGL(lin_dz_kernel<T>, dim3((unsigned)((n + cols - 1) / cols), (unsigned)groups), dim3(256), 0, s,
                     static_cast<const T*>(dy), dy_stride, static_cast<const T*>(z), z_stride, act, (int)m, (int)n,
                     static_cast<T*>(dz), partial);
}
template struct Ops<MIA_LINEAR_TYPE>;
#endif
}  // namespace lin
}  // namespace mia
