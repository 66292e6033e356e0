// Attention for the transformer blocks behind the encoder stem, forward and backward.
//
//   s = scale q k^T (masked), lse = log sum exp s, out = exp(s - lse) v
//   p = exp(s - lse), dp = dout v^T, delta = sum_d dout out, ds = p (dp - delta)
//   dv = p^T dout, dk = scale ds^T q, dq = scale ds k
//
// No kernel keeps s or p in memory: the forward runs over the keys once with a running maximum and
// sum, the backward recomputes p from lse.  Every kernel has the same shape.  A wave OWNS 16 or 32
// rows (queries in the forward and in dq, keys in dk / dv) whose vectors stay in registers as the
// second operand of the matrix instruction; the other side's rows STREAM through LDS in tiles that
// all four waves of the workgroup share.  A product tile then has the own rows as its columns:
// lane l holds column l & 15 and the stream rows 4 (l >> 4) + i of each 16 - which is, for two such
// blocks (one for float), exactly the operand layout of the next product's second operand if the
// sum over stream rows is taken in that order.  So p and ds go from one product into the next
// without leaving their registers; only the first operand (v, k, dout, q by columns) is read from
// LDS down the columns (ds_read_b64_tr_b16; float: ds_read_b32).  Row maxima and sums need two lane
// exchanges.  dk / dv and dq are two launches: one launch would need atomics for dq, whose order
// changes its bits.
//
// float16 has too few exponents for the gradients' p and ds as they are (1500 keys: p is about 2^-11, ds
// less by the size of dout, and below 2^-14 float16 loses bits).  They go into their products times
// powers of two, taken out again in float32 when the result is stored: Scale and att_range_kernel.
#pragma once
#include "nn_common.h"

namespace mia {
namespace att {
using namespace nn;

struct View {  // [batch, row, head, dim], dim contiguous, strides in elements
  const void* p;
  long long b, s, h;
};
struct Args {
  View q, k, v, out, dout;
  void* o0;           // forward: out; dq; dk          (contiguous [batch, row, head, dim])
  void* o1;           // dv
  float* lse;         // (batch, heads, sq): written by the forward, read by the backward
  float* stats;       // backward: lse / ln 2 (+inf for an empty row), then delta, (batch, heads, sq) each;
                      // dq writes them, dk / dv reads them; float16: with dk / dv's Scale in them
  float* range;       // float16 gradients: (batch, kv_heads, range_parts, 2) bounds of the norms of v and dout
  int range_parts;
  const int* lengths; // (batch) keys of each batch item, or null
  int batch, sq, sk, heads, kv_heads, dim;
  int pack;           // heads that share a workgroup's rows: 1, or heads / kv_heads (few queries)
  int causal;         // query i sees keys <= i + sk - sq
  float scale;
  int own_tiles;      // workgroups along the own rows
  int splits;         // parts of the stream rows (forward: of the keys)
  int keys_per_split;
  float* partial;     // forward, splits > 1: (splits, rows, dim) sums, then (splits, rows, 2) max and sum;
                      // gradients: (splits, elements of dq) or (splits, elements of dk and of dv)
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_huge_valf();
__device__ const u4 kZeros[1] = {};
__device__ const float kInfinity[1] = {kInf};

// DP: the head dimension rounded up to what is computed, a multiple of 32.
template <class T, int DP>
struct Shape {
  static constexpr int ES = (int)sizeof(T), V = 16 / ES;
  static constexpr int TILE = ES == 2 ? 64 : 32;   // stream rows of a tile
  static constexpr int WIDTH = DP <= 64 ? 64 : 128;  // elements of an LDS row
  static constexpr int PITCH = WIDTH * ES;         // bytes of an LDS row
  static constexpr int PIECES = PITCH / 16;
  static constexpr int CC = DP * ES / 64;          // matrix steps along dim
  static constexpr int DT = DP / 16;               // accumulators along dim
  static constexpr int RB = ES == 2 ? 2 : 1;       // 16-row blocks of one matrix step along stream rows
  static constexpr int BYTES = TILE * PITCH;
  static constexpr int PW = BYTES / 4096;          // 1 KiB pieces per wave and tile
};

// Piece c of LDS row r lies at position c ^ turn(r), so that neither kind of read meets itself on one of the
// 64 banks.  Reads of 16 bytes are served 16 lanes at a time, lanes 0-3, 12-15, 20-23, 24-27, then 4-7, 8-11,
// 16-19, 28-31, and so on: rows 0-3 and 12-15 of piece g with rows 4-11 of piece g + 1, which lie apart because
// turn is even (a turn by bit 3 of the row as well brought them together: 4 cycles more for each such read, 33 -
// 40 % of all LDS cycles; without it the counter says none).  Reads down the columns are served 32 lanes at a
// time: 32 bytes of each of 8 rows, whose turn / 2 differs (float: 64 bytes of every fourth row, turn / 4).
template <class T, int DP>
__device__ __forceinline__ int turn(int r) {
  if (sizeof(T) == 4) return r & 15;
  return DP <= 64 ? r & 6 : (r & 7) << 1;
}
// A lane's place in LDS for either kind of read of a tile that starts at byte `tile` (a multiple of 1024),
// worked out once: every other address is it, with bits above the bank turned (^) and constants added.
template <class T, int DP>
__device__ __forceinline__ unsigned rows_place(unsigned tile, int lane) {
  const int row = lane & 15, g = lane >> 4;
  return tile + row * Shape<T, DP>::PITCH + ((g ^ turn<T, DP>(row)) << 4);
}
template <class T, int DP>
__device__ __forceinline__ unsigned columns_place(unsigned tile, int lane) {
  using S = Shape<T, DP>;
  const int r = lane & 15, g = lane >> 4;
  if constexpr (S::ES == 2) {
    const int row = 4 * g + (r >> 2);
    return tile + row * S::PITCH + ((((r & 3) >> 1) ^ turn<T, DP>(row)) << 4) + 8 * (r & 1);
  } else {
    return tile + 4 * g * S::PITCH + (((r >> 2) ^ turn<T, DP>(4 * g)) << 4) + 4 * (r & 3);
  }
}
typedef const __attribute__((address_space(3))) u4* lds_u4;
typedef const __attribute__((address_space(3))) unsigned* lds_u1;
// 16 bytes of 16 rows: row block `rb`, piece 4 cc + (lane >> 4)
template <class T, int DP>
__device__ __forceinline__ u4 rows_fragment(unsigned place, int rb, int cc) {
  return *(lds_u4)(unsigned long long)((place ^ (cc << 6)) + rb * 16 * Shape<T, DP>::PITCH);
}
// Columns: lane's column is d = 16 dt + (lane & 15), its elements are the stream rows of step `st` in
// the order of the product tiles: rows 4 (lane >> 4) + i of each 16-row block.
template <class T, int DP>
__device__ __forceinline__ u4 columns_fragment(unsigned place, int st, int dt) {
  using S = Shape<T, DP>;
  if constexpr (S::ES == 2) {
    const unsigned at = (place ^ (dt << 5)) + st * 32 * S::PITCH;
    union {
      s4 h[2];
      u4 u;
    } x;
    x.h[0] = lds_read_column4(at);
    x.h[1] = lds_read_column4(at + 16 * S::PITCH);
    return x.u;
  } else {
    u4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = *(lds_u1)(unsigned long long)((place ^ ((dt << 6) | (i << 4))) + (16 * st + i) * S::PITCH);
    return x;
  }
}
// the product tiles of one step as the next product's second operand.  Two-byte types are rounded here, the type
// that the matrix instruction takes: one rounding beside the stored result's, 1.4 of it together.
template <class T>
__device__ __forceinline__ u4 to_operand(const f4* blocks) {
  if constexpr (sizeof(T) == 2) {
    const float v[8] = {blocks[0][0], blocks[0][1], blocks[0][2], blocks[0][3],
                        blocks[1][0], blocks[1][1], blocks[1][2], blocks[1][3]};
    return pack<T>(v);
  } else {
    return __builtin_bit_cast(u4, blocks[0]);
  }
}

// what the rounding to T took away
template <class T, int RB>
__device__ __forceinline__ u4 rest_operand(const f4* blocks) {
  f4 rest[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) rest[r][i] = blocks[r][i] - (float)(T)blocks[r][i];
  return to_operand<T>(rest);
}

// Loads tiles of stream rows; rows at or past `end` read as zero whatever memory holds there, and so
// do elements past dim through registers.  DMA: straight into LDS (pieces aligned, dim a whole
// number of them); a place is then a uniform base plus a fixed offset per lane.  Pieces between dim and DP
// stay as `clear` leaves them, zero: the other operand is zero there, and anything else might be infinite.
// Pieces from DP on are never read; where dim is DP, they repeat the row's first one.
template <class T, int DP, bool DMA>
struct Loader {
  using S = Shape<T, DP>;
  unsigned offset[S::PW];
  unsigned long long lanes[S::PW];  // that load
  u4 held[DMA ? 1 : S::PW];
  static __device__ __forceinline__ void where(int i, int wv, int lane, int& r, int& c) {
    const int s = (S::PW * wv + i) * 64 + lane;
    r = s / S::PIECES, c = (s % S::PIECES) ^ turn<T, DP>(r);
  }
  __device__ __forceinline__ void init(long long stride, int dim, int wv, int lane) {
#pragma unroll
    for (int i = 0; i < S::PW; ++i) {
      int r, c;
      where(i, wv, lane, r, c);
      offset[i] = (unsigned)((r * stride + (c * S::V < dim ? c * S::V : 0)) * S::ES);
      lanes[i] = __ballot(dim == DP || c * S::V < dim);
    }
  }
  // Zeros past dim in both buffers of a tile, before the first load into them.
  static __device__ __forceinline__ void clear(unsigned char* tile, int dim, int wv, int lane) {
    if constexpr (DMA) {
      if (dim == DP) return;
#pragma unroll
      for (int i = 0; i < S::PW; ++i) {
        int r, c;
        where(i, wv, lane, r, c);
        unsigned char* at = tile + ((S::PW * wv + i) * 64 + lane) * 16;
        if (c * S::V >= dim) *reinterpret_cast<u4*>(at) = *reinterpret_cast<u4*>(at + 2 * S::BYTES) = u4{0, 0, 0, 0};
      }
    }
  }
  __device__ __forceinline__ void issue(const void* base, long long stride, int row0, int end, int dim, unsigned lds,
                                        int wv, int lane) {
    const char* from = static_cast<const char*>(base) + (long long)row0 * stride * S::ES;
    if constexpr (DMA) {
      const unsigned dst = (unsigned)__builtin_amdgcn_readfirstlane((int)(lds + (unsigned)(S::PW * wv) * 1024u));
      if (row0 + S::TILE <= end) {
#pragma unroll
        for (int i = 0; i < S::PW; ++i) dma16(from, offset[i], dst + 1024u * i, lanes[i]);
      } else {
#pragma unroll
        for (int i = 0; i < S::PW; ++i) {
          int r, c;
          where(i, wv, lane, r, c);
          dma16(row0 + r < end ? from + offset[i] : reinterpret_cast<const char*>(kZeros), dst + 1024u * i, lanes[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < S::PW; ++i) {
        int r, c;
        where(i, wv, lane, r, c);
        held[i] = u4{0, 0, 0, 0};
        if (row0 + r < end && c * S::V < dim)
          held[i] = load_piece(reinterpret_cast<const T*>(from) + r * stride + c * S::V, dim - c * S::V,
                               (end - 1 - row0 - r) * stride + dim - c * S::V);
      }
    }
  }
  __device__ __forceinline__ void commit(unsigned char* tile, int wv, int lane) {
    if constexpr (!DMA) {
#pragma unroll
      for (int i = 0; i < S::PW; ++i)
        *reinterpret_cast<u4*>(tile + ((S::PW * wv + i) * 64 + lane) * 16) = held[i];
    }
  }
};
// Keeps the compiler from doing a rare branch's selects always.
__device__ __forceinline__ void rarely() { asm volatile(""); }

// An own row's vector as the second operand: step cc, elements V (4 cc + (lane >> 4)) ...; `behind`:
// elements from the row's start to the start of the view's last row
template <class T, int DP>
__device__ __forceinline__ void load_own(const T* row, bool in, int dim, long long behind, int lane, u4* out) {
  using S = Shape<T, DP>;
#pragma unroll
  for (int cc = 0; cc < S::CC; ++cc) {
    const int e = (4 * cc + (lane >> 4)) * S::V;
    out[cc] = u4{0, 0, 0, 0};
    if (in && e < dim) out[cc] = load_piece(row + e, dim - e, behind + dim - e);
  }
}
// An own column's results: 4 consecutive d of every accumulator per lane.
template <class T, int DT, int N>
__device__ __forceinline__ void store_own(T* row, int dim, int lane, const f4 (&acc)[DT][N], int c, float factor) {
  struct __attribute__((packed, aligned(sizeof(T)))) Four {
    T e[4];
  };
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int d = 16 * dt + 4 * (lane >> 4);
    Four v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.e[i] = (T)(acc[dt][c][i] * factor);
    if (d + 4 <= dim) {
      *reinterpret_cast<Four*>(row + d) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (d + i < dim) row[d + i] = v.e[i];
    }
  }
}

// The workgroup's pair (of batch item and head) and its index among the pair's `per` workgroups.
// Workgroups go to the eight XCDs in turn; all of a pair go to one XCD, whose L2 then holds its keys
// and values, and the pairs go round the XCDs, so that items of different lengths spread evenly.
// With few pairs (less than 64) that would leave XCDs without work: in order then.  False: none.
static inline long long order_grid(long long pairs, long long per) {
  return pairs < 64 ? pairs * per : (pairs + 7) / 8 * 8 * per;
}
// A launch counts its threads in 32 bits; nothing is enqueued that does not fit.
static inline int check_grid(long long grid) {
  if (grid < (1LL << 24)) return MIA_OK;
  set_error("too many rows for one call (%lld workgroups)", grid);
  return MIA_ERR_UNSUPPORTED;
}
__device__ __forceinline__ bool order(unsigned pairs, unsigned per, unsigned& pair, unsigned& index) {
  if (pairs < 64) {
    pair = blockIdx.x / per;
    index = blockIdx.x - pair * per;
    return true;
  }
  const unsigned local = blockIdx.x >> 3, turn = local / per;
  index = local - turn * per;
  pair = turn * 8 + (blockIdx.x & 7);
  return pair < pairs;
}
__device__ __forceinline__ int keys_of(const Args& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.sk) : p.sk;
}
// The batch item of rank `r` by length, the longest first: work that ends last should be short.  (Up to
// 64 items, one per lane; more, or no lengths: in order.)
__device__ __forceinline__ int longest(const Args& p, int r) {
  if (!p.lengths || p.batch > 64) return r;
  const int lane = threadIdx.x & 63;
  const int mine = lane < p.batch ? p.lengths[lane] : -1;
  int rank = 0;
  for (int j = 0; j < p.batch; ++j) {
    const int other = __builtin_amdgcn_readlane(mine, j);
    rank += other > mine || (other == mine && j < lane) ? 1 : 0;
  }
  return __builtin_ctzll(__ballot(lane < p.batch && rank == r));
}
// one v_maximum3_f32 for two of them (fmaxf quiets its operands first); a NaN stays one
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// sum / maximum over the four lanes that hold a column
__device__ __forceinline__ float column_max(float v) {
  v = maximum(v, __shfl_xor(v, 16));
  return maximum(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
// a value that all lanes share, in a scalar register
__device__ __forceinline__ float uniform(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Powers of two that p and dp - delta are taken times, so that ds = p (dp - delta) fills float16's range:
// |dp - delta| <= |dout| (|v| + |out|) <= 2 |dout| max |v|, a row's out being a mean of values, so ds times
// 2^(p + dp) with the largest power that keeps that bound below 2^14 cannot overflow; p itself, at most 1,
// takes at most 2^14.  The factor of dp goes into its own operand, dout in dq and v in dk / dv (rounded there
// only where it is less than 1, and then by less than 2^-17 of the largest), and into delta.
struct Scale {
  int p, dp;
};
__device__ __forceinline__ int above(float x) {  // the least e with x < 2^e; x not below 2^-60
  return __builtin_amdgcn_frexp_expf(fmaxf(x, 0x1p-60f));
}
// dq: own is |dout| of a row, other the largest |v|.  Only ds meets float16 there: p takes what dp cannot.
__device__ __forceinline__ Scale dq_scale(float own, float other) {
  const float bound = 2.0f * own * other;
  if (!(bound < kInf)) return {0, 0};
  const int room = 14 - above(bound);
  const int p = min(room, 14);
  return {p, max(0, min(min(room - p, 14 - above(own)), 14))};
}
// dk / dv: own is the largest |v|, other the largest |dout|.  p is dv's operand as well: never less than itself.
__device__ __forceinline__ Scale dkv_scale(float own, float other) {
  const float bound = 2.0f * own * other;
  if (!(bound < kInf)) return {0, 0};
  const int room = 14 - above(bound);
  const int p = max(0, min(room, 14));
  return {p, min(min(room - p, max(0, 14 - above(own))), 14)};
}
// bounds of the norms of a key head's values (x) and of its query heads' dout rows (y)
__device__ __forceinline__ float2 norms_of(const Args& p, int b, int kvh) {
  const float* from = p.range + ((long long)b * p.kv_heads + kvh) * p.range_parts * 2;
  float2 most = {0.0f, 0.0f};
  for (int i = 0; i < p.range_parts; ++i) most.x = fmaxf(most.x, from[2 * i]), most.y = fmaxf(most.y, from[2 * i + 1]);
  return most;
}
// an own row's vector times 2^e
template <class T, int N>
__device__ __forceinline__ void scale_own(u4 (&v)[N], int e) {
  const float f = exp2_fast((float)e);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float x[kPer16<T>];
    unpack<T>(v[i], x);
#pragma unroll
    for (int j = 0; j < kPer16<T>; ++j) x[j] *= f;
    v[i] = pack<T>(x);
  }
}
}  // namespace att

// Forward.  OT: blocks of 16 queries per wave.  bfloat16, 8 x 1500, 20 heads of 64: 118 - 125 us (740 - 780 TFLOP/s),
// of which the vector ALUs are busy 89: for 64 keys x 32 queries 175 instructions and 32
// exponentials beside 32 matrix ones (38 us); the rest of the time the four waves of a SIMD do not overlap.  Four waves
// (128 registers) instead of three: 157 -> 140.  4 x 2048, 16 heads of 128: 148 us (927).  One query on 1500 keys, 16 items, 20 heads:
// 26 us with the join, HBM.
// BOTH: what the rounding of p to a two-byte type takes away goes through a second product, and the error falls from
// 1.39 to 1.00 of a result rounded once.  For calls whose rows (up to 64 of a pair) fit one workgroup: memory sets
// their time and the matrix units are mostly idle (16 x 1 on 1500 keys, 20 heads of 64: 26.8 -> 26.9 us; 16 x 64:
// 39.7 -> 41.8; 8 x 48 on 448, 6 heads: 10.4 -> 11.0).  Not with more rows, where it costs 7 - 20 % (1 x 1500,
// 20 heads of 64: 40 -> 46 us).
template <class T, int DP, int OT, bool DMA, bool BOTH>
__global__ __launch_bounds__(256, DP * (int)sizeof(T) <= 128 ? 4 : 2) void att_fwd_kernel(att::Args p) {
  using namespace att;
  using S = Shape<T, DP>;
  constexpr int KB = S::TILE / 16, STEPS = KB / S::RB;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * S::BYTES];  // two buffers of k and v
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4;

  const int hgs = p.heads / p.pack;
  unsigned pair, index;
  if (!order((unsigned)(p.batch * hgs), (unsigned)(p.own_tiles * p.splits), pair, index)) return;
  const int split = (int)(index % (unsigned)p.splits);
  // (causal: the last rows see most keys, so they start first)
  const int at_tile = (int)(index / (unsigned)p.splits), tile = p.causal ? p.own_tiles - 1 - at_tile : at_tile;
  const int hg = (int)(pair % (unsigned)hgs), b = longest(p, (int)(pair / (unsigned)hgs));
  const int kvh = hg * p.pack / (p.heads / p.kv_heads);
  const int all_rows = p.sq * p.pack;
  const int row0 = tile * (64 * OT) + wv * (16 * OT);
  const int off = p.sk - p.sq;
  const float c = p.scale * kLog2e;

  int len = keys_of(p, b);
  int k_begin = split * p.keys_per_split;
  int k_end = min(len, k_begin + p.keys_per_split);
  const int first_row = tile * (64 * OT), last_row = min(all_rows, first_row + 64 * OT) - 1;
  if (p.causal) {  // the furthest key that a row of this workgroup sees
    const int far = first_row / p.sq == last_row / p.sq ? last_row % p.sq : p.sq - 1;
    k_end = min(k_end, far + off + 1);
  }

  u4 own[OT][S::CC];
  int limit[OT];  // keys that the lane's query sees
#pragma unroll
  for (int o = 0; o < OT; ++o) {
    const int r = row0 + 16 * o + (lane & 15);
    const bool in = r < all_rows;
    const int hl = in ? r / p.sq : 0, s = in ? r - hl * p.sq : 0;
    load_own<T, DP>(static_cast<const T*>(p.q.p) + b * p.q.b + s * p.q.s + (hg * p.pack + hl) * p.q.h, in, p.dim,
                    (p.sq - 1 - s) * p.q.s, lane, own[o]);
    limit[o] = p.causal ? min(len, s + off + 1) : len;
  }
  // every key before this one is seen by all of the wave's rows
  int open = len;
  if (p.causal) {
    const int last = min(all_rows, row0 + 16 * OT) - 1;
    const int near = row0 < all_rows && row0 / p.sq == last / p.sq ? row0 % p.sq : 0;
    open = min(len, near + off + 1);
  }

  f4 acc[S::DT][OT];
  float ref[OT], sum[OT];
#pragma unroll
  for (int o = 0; o < OT; ++o) {
    ref[o] = -kInf, sum[o] = 0.0f;
#pragma unroll
    for (int d = 0; d < S::DT; ++d) acc[d][o] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const T* kp = static_cast<const T*>(p.k.p) + b * p.k.b + kvh * p.k.h;
  const T* vp = static_cast<const T*>(p.v.p) + b * p.v.b + kvh * p.v.h;
  const unsigned lds0 = (unsigned)(unsigned long long)smem;
  const unsigned rows0 = rows_place<T, DP>(lds0, lane), columns0 = columns_place<T, DP>(lds0, lane);
  Loader<T, DP, DMA> lk, lv;
  lk.init(p.k.s, p.dim, wv, lane);
  lv.init(p.v.s, p.dim, wv, lane);
  lk.clear(smem, p.dim, wv, lane);
  lv.clear(smem + S::BYTES, p.dim, wv, lane);
  const int tiles = k_end > k_begin ? (k_end - k_begin + S::TILE - 1) / S::TILE : 0;
  if (tiles) {
    lk.issue(kp, p.k.s, k_begin, k_end, p.dim, lds0, wv, lane);
    lv.issue(vp, p.v.s, k_begin, k_end, p.dim, lds0 + S::BYTES, wv, lane);
  }
  for (int t = 0; t < tiles; ++t) {
    unsigned char* kt = smem + (t & 1) * 2 * S::BYTES;
    unsigned char* vt = kt + S::BYTES;
    lk.commit(kt, wv, lane);
    lv.commit(vt, wv, lane);
    wait_loads<0>();
    barrier_keep_loads();  // tile t is there, and nobody reads the other buffer any more
    const unsigned rows = rows0 + (t & 1) * 2 * S::BYTES, columns = columns0 + (t & 1) * 2 * S::BYTES;
    const int k0 = k_begin + t * S::TILE;
    if (t + 1 < tiles) {
      const unsigned next = lds0 + ((t + 1) & 1) * 2 * S::BYTES;
      lk.issue(kp, p.k.s, k0 + S::TILE, k_end, p.dim, next, wv, lane);
      lv.issue(vp, p.v.s, k0 + S::TILE, k_end, p.dim, next + S::BYTES, wv, lane);
    }
    if (row0 >= all_rows) continue;

    f4 s[KB][OT];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int o = 0; o < OT; ++o) s[kb][o] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int cc = 0; cc < S::CC; ++cc)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const u4 f = rows_fragment<T, DP>(rows, kb, cc);
#pragma unroll
        for (int o = 0; o < OT; ++o) s[kb][o] = Mma<T>::step(f, own[o][cc], s[kb][o]);
      }
    if (k0 + S::TILE > min(open, k_end)) {
      rarely();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int o = 0; o < OT; ++o)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[kb][o][i] = k0 + 16 * kb + 4 * g + i < min(limit[o], k_end) ? s[kb][o][i] : -kInf;
    }
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      float m = s[0][o][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = maximum(m, s[kb][o][i]);
      // The reference that exponents are taken against follows the running maximum only when that is
      // more than 8 above it: p then stays below 2^8 (far from any type's limit; a sum's precision does
      // not depend on it), and after the first tiles nothing is rescaled any more.
      if (__any(m * c > ref[o] + 8.0f)) {
        rarely();
        const float top = fmaxf(ref[o], column_max(m) * c);
        const float alpha = top == -kInf ? 1.0f : exp2_fast(ref[o] - top);  // nothing seen yet: 0 or nothing to do
        ref[o] = top;
        sum[o] *= alpha;
#pragma unroll
        for (int d = 0; d < S::DT; ++d) acc[d][o] *= alpha;
      }
      const float minus = ref[o] == -kInf ? 0.0f : -ref[o];  // a row that has seen nothing: exp2(-inf) = 0
      float part[2] = {0.0f, 0.0f};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = exp2_fast(fmaf(s[kb][o][i], c, minus));
          s[kb][o][i] = e;
          part[i & 1] += e;
        }
      sum[o] += part[0] + part[1];
    }
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      u4 pf[OT], rest[OT];
#pragma unroll
      for (int o = 0; o < OT; ++o) {
        f4 blocks[S::RB];
#pragma unroll
        for (int r = 0; r < S::RB; ++r) blocks[r] = s[st * S::RB + r][o];
        pf[o] = to_operand<T>(blocks);
        if constexpr (BOTH) rest[o] = rest_operand<T, S::RB>(blocks);
      }
#pragma unroll
      for (int d = 0; d < S::DT; ++d) {
        const u4 f = columns_fragment<T, DP>(columns + S::BYTES, st, d);
#pragma unroll
        for (int o = 0; o < OT; ++o) {
          acc[d][o] = Mma<T>::step(f, pf[o], acc[d][o]);
          if constexpr (BOTH) acc[d][o] = Mma<T>::step(f, rest[o], acc[d][o]);
        }
      }
    }
  }

#pragma unroll
  for (int o = 0; o < OT; ++o) {
    const int r = row0 + 16 * o + (lane & 15);
    if (r >= all_rows) continue;   // (its other three lanes leave too)
    const float total = column_sum(sum[o]);
    const int hl = r / p.sq, s = r - hl * p.sq, h = hg * p.pack + hl;
    const long long at = ((long long)b * p.heads + h) * p.sq + s;
    if (p.splits > 1) {
      const long long n = (long long)p.batch * p.heads * p.sq, row = split * n + at;
      store_own<float>(p.partial + row * p.dim, p.dim, lane, acc, o, 1.0f);
      if (g == 0) {
        float* ml = p.partial + (long long)p.splits * n * p.dim + row * 2;
        ml[0] = ref[o];
        ml[1] = total;
      }
    } else {
      // an empty row (sum 0) is zero; a NaN in the sum stays one
      store_own<T>(static_cast<T*>(p.o0) + (((long long)b * p.sq + s) * p.heads + h) * p.dim, p.dim, lane, acc, o,
                   total == 0.0f ? 0.0f : 1.0f / total);
      if (g == 0 && p.lse) p.lse[at] = total == 0.0f ? -kInf : fmaf(ref[o], kLn2, logf(total));
    }
  }
}

// The parts of a row that was split along the keys: one wave per row.
template <class T>
__global__ __launch_bounds__(256) void att_join_kernel(att::Args p) {
  using namespace att;
  const long long n = (long long)p.batch * p.heads * p.sq;
  const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (at >= n) return;
  const float* __restrict__ ml = p.partial + (long long)p.splits * n * p.dim;
  float top = -kInf;
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, ml[(s * n + at) * 2]);
  const float base = top == -kInf ? 0.0f : top;
  float total = 0.0f, v[2] = {};
  for (int s = 0; s < p.splits; ++s) {
    const long long row = s * n + at;
    const float w = exp2_fast(ml[row * 2] - base);
    total = fmaf(w, ml[row * 2 + 1], total);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (lane + 64 * j < p.dim) v[j] = fmaf(w, p.partial[row * p.dim + lane + 64 * j], v[j]);
  }
  const long long bh = at / p.sq;
  const int s = (int)(at - bh * p.sq), h = (int)(bh % p.heads);
  const long long b = bh / p.heads;
  T* out = static_cast<T*>(p.o0) + ((b * p.sq + s) * p.heads + h) * p.dim;
  const float f = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (lane + 64 * j < p.dim) out[lane + 64 * j] = (T)(v[j] * f);
  if (lane == 0 && p.lse) p.lse[at] = total == 0.0f ? -kInf : fmaf(top, kLn2, logf(total));
}

// Bounds of the norms of a key head's v rows and of the dout rows of its query heads, over 1 / range_parts of
// them: 16 lanes a row, each with the largest sum of squares of its own 16 bytes over all rows; added up at
// the end they are at least the largest norm's square, and no row waits for an exchange of lanes.  Reads both once:
// 8 x 1500, 20 heads of 64: 15 us (61 MB, HBM) of a backward pass of 391; 16 x 1 on 1500: 15 of 102; 2 x 100, 6 heads: 3
// of 29.  What it buys: 1.7 - 4.7 times the error of a result rounded once, with dout of 1e-2 ... 1e-5, become 1.4.
template <class T>
__global__ __launch_bounds__(256) void att_range_kernel(att::Args p) {
  using namespace att;
  constexpr int V = kPer16<T>, AHEAD = 8;
  __shared__ float red[4][2];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int part = (int)(blockIdx.x % (unsigned)p.range_parts), pair = (int)(blockIdx.x / (unsigned)p.range_parts);
  const int kvh = pair % p.kv_heads, b = pair / p.kv_heads, group = p.heads / p.kv_heads;
  const int e = (lane & 15) * V;
  // rows of one head from `base` on, `count` of them
  auto largest = [&](const T* base, long long stride, int count, float most) {
    const int begin = (int)((long long)count * part / p.range_parts), end = (int)((long long)count * (part + 1) / p.range_parts);
    for (int row0 = begin + (int)(threadIdx.x >> 4); row0 < end; row0 += 16 * AHEAD) {
      u4 raw[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int row = row0 + 16 * i;
        raw[i] = u4{0, 0, 0, 0};
        if (row < end && e < p.dim)
          raw[i] = load_piece(base + row * stride + e, p.dim - e, (count - 1 - row) * stride + p.dim - e);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        float x[V], s = 0.0f;
        unpack<T>(raw[i], x);
#pragma unroll
        for (int j = 0; j < V; ++j) s = fmaf(x[j], x[j], s);
        most = fmaxf(most, s);
      }
    }
    return most;
  };
  float v = largest(static_cast<const T*>(p.v.p) + b * p.v.b + kvh * p.v.h, p.v.s, keys_of(p, b), 0.0f), g = 0.0f;
  for (int h = kvh * group; h < (kvh + 1) * group; ++h)
    g = largest(static_cast<const T*>(p.dout.p) + b * p.dout.b + h * p.dout.h, p.dout.s, p.sq, g);
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o)), g = fmaxf(g, __shfl_xor(g, o));
#pragma unroll
  for (int o = 8; o; o >>= 1) v += __shfl_xor(v, o), g += __shfl_xor(g, o);
  if (lane == 0) red[wv][0] = v, red[wv][1] = g;
  __syncthreads();
  if (threadIdx.x < 2)
    p.range[(long long)blockIdx.x * 2 + threadIdx.x] = sqrtf(fmaxf(
        fmaxf(red[0][threadIdx.x], red[1][threadIdx.x]), fmaxf(red[2][threadIdx.x], red[3][threadIdx.x])));
}

// dq: own rows are queries, k and v stream.  Runs first and leaves for dk / dv what each query needs there:
// stats[0] = lse / ln 2 (+inf for an empty row: its p becomes 0), stats[1] = delta = sum_d dout out.
// BOTH: as in the forward, for ds and up to 64 queries; the error of dq falls from 1.38 - 1.50 to 1.00 - 1.04 of
// a result rounded once.  The whole backward pass (bfloat16): 1 x 3662 keys 16.5 -> 17.9 us,
// 16 x 1 on 1500, 20 heads of 64: 86 -> 89, 16 x 64: 94 -> 101.  dk / dv keep one part (1.41): with two they would have
// to work on one block of keys per wave (16 x 1: 86 -> 106 us).
template <class T, int DP, int OT, bool DMA, bool BOTH>
__global__ __launch_bounds__(256, 2) void att_dq_kernel(att::Args p) {
  using namespace att;
  using S = Shape<T, DP>;
  constexpr int STEPS = S::TILE / 16 / S::RB;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * S::BYTES];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4;
  unsigned pair, index;
  if (!order((unsigned)(p.batch * p.heads), (unsigned)(p.own_tiles * p.splits), pair, index)) return;
  const int split = (int)(index % (unsigned)p.splits), at_tile = (int)(index / (unsigned)p.splits);
  const int tile = p.causal ? p.own_tiles - 1 - at_tile : at_tile;
  const int h = (int)(pair % (unsigned)p.heads), b = longest(p, (int)(pair / (unsigned)p.heads));
  const int kvh = h / (p.heads / p.kv_heads);
  const int row0 = tile * (64 * OT) + wv * (16 * OT);
  const int off = p.sk - p.sq;
  const float c = p.scale * kLog2e;
  const int len = keys_of(p, b);
  int k_end = len;
  if (p.causal) k_end = min(k_end, min(p.sq, tile * (64 * OT) + 64 * OT) + off);
  const int open = p.causal ? min(len, row0 + off + 1) : len;

  const long long n = (long long)p.batch * p.heads * p.sq;
  constexpr bool SCALED = std::is_same<T, _Float16>::value;
  u4 oq[OT][S::CC], og[OT][S::CC];
  float lse2[OT], delta[OT], factor[OT];
  int limit[OT];
  float2 most = {0.0f, 0.0f};
  Scale there = {0, 0};  // of dk / dv
  if constexpr (SCALED) most = norms_of(p, b, kvh), there = dkv_scale(most.x, most.y);
#pragma unroll
  for (int o = 0; o < OT; ++o) {
    const int s = row0 + 16 * o + (lane & 15);
    const bool in = s < p.sq;
    load_own<T, DP>(static_cast<const T*>(p.q.p) + b * p.q.b + s * p.q.s + h * p.q.h, in, p.dim,
                    (p.sq - 1 - s) * p.q.s, lane, oq[o]);
    load_own<T, DP>(static_cast<const T*>(p.dout.p) + b * p.dout.b + s * p.dout.s + h * p.dout.h, in, p.dim,
                    (p.sq - 1 - s) * p.dout.s, lane, og[o]);
    u4 oo[S::CC];
    load_own<T, DP>(static_cast<const T*>(p.out.p) + b * p.out.b + s * p.out.s + h * p.out.h, in, p.dim,
                    (p.sq - 1 - s) * p.out.s, lane, oo);
    float d = 0.0f, gg = 0.0f;
#pragma unroll
    for (int cc = 0; cc < S::CC; ++cc) {
      float x[S::V], y[S::V];
      unpack<T>(oo[cc], x);
      unpack<T>(og[o][cc], y);
#pragma unroll
      for (int j = 0; j < S::V; ++j) {
        d = fmaf(x[j], y[j], d);
        if constexpr (SCALED) gg = fmaf(y[j], y[j], gg);
      }
    }
    const long long at = ((long long)b * p.heads + h) * p.sq + s;
    const float l = in ? p.lse[at] : -kInf;
    delta[o] = column_sum(d);
    lse2[o] = l == -kInf ? kInf : l * kLog2e;
    factor[o] = p.scale;
    if (in && g == 0 && split == 0) {
      p.stats[at] = SCALED ? lse2[o] - (float)there.p : lse2[o];
      p.stats[n + at] = SCALED ? ldexpf(delta[o], there.dp) : delta[o];
    }
    if constexpr (SCALED) {
      const Scale here = dq_scale(sqrtf(column_sum(gg)), most.x);
      lse2[o] -= (float)here.p;
      delta[o] = ldexpf(delta[o], here.dp);
      scale_own<T>(og[o], here.dp);
      factor[o] = ldexpf(p.scale, -here.p - here.dp);
    }
    limit[o] = p.causal ? min(len, s + off + 1) : len;
  }
  f4 acc[S::DT][OT];
#pragma unroll
  for (int d = 0; d < S::DT; ++d)
#pragma unroll
    for (int o = 0; o < OT; ++o) acc[d][o] = f4{0.0f, 0.0f, 0.0f, 0.0f};

  const T* kp = static_cast<const T*>(p.k.p) + b * p.k.b + kvh * p.k.h;
  const T* vp = static_cast<const T*>(p.v.p) + b * p.v.b + kvh * p.v.h;
  const unsigned lds0 = (unsigned)(unsigned long long)smem;
  const unsigned rows0 = rows_place<T, DP>(lds0, lane), columns0 = columns_place<T, DP>(lds0, lane);
  Loader<T, DP, DMA> lk, lv;
  lk.init(p.k.s, p.dim, wv, lane);
  lv.init(p.v.s, p.dim, wv, lane);
  lk.clear(smem, p.dim, wv, lane);
  lv.clear(smem + S::BYTES, p.dim, wv, lane);
  const int all = k_end > 0 ? (k_end + S::TILE - 1) / S::TILE : 0;
  const int begin = (int)((long long)all * split / p.splits), end = (int)((long long)all * (split + 1) / p.splits);
  if (begin < end) {
    const unsigned at = lds0 + (begin & 1) * 2 * S::BYTES;
    lk.issue(kp, p.k.s, begin * S::TILE, k_end, p.dim, at, wv, lane);
    lv.issue(vp, p.v.s, begin * S::TILE, k_end, p.dim, at + S::BYTES, wv, lane);
  }
  for (int t = begin; t < end; ++t) {
    unsigned char* kt = smem + (t & 1) * 2 * S::BYTES;
    unsigned char* vt = kt + S::BYTES;
    lk.commit(kt, wv, lane);
    lv.commit(vt, wv, lane);
    wait_loads<0>();
    barrier_keep_loads();
    const unsigned rows = rows0 + (t & 1) * 2 * S::BYTES, columns = columns0 + (t & 1) * 2 * S::BYTES;
    const int k0 = t * S::TILE;
    if (t + 1 < end) {
      const unsigned next = lds0 + ((t + 1) & 1) * 2 * S::BYTES;
      lk.issue(kp, p.k.s, k0 + S::TILE, k_end, p.dim, next, wv, lane);
      lv.issue(vp, p.v.s, k0 + S::TILE, k_end, p.dim, next + S::BYTES, wv, lane);
    }
    if (row0 >= p.sq) continue;
    const bool masked = k0 + S::TILE > min(open, k_end);
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      f4 s[S::RB][OT], dp[S::RB][OT];
#pragma unroll
      for (int r = 0; r < S::RB; ++r)
#pragma unroll
        for (int o = 0; o < OT; ++o) {  // dp begins at -delta: it is only used less delta
          s[r][o] = f4{0.0f, 0.0f, 0.0f, 0.0f};
          dp[r][o] = f4{-delta[o], -delta[o], -delta[o], -delta[o]};
        }
#pragma unroll
      for (int cc = 0; cc < S::CC; ++cc)
#pragma unroll
        for (int r = 0; r < S::RB; ++r) {
          const u4 fk = rows_fragment<T, DP>(rows, st * S::RB + r, cc);
          const u4 fv = rows_fragment<T, DP>(rows + S::BYTES, st * S::RB + r, cc);
#pragma unroll
          for (int o = 0; o < OT; ++o) {
            s[r][o] = Mma<T>::step(fk, oq[o][cc], s[r][o]);
            dp[r][o] = Mma<T>::step(fv, og[o][cc], dp[r][o]);
          }
        }
      if (masked) {
        rarely();
#pragma unroll
        for (int o = 0; o < OT; ++o)
#pragma unroll
          for (int r = 0; r < S::RB; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              s[r][o][i] = k0 + 16 * (st * S::RB + r) + 4 * g + i < limit[o] ? s[r][o][i] : -kInf;
      }
      u4 df[OT], rest[OT];
#pragma unroll
      for (int o = 0; o < OT; ++o) {
        f4 blocks[S::RB];
#pragma unroll
        for (int r = 0; r < S::RB; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            blocks[r][i] = exp2_fast(fmaf(s[r][o][i], c, -lse2[o])) * dp[r][o][i];
          }
        df[o] = to_operand<T>(blocks);
        if constexpr (BOTH) rest[o] = rest_operand<T, S::RB>(blocks);
      }
#pragma unroll
      for (int d = 0; d < S::DT; ++d) {
        const u4 f = columns_fragment<T, DP>(columns, st, d);
#pragma unroll
        for (int o = 0; o < OT; ++o) {
          acc[d][o] = Mma<T>::step(f, df[o], acc[d][o]);
          if constexpr (BOTH) acc[d][o] = Mma<T>::step(f, rest[o], acc[d][o]);
        }
      }
    }
  }
#pragma unroll
  for (int o = 0; o < OT; ++o) {
    const int s = row0 + 16 * o + (lane & 15);
    if (s >= p.sq) continue;
    const long long at = (((long long)b * p.sq + s) * p.heads + h) * p.dim;
    if (p.splits > 1) store_own<float>(p.partial + split * n * p.dim + at, p.dim, lane, acc, o, factor[o]);
    else store_own<T>(static_cast<T*>(p.o0) + at, p.dim, lane, acc, o, factor[o]);
  }
}

// dk and dv: own rows are keys, q and dout stream, over all heads that share the key head.  With dq, bfloat16,
// 8 x 1500, 20 heads of 64: 359 us.  Two waves per SIMD: for three the registers spill (438 -> 552 us).
template <class T, int DP, int OT, bool DMA>
__global__ __launch_bounds__(256, DP * sizeof(T) > 256 ? 1 : 2) void att_dkv_kernel(att::Args p) {
  using namespace att;
  using S = Shape<T, DP>;
  constexpr int STEPS = S::TILE / 16 / S::RB;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * S::BYTES];
  __shared__ float rows_lse[2][64], rows_delta[2][64];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4;
  unsigned pair, index;
  if (!order((unsigned)(p.batch * p.kv_heads), (unsigned)(p.own_tiles * p.splits), pair, index)) return;
  const int split = (int)(index % (unsigned)p.splits);
  const int tile = (int)(index / (unsigned)p.splits);  // (causal: the first keys are seen by most queries)
  const int kvh = (int)(pair % (unsigned)p.kv_heads), b = (int)(pair / (unsigned)p.kv_heads);
  const int group = p.heads / p.kv_heads;
  const int key0 = tile * (64 * OT), row0 = key0 + wv * (16 * OT);
  const int off = p.sk - p.sq;
  const float c = p.scale * kLog2e;
  const int len = keys_of(p, b);

  u4 ok[OT][S::CC], ov[OT][S::CC];
#pragma unroll
  for (int o = 0; o < OT; ++o) {
    const int s = row0 + 16 * o + (lane & 15);
    load_own<T, DP>(static_cast<const T*>(p.k.p) + b * p.k.b + (long long)s * p.k.s + kvh * p.k.h, s < len, p.dim,
                    (p.sk - 1 - s) * p.k.s, lane, ok[o]);
    load_own<T, DP>(static_cast<const T*>(p.v.p) + b * p.v.b + (long long)s * p.v.s + kvh * p.v.h, s < len, p.dim,
                    (p.sk - 1 - s) * p.v.s, lane, ov[o]);
  }
  float of_dk = p.scale, of_dv = 1.0f;
  if constexpr (std::is_same<T, _Float16>::value) {
    const float2 most = norms_of(p, b, kvh);
    const Scale sc = dkv_scale(most.x, most.y);
    of_dk = uniform(ldexpf(p.scale, -sc.p - sc.dp)), of_dv = uniform(ldexpf(1.0f, -sc.p));
#pragma unroll
    for (int o = 0; o < OT; ++o) scale_own<T>(ov[o], sc.dp);
  }
  f4 dk[S::DT][OT], dv[S::DT][OT];
#pragma unroll
  for (int d = 0; d < S::DT; ++d)
#pragma unroll
    for (int o = 0; o < OT; ++o) dk[d][o] = dv[d][o] = f4{0.0f, 0.0f, 0.0f, 0.0f};

  // the first query that sees any of these keys; a workgroup past the length has nothing to do
  const int first = p.causal ? max(0, key0 - off) / S::TILE * S::TILE : 0;
  const int per_head = key0 < len && first < p.sq ? (p.sq - first + S::TILE - 1) / S::TILE : 0;
  const int all = per_head * group;
  const int begin = (int)((long long)all * split / p.splits), end = (int)((long long)all * (split + 1) / p.splits);
  const long long n = (long long)p.batch * p.heads * p.sq;
  const unsigned lds0 = (unsigned)(unsigned long long)smem;
  const unsigned rows0 = rows_place<T, DP>(lds0, lane), columns0 = columns_place<T, DP>(lds0, lane);
  const unsigned lse_at = (unsigned)(unsigned long long)&rows_lse[0][0];
  const unsigned delta_at = (unsigned)(unsigned long long)&rows_delta[0][0];
  Loader<T, DP, DMA> lq, lg;
  lq.init(p.q.s, p.dim, wv, lane);
  lg.init(p.dout.s, p.dim, wv, lane);
  lq.clear(smem, p.dim, wv, lane);
  lg.clear(smem + S::BYTES, p.dim, wv, lane);
  auto issue = [&](int t) {
    const int h = kvh * group + t / per_head, q0 = first + t % per_head * S::TILE;
    const unsigned at = lds0 + (t & 1) * 2 * S::BYTES;
    lq.issue(static_cast<const T*>(p.q.p) + b * p.q.b + h * p.q.h, p.q.s, q0, p.sq, p.dim, at, wv, lane);
    lg.issue(static_cast<const T*>(p.dout.p) + b * p.dout.b + h * p.dout.h, p.dout.s, q0, p.sq, p.dim, at + S::BYTES,
             wv, lane);
    const bool in = lane < S::TILE && q0 + lane < p.sq;
    const float* from = p.stats + ((long long)b * p.heads + h) * p.sq + q0 + lane;
    if (wv == 0) dma4(in ? from : kInfinity, (unsigned)__builtin_amdgcn_readfirstlane((int)(lse_at + (t & 1) * 256u)));
    if (wv == 1)
      dma4(in ? from + n : reinterpret_cast<const float*>(kZeros),
           (unsigned)__builtin_amdgcn_readfirstlane((int)(delta_at + (t & 1) * 256u)));
  };
  if (begin < end) issue(begin);
  for (int t = begin; t < end; ++t) {
    unsigned char* qt = smem + (t & 1) * 2 * S::BYTES;
    unsigned char* gt = qt + S::BYTES;
    lq.commit(qt, wv, lane);
    lg.commit(gt, wv, lane);
    wait_loads<0>();
    barrier_keep_loads();
    const unsigned rows = rows0 + (t & 1) * 2 * S::BYTES, columns = columns0 + (t & 1) * 2 * S::BYTES;
    const int q0 = first + t % per_head * S::TILE;
    if (t + 1 < end) issue(t + 1);
    if (row0 >= len) continue;
    const bool masked = row0 + 16 * OT > len || (p.causal && row0 + 16 * OT - 1 > q0 + off);
    // the row fragments of a step are read while the step before it works on its products
    u4 rq[S::RB][S::CC], rg[S::RB][S::CC];
    f4 lse2[S::RB], delta[S::RB];
    auto read_rows = [&](int st) {
#pragma unroll
      for (int r = 0; r < S::RB; ++r) {
        const int at = 16 * (st * S::RB + r) + 4 * g;
        lse2[r] = *reinterpret_cast<const f4*>(&rows_lse[t & 1][at]);
        delta[r] = *reinterpret_cast<const f4*>(&rows_delta[t & 1][at]);
#pragma unroll
        for (int cc = 0; cc < S::CC; ++cc) {
          rq[r][cc] = rows_fragment<T, DP>(rows, st * S::RB + r, cc);
          rg[r][cc] = rows_fragment<T, DP>(rows + S::BYTES, st * S::RB + r, cc);
        }
      }
    };
    read_rows(0);
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      f4 s[S::RB][OT], dp[S::RB][OT];  // dp begins at -delta: it is only used less delta
#pragma unroll
      for (int r = 0; r < S::RB; ++r)
#pragma unroll
        for (int o = 0; o < OT; ++o) s[r][o] = f4{0.0f, 0.0f, 0.0f, 0.0f}, dp[r][o] = -delta[r];
#pragma unroll
      for (int cc = 0; cc < S::CC; ++cc)
#pragma unroll
        for (int r = 0; r < S::RB; ++r)
#pragma unroll
          for (int o = 0; o < OT; ++o) {
            s[r][o] = Mma<T>::step(rq[r][cc], ok[o][cc], s[r][o]);
            dp[r][o] = Mma<T>::step(rg[r][cc], ov[o][cc], dp[r][o]);
          }
      f4 minus[S::RB];
#pragma unroll
      for (int r = 0; r < S::RB; ++r) minus[r] = -lse2[r];
      if (st + 1 < STEPS) read_rows(st + 1);
      if (masked) {
        rarely();
#pragma unroll
        for (int o = 0; o < OT; ++o) {
          const int key = row0 + 16 * o + (lane & 15);
#pragma unroll
          for (int r = 0; r < S::RB; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int q = q0 + 16 * (st * S::RB + r) + 4 * g + i;
              s[r][o][i] = key < len && (!p.causal || key <= q + off) ? s[r][o][i] : -kInf;
            }
        }
      }
      u4 pf[OT], df[OT];
#pragma unroll
      for (int o = 0; o < OT; ++o) {
        f4 pb[S::RB], db[S::RB];
#pragma unroll
        for (int r = 0; r < S::RB; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = exp2_fast(fmaf(s[r][o][i], c, minus[r][i]));
            pb[r][i] = e;
            db[r][i] = e * dp[r][o][i];
          }
        pf[o] = to_operand<T>(pb);
        df[o] = to_operand<T>(db);
      }
#pragma unroll
      for (int d = 0; d < S::DT; ++d) {
        const u4 fg = columns_fragment<T, DP>(columns + S::BYTES, st, d);
        const u4 fq = columns_fragment<T, DP>(columns, st, d);
#pragma unroll
        for (int o = 0; o < OT; ++o) {
          dv[d][o] = Mma<T>::step(fg, pf[o], dv[d][o]);
          dk[d][o] = Mma<T>::step(fq, df[o], dk[d][o]);
        }
      }
    }
  }
#pragma unroll
  for (int o = 0; o < OT; ++o) {
    const int s = row0 + 16 * o + (lane & 15);
    if (s >= p.sk) continue;
    if (s >= len) {  // zero whatever dout holds (0 x inf in the sums would not be)
#pragma unroll
      for (int d = 0; d < S::DT; ++d) dk[d][o] = dv[d][o] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const long long at = (((long long)b * p.sk + s) * p.kv_heads + kvh) * p.dim;
    if (p.splits > 1) {
      const long long count = (long long)p.batch * p.sk * p.kv_heads * p.dim;
      store_own<float>(p.partial + 2 * split * count + at, p.dim, lane, dk, o, of_dk);
      store_own<float>(p.partial + (2 * split + 1) * count + at, p.dim, lane, dv, o, of_dv);
    } else {
      store_own<T>(static_cast<T*>(p.o0) + at, p.dim, lane, dk, o, of_dk);
      store_own<T>(static_cast<T*>(p.o1) + at, p.dim, lane, dv, o, of_dv);
    }
  }
}

// Gradients' parts added in order: out[i] = sum over splits of partial[split * total + i], i < total; the
// first n go to out0, the rest to out1.
template <class T>
__global__ __launch_bounds__(256) void att_add_kernel(const float* __restrict__ partial, long long total, int splits,
                                                      long long n, T* __restrict__ out0, T* __restrict__ out1) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    float v = partial[i];
    for (int s = 1; s < splits; ++s) v += partial[s * total + i];
    (i < n ? out0[i] : out1[i - n]) = (T)v;
  }
}

namespace att {
constexpr int kCus = 256;

struct Plan {
  int pack, own_tiles, splits, keys_per_split, own_blocks;
};
constexpr int kFewQueries = 64;  // with no more, two-byte p (forward) and ds (dq) go into their product in two parts
// Queries: 128 per workgroup (32 per wave), or 64 where that leaves compute units without work; then
// the keys are split until there are two workgroups per unit.
static Plan plan_forward(long long batch, long long sq, long long sk, int heads, int kv_heads) {
  Plan p;
  const int group = heads / kv_heads;
  p.pack = sq * group <= 64 ? group : 1;
  const long long rows = sq * p.pack, outer = batch * (heads / p.pack);
  p.own_blocks = outer * ((rows + 127) / 128) >= 2 * kCus && rows > 64 ? 2 : 1;
  p.own_tiles = (int)((rows + 64 * p.own_blocks - 1) / (64 * p.own_blocks));
  const long long groups = outer * p.own_tiles;
  long long splits = groups ? (4 * kCus) / groups : 1;
  const long long most = (sk + 255) / 256;  // at least 256 keys each
  if (splits > most) splits = most;
  if (splits > 64) splits = 64;
  if (splits < 1) splits = 1;
  long long per = (sk + splits - 1) / splits;
  per = (per + 63) / 64 * 64;
  if (per < 64) per = 64;
  p.splits = (int)((sk + per - 1) / per);
  if (p.splits < 1) p.splits = 1;
  p.keys_per_split = (int)per;
  return p;
}
// One gradient kernel: `outer` pairs of `own` rows each, `stream` tiles to run over per workgroup.
struct GradPlan {
  int own_blocks, own_tiles, splits;
};
static GradPlan plan_gradient(long long outer, long long own, long long stream, bool two_blocks) {
  GradPlan p;
  p.own_blocks = two_blocks && own > 64 && outer * ((own + 127) / 128) >= 2 * kCus ? 2 : 1;
  p.own_tiles = (int)((own + 64 * p.own_blocks - 1) / (64 * p.own_blocks));
  const long long groups = outer * p.own_tiles;
  long long splits = groups ? 2 * kCus / groups : 1;  // two workgroups per compute unit
  if (splits > stream / 4) splits = stream / 4;       // of at least four tiles each
  if (splits > 16) splits = 16;
  p.splits = splits < 1 ? 1 : (int)splits;
  return p;
}
static long long stream_tiles(long long rows, size_t es) { return (rows + (es == 2 ? 63 : 31)) / (es == 2 ? 64 : 32); }
static GradPlan plan_dkv(long long batch, long long sq, long long sk, int heads, int kv_heads, int dim, size_t es) {
  // (two blocks of keys with vectors of more than 128 bytes would not fit the registers)
  return plan_gradient(batch * kv_heads, sk, stream_tiles(sq, es) * (heads / kv_heads), dim * (int)es <= 128);
}
static GradPlan plan_dq(long long batch, long long sq, long long sk, int heads, size_t es) {
  return plan_gradient(batch * heads, sq, stream_tiles(sk, es), true);
}
// Workgroups of a pair of att_range_kernel: four per compute unit, of at least 128 rows each.
static int range_parts(long long batch, long long sq, long long sk, int heads, int kv_heads) {
  const long long pairs = batch * kv_heads, rows = sk + sq * (heads / kv_heads);
  long long parts = pairs ? (4 * kCus + pairs - 1) / pairs : 1;
  if (parts > rows / 128) parts = rows / 128;
  return (int)(parts < 1 ? 1 : parts > 64 ? 64 : parts);
}
static size_t stats_bytes(long long rows) { return align256((size_t)2 * rows * sizeof(float)); }
static size_t range_bytes(long long batch, int kv_heads, int parts) {
  return align256((size_t)2 * batch * kv_heads * parts * sizeof(float));
}
static size_t gradient_bytes(long long batch, long long sq, long long sk, int heads, int kv_heads, int dim, int dtype) {
  const size_t es = dtype_size(dtype);
  const GradPlan k = plan_dkv(batch, sq, sk, heads, kv_heads, dim, es), q = plan_dq(batch, sq, sk, heads, es);
  const size_t kb = k.splits > 1 ? (size_t)2 * k.splits * batch * sk * kv_heads * dim * sizeof(float) : 0;
  const size_t qb = q.splits > 1 ? (size_t)q.splits * batch * sq * heads * dim * sizeof(float) : 0;
  const size_t range = dtype == MIA_F16 ? range_bytes(batch, kv_heads, range_parts(batch, sq, sk, heads, kv_heads)) : 0;
  return stats_bytes(batch * heads * sq) + range + (kb > qb ? kb : qb);
}

template <class T>
struct Ops {
  static int forward(Args a, hipStream_t s);
  static int backward(Args a, float* stats, void* dq, void* dk, void* dv, hipStream_t s);
};
#ifdef MIA_ATTENTION_TYPE
// 16-byte pieces are aligned, a tile's rows lie within 32 bits of offset
static bool pieces_ok(const View& v, size_t es) {
  const long long n = (long long)(16 / es);
  return aligned16(v.p) && v.b % n == 0 && v.s % n == 0 && v.h % n == 0 && v.s * (long long)es < (1LL << 25);
}
#define MIA_ATT_ONE(grid, kernel, ...) \
  hipLaunchKernelGGL((kernel<T, __VA_ARGS__>), dim3((unsigned)(grid)), dim3(256), 0, s, a)
#define MIA_ATT_LAUNCH(grid, kernel, ot, ...)                                                  \
  do {                                                                                         \
    if (a.dim <= 32) MIA_ATT_ONE(grid, kernel, 32, ot, decltype(dma)::value __VA_ARGS__);      \
    else if (a.dim <= 64) MIA_ATT_ONE(grid, kernel, 64, ot, decltype(dma)::value __VA_ARGS__); \
    else if (a.dim <= 96) MIA_ATT_ONE(grid, kernel, 96, ot, decltype(dma)::value __VA_ARGS__); \
    else MIA_ATT_ONE(grid, kernel, 128, ot, decltype(dma)::value __VA_ARGS__);                 \
  } while (0)
#define MIA_ATT_COMMA ,
// forward and dq: one block of queries a wave with both parts of p or ds, or without
#define MIA_ATT_LAUNCH_QUERIES(grid, kernel, blocks)                                                     \
  do {                                                                                                   \
    constexpr bool rounds = sizeof(T) == 2; /* (float: nothing is rounded) */                            \
    if (blocks == 2) MIA_ATT_LAUNCH(grid, kernel, 2, MIA_ATT_COMMA false);                               \
    else if (rounds && a.sq <= kFewQueries) MIA_ATT_LAUNCH(grid, kernel, 1, MIA_ATT_COMMA rounds);       \
    else MIA_ATT_LAUNCH(grid, kernel, 1, MIA_ATT_COMMA false);                                           \
  } while (0)

template <class F>
static void with_dma(bool dma, F f) {
  if (dma) f(std::true_type());
  else f(std::false_type());
}

template <class T>
int Ops<T>::forward(Args a, hipStream_t s) {
  const Plan pl = plan_forward(a.batch, a.sq, a.sk, a.heads, a.kv_heads);
  a.pack = pl.pack, a.own_tiles = pl.own_tiles, a.splits = pl.splits, a.keys_per_split = pl.keys_per_split;
  const long long grid = order_grid((long long)a.batch * (a.heads / a.pack), (long long)a.own_tiles * a.splits);
  const int rc = check_grid(grid);
  if (rc != MIA_OK) return rc;
  const bool dma = a.dim % (16 / (int)sizeof(T)) == 0 && pieces_ok(a.k, sizeof(T)) && pieces_ok(a.v, sizeof(T));
  with_dma(dma, [&](auto dma) { 
    MIA_ATT_LAUNCH_QUERIES(grid, att_fwd_kernel, pl.own_blocks);
  });
  if (a.splits > 1) {
    const long long rows = (long long)a.batch * a.heads * a.sq;
    hipLaunchKernelGGL(att_join_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
  }
  return MIA_OK;
}
template <class T>
int Ops<T>::backward(Args a, float* stats, void* dq, void* dk, void* dv, hipStream_t s) {
  const long long rows = (long long)a.batch * a.heads * a.sq;
  const bool whole = a.dim % (16 / (int)sizeof(T)) == 0;
  const GradPlan of_dq = plan_dq(a.batch, a.sq, a.sk, a.heads, sizeof(T));
  const GradPlan of_dkv = plan_dkv(a.batch, a.sq, a.sk, a.heads, a.kv_heads, a.dim, sizeof(T));
  const long long dq_grid = order_grid((long long)a.batch * a.heads, (long long)of_dq.own_tiles * of_dq.splits);
  const long long dkv_grid = order_grid((long long)a.batch * a.kv_heads, (long long)of_dkv.own_tiles * of_dkv.splits);
  const int rc = check_grid(dq_grid > dkv_grid ? dq_grid : dkv_grid);
  if (rc != MIA_OK) return rc;
  a.stats = stats, a.pack = 1;
  a.partial = stats + stats_bytes(rows) / sizeof(float);
  if constexpr (std::is_same<T, _Float16>::value) {
    a.range = a.partial, a.range_parts = range_parts(a.batch, a.sq, a.sk, a.heads, a.kv_heads);
    a.partial += range_bytes(a.batch, a.kv_heads, a.range_parts) / sizeof(float);
    const long long range_grid = (long long)a.batch * a.kv_heads * a.range_parts;
    const int fits = check_grid(range_grid);
    if (fits != MIA_OK) return fits;
    hipLaunchKernelGGL(att_range_kernel<T>, dim3((unsigned)range_grid), dim3(256), 0, s, a);
  }
  auto add = [&](long long total, long long n, void* out0, void* out1) {
    const long long blocks = (total + 255) / 256;
    hipLaunchKernelGGL(att_add_kernel<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, a.partial,
                       total, a.splits, n, static_cast<T*>(out0), static_cast<T*>(out1));
  };
  if (rows) {
    a.own_tiles = of_dq.own_tiles, a.splits = of_dq.splits;
    a.o0 = dq, a.o1 = nullptr;
    with_dma(whole && pieces_ok(a.k, sizeof(T)) && pieces_ok(a.v, sizeof(T)), [&](auto dma) {
      MIA_ATT_LAUNCH_QUERIES(dq_grid, att_dq_kernel, of_dq.own_blocks);
    });
    if (a.splits > 1) add(rows * a.dim, rows * a.dim, dq, nullptr);
  }
  if (a.sk) {
    a.own_tiles = of_dkv.own_tiles, a.splits = of_dkv.splits;
    a.o0 = dk, a.o1 = dv;
    with_dma(whole && pieces_ok(a.q, sizeof(T)) && pieces_ok(a.dout, sizeof(T)), [&](auto dma) {
      if (of_dkv.own_blocks == 2) {
        if constexpr (sizeof(T) == 2) {
          if (a.dim <= 32) MIA_ATT_ONE(dkv_grid, att_dkv_kernel, 32, 2, decltype(dma)::value);
          else MIA_ATT_ONE(dkv_grid, att_dkv_kernel, 64, 2, decltype(dma)::value);
        } else {
          MIA_ATT_ONE(dkv_grid, att_dkv_kernel, 32, 2, decltype(dma)::value);
        }
      } else {
        MIA_ATT_LAUNCH(dkv_grid, att_dkv_kernel, 1, );
      }
    });
    if (a.splits > 1) {
      const long long n = (long long)a.batch * a.sk * a.kv_heads * a.dim;
      add(2 * n, n, dk, dv);
    }
  }
  return MIA_OK;
}
template struct Ops<MIA_ATTENTION_TYPE>;
#endif
}  // namespace att
}  // namespace mia
