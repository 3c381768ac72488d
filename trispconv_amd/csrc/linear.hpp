// y = act(x W^T + bias) + residual for the rows of a feature tensor.
//
//   v[r][o] = sum_i x[r][i] w[o][i]  (f32 sums),  v += bias[o],
//   v = act(v),  v += residual[r][o],  one rounding to the rows' type.
#pragma once

#include "activation.hpp"
#include "sequence.hpp"

#include <algorithm>

namespace tsc {

struct LinearArgs {
  const void* x;
  int64_t x_stride;
  const void* w;
  int64_t w_stride;
  const void* bias;
  int bias_dtype;
  const void* residual;
  int64_t r_stride;
  int act;
  void* out;
  int64_t n;
  int c_in, c_out;
};

template <typename T>
int launch_linear(const LinearArgs& a, hipStream_t s);

namespace {

template <typename T>
__device__ __forceinline__ float activate_any(int act, float v) {
  switch (act) {
    case TSC_ACT_RELU: return activate<TSC_ACT_RELU, T>(v);
    case TSC_ACT_GELU: return activate<TSC_ACT_GELU, T>(v);
    case TSC_ACT_GELU_TANH: return activate<TSC_ACT_GELU_TANH, T>(v);
    case TSC_ACT_SILU: return activate<TSC_ACT_SILU, T>(v);
    default: return v;
  }
}

// ------------------------------------------------------------- few rows --
// Up to kFewRows rows: a wave per output column, the lanes share out the
// inputs.  Bound by reading W once.
constexpr int kFewRows = 8;

template <typename T, int ROWS>
__global__ void __launch_bounds__(256) linear_few_kernel(LinearArgs a) {
  constexpr int P = kPer16<T>;
  const int lane = threadIdx.x % kWave;
  const int o = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / kWave);
  if (o >= a.c_out) return;
  const T* x = static_cast<const T*>(a.x);
  const T* w = static_cast<const T*>(a.w) + o * a.w_stride;
  float acc[ROWS] = {};
  for (int i = lane * P; i < a.c_in; i += kWave * P) {
    const bool whole = i + P <= a.c_in;
    const int4v wv = whole ? load16_unaligned(w + i) : load16_partial(w + i, a.c_in - i);
    T we[P];
    __builtin_memcpy(we, &wv, 16);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (r >= a.n) break;
      const T* xr = x + r * a.x_stride + i;
      const int4v xv = whole ? load16_unaligned(xr) : load16_partial(xr, a.c_in - i);
      T xe[P];
      __builtin_memcpy(xe, &xv, 16);
#pragma unroll
      for (int e = 0; e < P; ++e) acc[r] = __builtin_fmaf(to_f32(xe[e]), to_f32(we[e]), acc[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) acc[r] += __shfl_xor(acc[r], d, kWave);
    if (lane == r && r < a.n) {
      float v = acc[r];
      if (a.bias) v += load_any(a.bias, a.bias_dtype, o);
      v = activate_any<T>(a.act, v);
      if (a.residual) v += to_f32(static_cast<const T*>(a.residual)[r * a.r_stride + o]);
      static_cast<T*>(a.out)[(int64_t)r * a.c_out + o] = from_f32<T>(v);
    }
  }
}

// Eight neighbouring values at any alignment, of which `have` exist.
template <typename T>
struct Eight {
  T e[8];
  __device__ __forceinline__ void load(const T* p, int have) {
    if (have >= 8) {
      __builtin_memcpy(e, p, sizeof e);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = i < have ? p[i] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void store(T* p, int have) const {
    if (have >= 8) {
      __builtin_memcpy(p, e, sizeof e);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < have) p[i] = e[i];
    }
  }
};

// Eight of the bias, as they lie in memory until they are used: asked for before
// the products, converted after them.
struct BiasEight {
  int4v raw[2] = {int4v(0), int4v(0)};
  template <typename B>
  __device__ __forceinline__ void load_as(const void* p, int64_t at, int have) {
    Eight<B> e;
    e.load(static_cast<const B*>(p) + at, have);
    __builtin_memcpy(raw, e.e, sizeof e.e);
  }
  __device__ __forceinline__ void load(const void* p, int dtype, int64_t at, int have) {
    if (!p || have <= 0) return;
    if (dtype == TSC_F32) load_as<float>(p, at, have);
    else if (dtype == TSC_F16) load_as<__half>(p, at, have);
    else load_as<__hip_bfloat16>(p, at, have);
  }
  template <typename B>
  __device__ __forceinline__ void values_as(float v[8]) const {
    Eight<B> e;
    __builtin_memcpy(e.e, raw, sizeof e.e);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e.e[i]);
  }
  __device__ __forceinline__ void values(const void* p, int dtype, float v[8]) {
    asm volatile("" : "+v"(raw[0]), "+v"(raw[1]));  // not before here
    if (!p) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    } else if (dtype == TSC_F32) {
      values_as<float>(v);
    } else if (dtype == TSC_F16) {
      values_as<__half>(v);
    } else {
      values_as<__hip_bfloat16>(v);
    }
  }
};

// ---------------------------------------------------------------- tiles --
// 16-byte chunk c of row r of an operand tile is stored in slot c ^ s(r), so
// that the 16 lanes LDS serves at a time (one chunk of 16 rows) find them in
// different 16-byte columns of its 256 bytes a cycle.
template <int RB>
__device__ __forceinline__ int tile_slot(int r, int c) {
  return RB == 64 ? c ^ ((r >> 2) & 3) : c ^ ((r >> 1) & 7);
}

// ROWS rows of RB bytes of an operand, one k tile after the other.
template <typename T, int ROWS, int RB, int THREADS, bool ALIGNED>
struct OperandStage {
  static constexpr int CH = RB / 16, ROUNDS = ROWS * CH / THREADS;
  static_assert(ROWS * CH % THREADS == 0 && THREADS % (16 * CH) == 0, "whole rounds of like lanes");
  const T* src;       // the lane's row in round 0, at its chunk
  uint32_t offset[ROUNDS];
  const T* base;
  int chunk, first_row, rows_left, wave;
  int64_t stride;
  int4v held[ALIGNED ? 1 : ROUNDS];

  // rows from `row` on of a tensor with `rows` of them; the ones past the
  // last are the last again (their products are never stored)
  __device__ __forceinline__ void begin(const T* p, int64_t stride_, int64_t row, int64_t rows) {
    const int lane = threadIdx.x % kWave;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    base = p + row * stride_;
    stride = stride_;
    rows_left = static_cast<int>(min(rows - row, (int64_t)ROWS));
    const int slot = wave * kWave + lane;
    first_row = slot / CH;
    chunk = tile_slot<RB>(first_row, slot % CH);
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i)
      offset[i] = static_cast<uint32_t>(min(first_row + i * (THREADS / CH), rows_left - 1) * stride * (int)sizeof(T)) +
                  chunk * 16;
  }
  // k tile kt (of `left` values from its first one on) into LDS (ALIGNED) or registers
  __device__ __forceinline__ void load(int kt, int left, char* tile) {
    const T* at = base + (int64_t)kt * (RB / (int)sizeof(T));
    if constexpr (ALIGNED) {
      const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds_address(tile) + wave * 1024);
      if (left >= RB / (int)sizeof(T)) {
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) load_to_lds(at, offset[i], m0 + i * THREADS * 16);
      } else {
        const bool in = chunk * kPer16<T> < left;
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
          load_to_lds(at, offset[i], m0 + i * THREADS * 16, in);
          if (!in) *reinterpret_cast<int4v*>(tile + (i * THREADS + threadIdx.x) * 16) = int4v(0);
        }
      }
    } else {
      const int have = left - chunk * kPer16<T>;
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        const T* p = reinterpret_cast<const T*>(reinterpret_cast<const char*>(at) + offset[i]);
        held[i] = have >= kPer16<T> ? load16_unaligned(p) : load16_partial(p, have);
      }
    }
  }
  __device__ __forceinline__ void store(char* tile) const {
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i)
        *reinterpret_cast<int4v*>(tile + (i * THREADS + threadIdx.x) * 16) = held[i];
    }
  }
};

// The workgroup's tile: false for the few workgroups that have none.  Tiles next
// to each other run on one XCD (workgroups go round the eight in turn), eight
// bands of rows at a time: they share W's tiles and x's bands in its L2.
__device__ __forceinline__ bool find_tile(int tiles_m, int tiles_n, int& tm, int& tn) {
  const int tiles = tiles_m * tiles_n, per = (tiles + 7) / 8;
  const int id = blockIdx.x % 8 * per + blockIdx.x / 8;
  if ((int)blockIdx.x / 8 >= per || id >= tiles) return false;
  constexpr int BANDS = 8;
  const int group = id / (BANDS * tiles_n), in_group = id - group * BANDS * tiles_n;
  const int bands = min(BANDS, tiles_m - group * BANDS);
  tn = in_group / bands;
  tm = group * BANDS + in_group - tn * bands;
  return true;
}

// Bytes of a row of 32-bit sums on their way out.
constexpr int leave_line(int columns) { return columns * 4 + 16; }

// A wave's sums leave: rows wave_row on, 32 MB of them, by NW columns, of which
// the lane's eight begin at column o.  Through `mine`, 32 lines of the wave's
// own LDS, so that rows are written (and the residual read) as whole 16-byte
// pieces side by side, with a lane's columns, and so its bias, the same in
// every row.
template <typename T, int NW, int NB, int MB>
__device__ __forceinline__ void leave(const LinearArgs& a, const f32x16 (&acc)[NB][MB], char* mine,
                                      int64_t wave_row, int o, BiasEight& bias_raw) {
  // 32 rows of the wave at a time through its own LDS
  constexpr int LINE = leave_line(NW), LANES = NW / 8, ROWS = kWave / LANES, ROUNDS = (32 + ROWS - 1) / ROWS;
  const int lane = threadIdx.x % kWave, half = lane / 32, col = lane % 32, have = a.c_out - o;
  float bias[8];
  bias_raw.values(a.bias, a.bias_dtype, bias);
  const uint32_t out_step = static_cast<uint32_t>(a.c_out) * sizeof(T);
  const uint32_t out_at = lane / LANES * out_step + o * (uint32_t)sizeof(T);
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int64_t first = wave_row + mb * 32;
    const int rows = static_cast<int>(min((int64_t)32, a.n - first));
    if (rows <= 0) break;
    // (lanes past a whole number of rows have none)
    const int mine_to = kWave % LANES == 0 || lane < ROWS * LANES ? rows : 0;
    Eight<T> res[ROUNDS];
    if (a.residual) {
      const T* p = static_cast<const T*>(a.residual) + first * a.r_stride + o;
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        const int r = i * ROWS + lane / LANES;
        if (r < mine_to) res[i].load(p + r * a.r_stride, have);
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 v = {acc[nb][mb][4 * i], acc[nb][mb][4 * i + 1], acc[nb][mb][4 * i + 2], acc[nb][mb][4 * i + 3]};
        *reinterpret_cast<f32x4*>(mine + col * LINE + (nb * 32 + 8 * i + 4 * half) * 4) = v;
      }
    __builtin_amdgcn_wave_barrier();
    char* out = static_cast<char*>(a.out) + first * a.c_out * (int64_t)sizeof(T);
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const int r = i * ROWS + lane / LANES;
      float v[8];
      __builtin_memcpy(v, mine + (kWave % LANES ? min(r, 31) : r) * LINE + lane % LANES * 32, 32);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += bias[e];
      switch (a.act) {
        case TSC_ACT_RELU: for (float& e : v) e = activate<TSC_ACT_RELU, T>(e); break;
        case TSC_ACT_GELU: for (float& e : v) e = activate<TSC_ACT_GELU, T>(e); break;
        case TSC_ACT_GELU_TANH: for (float& e : v) e = activate<TSC_ACT_GELU_TANH, T>(e); break;
        case TSC_ACT_SILU: for (float& e : v) e = activate<TSC_ACT_SILU, T>(e); break;
        default: break;
      }
      if (a.residual) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += to_f32(res[i].e[e]);
      }
      Eight<T> y;
      round_to<T, 8>(v, y.e);
      if (r < mine_to) y.store(reinterpret_cast<T*>(out + (out_at + i * ROWS * out_step)), have);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// A tile of BM rows by BN columns, WM x WN waves, each MW x NW of it in 32x32
// blocks: columns of W as the rows of the product, rows of x as its columns.
// Operand tiles of RB bytes a row go round STAGES buffers of LDS through
// direct-to-LDS loads, one barrier a tile.
template <typename T, int BM, int BN, int WM, int WN, int RB, int STAGES, bool ALIGNED, int OCC>
__global__ void __launch_bounds__(kWave* WM* WN, OCC) linear_tile_kernel(LinearArgs a, int tiles_m, int tiles_n) {
  constexpr int THREADS = kWave * WM * WN, MW = BM / WM, NW = BN / WN, MB = MW / 32, NB = NW / 32;
  constexpr int STAGE = (BM + BN) * RB, KT = RB / (int)sizeof(T), STEPS = RB / 32;
  constexpr int LOADS = (BM + BN) * RB / 16 / THREADS;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x % kWave, half = lane / 32, col = lane % 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);

  int tm, tn;
  if (!find_tile(tiles_m, tiles_n, tm, tn)) return;
  const int64_t row0 = (int64_t)tm * BM;
  const int col0 = tn * BN;

  OperandStage<T, BM, RB, THREADS, ALIGNED> xs;
  OperandStage<T, BN, RB, THREADS, ALIGNED> ws;
  xs.begin(static_cast<const T*>(a.x), a.x_stride, row0, a.n);
  ws.begin(static_cast<const T*>(a.w), a.w_stride, col0, a.c_out);
  auto load = [&](int kt) {
    char* tile = lds + kt % STAGES * STAGE;
    xs.load(kt, a.c_in - kt * KT, tile);
    ws.load(kt, a.c_in - kt * KT, tile + BM * RB);
  };
  auto store = [&](int kt) {
    char* tile = lds + kt % STAGES * STAGE;
    xs.store(tile);
    ws.store(tile + BM * RB);
  };

  constexpr int LINE = leave_line(NW), LANES = NW / 8;
  const int o = col0 + wave % WN * NW + lane % LANES * 8;
  BiasEight bias;  // of the lane's eight columns

  f32x16 acc[NB][MB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) acc[nb][mb] = f32x16(0.f);

  const int kts = (a.c_in + KT - 1) / KT;
  const int mrow = wave / WN * MW + col, nrow = wave % WN * NW + col;
  for (int kt = 0; kt < STAGES - 1 && kt < kts; ++kt) {
    load(kt);
    if (!ALIGNED) store(kt);
  }
  bias.load(a.bias, a.bias_dtype, o, a.c_out - o);
  for (int kt = 0; kt < kts; ++kt) {
    if constexpr (ALIGNED) {
      // loads finish in order: with STAGES - 2 later tiles of LOADS each in
      // flight, this one is there; near the end (where a partial tile may be
      // fewer loads) wait for all
      if (kt + STAGES - 1 < kts) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((STAGES - 2) * LOADS) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    } else {
      __syncthreads();
    }
    const bool more = kt + STAGES - 1 < kts;
    if (more) load(kt + STAGES - 1);
    const char* xt = lds + kt % STAGES * STAGE;
    const char* wt = xt + BM * RB;
    // The reads of a step between the matrix instructions of the one before,
    // for tiles of four steps (us, both orders in turn, bf16: 10000 x 2048 ->
    // 2048 86 against 91, 16000 x 1024 -> 1024 42.1 against 43.1, 65536 x 1024
    // -> 4096 with SiLU 608 against 621; with the two steps of 64-byte rows nothing, or
    // 1% more at 100000 x 512 -> 384)
    if constexpr (RB == 128) __builtin_amdgcn_iglp_opt(0);
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      int4v xf[MB], wf[NB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
        xf[mb] = *reinterpret_cast<const int4v*>(xt + (mrow + mb * 32) * RB + tile_slot<RB>(mrow, 2 * st + half) * 16);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        wf[nb] = *reinterpret_cast<const int4v*>(wt + (nrow + nb * 32) * RB + tile_slot<RB>(nrow, 2 * st + half) * 16);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[nb][mb] = mma32<T>(wf[nb], xf[mb], acc[nb][mb]);
    }
    if (!ALIGNED && more) store(kt + STAGES - 1);
  }
  __syncthreads();

  leave<T, NW>(a, acc, lds + wave * 32 * LINE, row0 + wave / WN * MW, o, bias);
}

template <typename T, int BM, int BN, int WM, int WN, int RB, int STAGES, bool ALIGNED, int OCC>
int launch_tile(const LinearArgs& a, hipStream_t s) {
  constexpr int main_bytes = STAGES * (BM + BN) * RB, out_bytes = WM * WN * 32 * (BN / WN * 4 + 16);
  constexpr int bytes = main_bytes > out_bytes ? main_bytes : out_bytes;
  auto kernel = &linear_tile_kernel<T, BM, BN, WM, WN, RB, STAGES, ALIGNED, OCC>;
  if (bytes > 65536)
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes)) return rc;
  const int64_t tm = ceil_div(a.n, BM), tn = ceil_div(a.c_out, BN), blocks = align_up(tm * tn, 8);
  TSC_REQUIRE(blocks * kWave * WM * WN < (1ll << 32), "linear_act: too many tiles");
  kernel<<<static_cast<unsigned>(blocks), kWave * WM * WN, bytes, s>>>(a, static_cast<int>(tm), static_cast<int>(tn));
  TSC_LAUNCH_CHECK("linear_act");
  return 0;
}

// ------------------------------------------------------ f32 on bf16 units --
// An f32 value of 2^-110 or more is the sum of three bf16 values exactly (8 bits
// each of its 24; subnormal ones, which the unit keeps, end at 2^-133):
// hi + mid + lo, mid within 2^-8 and lo within 2^-16 of it.  Of the nine
// products of two such sums the three of 2^-24 and less are left out (together
// at most 2^-23 of the whole, an f32 rounding or two), and six bf16 matrix
// instructions take the place of eight f32 ones that each last twice as long.
struct Split8 {
  int4v hi, mid, lo;
};

__device__ __forceinline__ Split8 split8(const float v[8]) {
  Split8 s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = v[2 * i], y = v[2 * i + 1];
    auto part = [&] {  // both rounded to bf16 and taken off
      const int p = pack2<__hip_bfloat16>(x, y);
      x -= __builtin_bit_cast(float, p << 16);
      y -= __builtin_bit_cast(float, p & 0xffff0000);
      return p;
    };
    s.hi[i] = part();
    s.mid[i] = part();
    s.lo[i] = pack2<__hip_bfloat16>(x, y);
  }
  return s;
}

// c += a b, both in three parts, the small products first.
__device__ __forceinline__ f32x16 mma32_split(const int4v a[3], const int4v b[3], f32x16 c) {
  using B = __hip_bfloat16;
  c = mma32<B>(a[2], b[0], c);
  c = mma32<B>(a[0], b[2], c);
  c = mma32<B>(a[1], b[1], c);
  c = mma32<B>(a[1], b[0], c);
  c = mma32<B>(a[0], b[1], c);
  return mma32<B>(a[0], b[0], c);
}

// Sums that the split cannot be trusted with are computed again on the f32 unit, a
// block of 32 x 32 at a time; which they are goes by a sum's own row and column,
// so that no other sum changes and the tile does not matter.
//   * Not finite (an infinity has no parts, and 0 times it would be NaN), or under
//     2^-64 without being zero (products of small parts are lost).
//   * A value below 2^-110 leaves up to 2^-134, times the other operand.  Where a
//     row of x has such values, that adds up to at most c_in max|w| 2^-134 over
//     the column's weights w, and likewise for a row of W: sums below 2^28 times
//     that, zeros as well.
// Whether a tile has such a value, and its largest, is known from the split's
// registers (2 operations a value: 20,000 x 1024 -> 1024 with GELU 244 us, without
// 235; 60,000 x 768 -> 192 131 against 125).  The ranges of its rows are read only
// where one of its sums is below what the tile's largest value could cost (a value of
// 1e-36 in every row: the same times; with the ranges read for all tiles 1540 and
// 1030).
__device__ __forceinline__ bool doubtful(float v) {
  const float m = __builtin_fabsf(v);
  return !(m >= 0x1p-64f && m < __builtin_inff()) && v != 0.f;
}

// A row's values: the largest, and whether one other than zero is below 2^-110.
struct RowRange {
  float most;
  uint32_t small;
};
// A value's magnitude as a number that orders them, zero last: the bits without
// the sign, shifted left, minus one.
__device__ __forceinline__ uint32_t place(float v) { return (__builtin_bit_cast(uint32_t, v) << 1) - 1u; }
constexpr uint32_t kSplitHolds = ((127u - 110u) << 24) - 1u;  // 2^-110's

// ROWS rows of 32 values of an operand: from memory to registers, and from
// there, split, to LDS (three planes of 64 bytes a row).
template <int ROWS, int THREADS>
struct SplitStage {
  static constexpr int ROUNDS = ROWS * 4 / THREADS, PLANE = ROWS * 64;
  static_assert(ROWS * 4 % THREADS == 0, "whole rounds");
  const char* base;
  uint32_t offset[ROUNDS];
  float held[ROUNDS][8];
  __device__ __forceinline__ void begin(const float* p, int64_t stride, int64_t row, int64_t rows) {
    base = reinterpret_cast<const char*>(p + row * stride);
    const int last = static_cast<int>(min(rows - row, (int64_t)ROWS)) - 1;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const int r = (i * THREADS + threadIdx.x) / 4;
      offset[i] = static_cast<uint32_t>(min(r, last) * stride * 4) + threadIdx.x % 4 * 32;
    }
  }
  __device__ __forceinline__ void load(int kt, int left) {
    const int have = left - (int)threadIdx.x % 4 * 8;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const float* p = reinterpret_cast<const float*>(base + kt * 128ll + offset[i]);
      if (have >= 8) {
        __builtin_memcpy(held[i], p, 32);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) held[i][e] = e < have ? p[e] : 0.f;
      }
    }
  }
  // least, most: the smallest place() and the largest magnitude so far
  __device__ __forceinline__ void store(char* tile, uint32_t& least, float& most) const {
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        least = min(least, place(held[i][e]));
        most = fmaxf(most, __builtin_fabsf(held[i][e]));
      }
      const int r = (i * THREADS + threadIdx.x) / 4;
      char* at = tile + r * 64 + tile_slot<64>(r, threadIdx.x % 4) * 16;
      const Split8 s = split8(held[i]);
      *reinterpret_cast<int4v*>(at) = s.hi;
      *reinterpret_cast<int4v*>(at + PLANE) = s.mid;
      *reinterpret_cast<int4v*>(at + 2 * PLANE) = s.lo;
    }
  }
};

// LDS for the parts of two operand tiles, and for the sums on their way out.
constexpr int split_pool_bytes(int bm, int bn, int wm, int wn) {
  const int parts = 3 * (bm + bn) * 64, out = wm * wn * 32 * leave_line(bn / wn);
  return parts > out ? parts : out;
}

// Tiles as in linear_tile_kernel, for f32 tensors: split on the way into LDS,
// with the next k tile's values on their way to registers meanwhile.
template <int BM, int BN, int WM, int WN, int OCC>
__global__ void __launch_bounds__(kWave* WM* WN, OCC) linear_split_kernel(LinearArgs a, int tiles_m, int tiles_n) {
  constexpr int THREADS = kWave * WM * WN, MW = BM / WM, NW = BN / WN, MB = MW / 32, NB = NW / 32;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x % kWave, half = lane / 32, col = lane % 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int tm, tn;
  if (!find_tile(tiles_m, tiles_n, tm, tn)) return;
  const int64_t row0 = (int64_t)tm * BM;
  const int col0 = tn * BN;
  SplitStage<BM, THREADS> xs;
  SplitStage<BN, THREADS> ws;
  xs.begin(static_cast<const float*>(a.x), a.x_stride, row0, a.n);
  ws.begin(static_cast<const float*>(a.w), a.w_stride, col0, a.c_out);
  constexpr int LINE = leave_line(NW), LANES = NW / 8;
  const int o = col0 + wave % WN * NW + lane % LANES * 8;
  BiasEight bias;  // of the lane's eight columns

  f32x16 acc[NB][MB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) acc[nb][mb] = f32x16(0.f);
  const int kts = (a.c_in + 31) / 32;
  const int mrow = wave / WN * MW + col, nrow = wave % WN * NW + col;
  const char *xt = lds, *wt = lds + 3 * BM * 64;
  uint32_t least = 0xffffffffu;
  float most = 0.f;
  if (kts > 0) {
    xs.load(0, a.c_in);
    ws.load(0, a.c_in);
  }
  bias.load(a.bias, a.bias_dtype, o, a.c_out - o);
  for (int kt = 0; kt < kts; ++kt) {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    xs.store(lds, least, most);
    ws.store(lds + 3 * BM * 64, least, most);
    asm volatile("" : "+v"(least), "+v"(most));  // before the next values take registers
    if (kt + 1 < kts) {
      xs.load(kt + 1, a.c_in - (kt + 1) * 32);
      ws.load(kt + 1, a.c_in - (kt + 1) * 32);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      int4v xf[MB][3], wf[NB][3];
#pragma unroll
      for (int p = 0; p < 3; ++p) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
          xf[mb][p] = *reinterpret_cast<const int4v*>(xt + p * BM * 64 + (mrow + mb * 32) * 64 +
                                                      tile_slot<64>(mrow, 2 * st + half) * 16);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          wf[nb][p] = *reinterpret_cast<const int4v*>(wt + p * BN * 64 + (nrow + nb * 32) * 64 +
                                                      tile_slot<64>(nrow, 2 * st + half) * 16);
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[nb][mb] = mma32_split(wf[nb], xf[mb], acc[nb][mb]);
    }
  }
  RowRange* ranges = reinterpret_cast<RowRange*>(lds + split_pool_bytes(BM, BN, WM, WN));
  const float weight = a.c_in * 0x1p-106f;
  bool small = __syncthreads_or(least < kSplitHolds);
  if (small) {  // does a sum come near what any row or column of the tile may lose?
#pragma unroll
    for (int x = 1; x < kWave; x <<= 1) most = fmaxf(most, __shfl_xor(most, x, kWave));
    if (lane == 0) ranges[wave].most = most;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < WM * WN; ++x) most = fmaxf(most, ranges[x].most);
    bool near = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 16; ++i) near |= __builtin_fabsf(acc[nb][mb][i]) < 2.f * most * weight;
    small = __syncthreads_or(near);
  }
  if (small) {  // the ranges of the tile's rows, read once more: eight lanes a row
    static_assert((BM + BN) % (THREADS / 8) == 0, "whole rounds");
#pragma unroll 2
    for (int r = threadIdx.x / 8; r < BM + BN; r += THREADS / 8) {
      const float* p = r < BM ? static_cast<const float*>(a.x) + min(row0 + r, a.n - 1) * a.x_stride
                              : static_cast<const float*>(a.w) + min(col0 + r - BM, a.c_out - 1) * a.w_stride;
      uint32_t first = 0xffffffffu;
      float top = 0.f;
#pragma unroll 4
      for (int k = lane % 8; k < a.c_in; k += 8) {
        first = min(first, place(p[k]));
        top = fmaxf(top, __builtin_fabsf(p[k]));
      }
#pragma unroll
      for (int x = 1; x < 8; x <<= 1) {
        first = min(first, static_cast<uint32_t>(__shfl_xor(static_cast<int>(first), x, kWave)));
        top = fmaxf(top, __shfl_xor(top, x, kWave));
      }
      if (lane % 8 == 0) ranges[r] = RowRange{top, first < kSplitHolds};
    }
    __syncthreads();
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      uint32_t redo = 0;  // bit i: sum i is computed again
#pragma unroll
      for (int i = 0; i < 16; ++i) redo |= (doubtful(acc[nb][mb][i]) ? 1u : 0u) << i;
      if (small) {
        const RowRange xr = ranges[mrow + mb * 32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const RowRange wr = ranges[BM + wave % WN * NW + nb * 32 + 8 * (i / 4) + 4 * half + i % 4];
          const float loss = (xr.small ? wr.most : 0.f) + (wr.small ? xr.most : 0.f);
          redo |= (__builtin_fabsf(acc[nb][mb][i]) < loss * weight ? 1u : 0u) << i;
        }
      }
      if (!__any(redo)) continue;
      const float* x = static_cast<const float*>(a.x) +
                       min(row0 + wave / WN * MW + mb * 32 + col, a.n - 1) * a.x_stride;
      const float* w = static_cast<const float*>(a.w) +
                       min(col0 + wave % WN * NW + nb * 32 + col, a.c_out - 1) * a.w_stride;
      f32x16 sum = f32x16(0.f);
#pragma unroll 4
      for (int k = half; k < a.c_in + half; k += 2) {
        const bool in = k < a.c_in;
        sum = __builtin_amdgcn_mfma_f32_32x32x2f32(in ? w[k] : 0.f, in ? x[k] : 0.f, sum, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[nb][mb][i] = redo >> i & 1u ? sum[i] : acc[nb][mb][i];
    }
  leave<float, NW>(a, acc, lds + wave * 32 * LINE, row0 + wave / WN * MW, o, bias);
}

template <int BM, int BN, int WM, int WN, int OCC>
int launch_split(const LinearArgs& a, hipStream_t s) {
  constexpr int bytes = split_pool_bytes(BM, BN, WM, WN) + (BM + BN) * (int)sizeof(RowRange);
  auto kernel = &linear_split_kernel<BM, BN, WM, WN, OCC>;
  if (bytes > 65536)
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes)) return rc;
  const int64_t tm = ceil_div(a.n, BM), tn = ceil_div(a.c_out, BN), blocks = align_up(tm * tn, 8);
  TSC_REQUIRE(blocks * kWave * WM * WN < (1ll << 32), "linear_act: too many tiles");
  kernel<<<static_cast<unsigned>(blocks), kWave * WM * WN, bytes, s>>>(a, static_cast<int>(tm), static_cast<int>(tn));
  TSC_LAUNCH_CHECK("linear_act_split");
  return 0;
}

// ------------------------------------------------------------- some rows --
// Tiles of 32 x 32 for calls whose larger tiles would leave most CUs idle: the
// eight waves of a workgroup share out the inputs (wave w takes steps w, w + 8,
// ...), read their operands straight into registers, and their sums meet in
// LDS, always in the same order.  Bound by the latency of a few dependent
// reads.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(512, 2) linear_rows_kernel(LinearArgs a) {
  constexpr int P = kPer16<T>, STEP = 2 * P;
  __shared__ __align__(16) float sums[8][32][36];  // [wave][row][column]
  const int lane = threadIdx.x % kWave, half = lane / 32, col = lane % 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t row0 = blockIdx.y * 32ll;
  const int col0 = blockIdx.x * 32;
  const T* x = static_cast<const T*>(a.x) + min(row0 + col, a.n - 1) * a.x_stride;
  const T* w = static_cast<const T*>(a.w) + min(col0 + col, a.c_out - 1) * a.w_stride;
  f32x16 acc = f32x16(0.f);
  const int whole = a.c_in / STEP;  // steps that end within the inputs
#pragma unroll 4
  for (int st = wave; st < whole; st += 8) {
    const int i = st * STEP + half * P;
    int4v wf, xf;
    if constexpr (ALIGNED) {
      wf = *reinterpret_cast<const int4v*>(w + i);
      xf = *reinterpret_cast<const int4v*>(x + i);
    } else {
      wf = load16_unaligned(w + i);
      xf = load16_unaligned(x + i);
    }
    acc = mma32<T>(wf, xf, acc);
  }
  if (whole % 8 == wave && whole * STEP < a.c_in) {
    const int i = whole * STEP + half * P, have = max(0, min(P, a.c_in - i));
    acc = mma32<T>(load16_partial(w + i, have), load16_partial(x + i, have), acc);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 v = {acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]};
    *reinterpret_cast<f32x4*>(&sums[wave][col][8 * i + 4 * half]) = v;
  }
  __syncthreads();
  const int r = threadIdx.x / 16, c = threadIdx.x % 16 * 2;
  const int64_t row = row0 + r;
  if (row >= a.n) return;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int o = col0 + c + e;
    if (o >= a.c_out) return;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += sums[k][r][c + e];
    if (a.bias) v += load_any(a.bias, a.bias_dtype, o);
    v = activate_any<T>(a.act, v);
    if (a.residual) v += to_f32(static_cast<const T*>(a.residual)[row * a.r_stride + o]);
    static_cast<T*>(a.out)[row * a.c_out + o] = from_f32<T>(v);
  }
}

template <typename T, bool ALIGNED>
int launch_rows(const LinearArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(ceil_div(a.c_out, 32)), static_cast<unsigned>(ceil_div(a.n, 32)));
  linear_rows_kernel<T, ALIGNED><<<grid, 512, 0, s>>>(a);
  TSC_LAUNCH_CHECK("linear_act_rows");
  return 0;
}

template <typename T, int ROWS>
int launch_few(const LinearArgs& a, hipStream_t s) {
  linear_few_kernel<T, ROWS><<<static_cast<unsigned>(ceil_div(a.c_out, 4)), 256, 0, s>>>(a);
  TSC_LAUNCH_CHECK("linear_act_few");
  return 0;
}

inline bool half_empty(int columns) { return (columns - 1) % 128 < 64; }

template <typename T, bool ALIGNED>
int launch_sized(const LinearArgs& a, hipStream_t s) {
  auto tiles = [&](int rows, int columns) { return ceil_div(a.n, rows) * ceil_div(a.c_out, columns); };
  // Tiles of 256 rows read least per product, but one workgroup fills a CU: the
  // last round of the 256 CUs takes as long as the others, with nothing beside
  // it while its sums leave.  Smaller tiles follow each other, at 1.3 times the
  // time a product (65536 x 1024 -> 4096 f16 610 us, in 128 x 128 tiles 800).
  // So the products of a CU decide, for sums long enough to be most of the time
  // (f16, us, 256 x 256, 256 x 192, small: 60013 x 768 -> 192 37.1 31.7 46.5;
  // 60000 x 2048 -> 256 84.5 122 109; 10000 x 2048 -> 2048 123 102 122;
  // 16000 x 1024 -> 1024 42.8 61.5 51.2; 100000 x 512 -> 384 99 86 73)
  if (a.c_in >= 512) {
    const auto rounds = [&](int columns) { return ceil_div(tiles(256, columns), 256) * 256 * columns; };
    const int64_t small = a.n * align_up(a.c_out, 64) / 256 * 13 / 10;
    if (rounds(256) <= std::min(rounds(192), small)) return launch_tile<T, 256, 256, 2, 4, 128, 2, ALIGNED, 2>(a, s);
    if (rounds(192) < small) return launch_tile<T, 256, 192, 4, 2, 128, 2, ALIGNED, 2>(a, s);
  }
  if (tiles(128, 128) >= 256) {
    // 64 columns where tiles of 128 would leave half of the last one empty
    // (100000 x 64 -> 64 16.7 us, in 128 x 128 tiles 25.7)
    if (half_empty(a.c_out)) return launch_tile<T, 128, 64, 2, 2, 64, 2, ALIGNED, 2>(a, s);
    return launch_tile<T, 128, 128, 2, 2, 64, 2, ALIGNED, 2>(a, s);
  }
  return launch_tile<T, 64, 64, 2, 2, 128, 3, ALIGNED, 2>(a, s);
}

}  // namespace

template <typename T>
int launch_linear(const LinearArgs& a, hipStream_t s) {
  if (a.n <= 1) return launch_few<T, 1>(a, s);
  if (a.n <= kFewRows) return launch_few<T, kFewRows>(a, s);
  const int64_t e = kPer16<T>;
  // 16-byte pieces at 16-byte addresses, rows of a tile within 32-bit offsets
  const bool aligned = a.c_in % e == 0 && a.x_stride % e == 0 && a.w_stride % e == 0 &&
                       reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && reinterpret_cast<uintptr_t>(a.w) % 16 == 0;
  const bool near = std::max(a.x_stride, a.w_stride) < (1 << 21);
  TSC_REQUIRE(near, "linear_act: row strides over 2^21 elements are not supported");
  // Tiles of 64 x 64 on fewer than half the CUs (f32, whose waves wait longer
  // between barriers: up to 200): 16 x 2048 -> 4096 bf16 8.6 us, in tiles 13.3;
  // 100 x 1024 -> 4096 (128 tiles) 9.9 against 8.5, f32 20.4 against 27.4;
  // 1000 x 1024 -> 1024 (256 tiles) 17.9 against 9.0, f32 35.9 against 29.3
  if (ceil_div(a.n, 64) * ceil_div(a.c_out, 64) < (kIs16<T> ? 128 : 200))
    return aligned ? launch_rows<T, true>(a, s) : launch_rows<T, false>(a, s);
  if constexpr (!kIs16<T>) {
    // as for 16 bits (60000 x 768 -> 192: 128 x 64 129 us, 128 x 128 147)
    if (ceil_div(a.n, 128) * ceil_div(a.c_out, 128) < 256) return launch_split<64, 64, 2, 2, 3>(a, s);
    return half_empty(a.c_out) ? launch_split<128, 64, 2, 2, 3>(a, s) : launch_split<128, 128, 2, 2, 2>(a, s);
  } else {
    return aligned ? launch_sized<T, true>(a, s) : launch_sized<T, false>(a, s);
  }
}

}  // namespace tsc
