// Attention of packed sequences in a sliding window, with sinks.
//
// Sample b owns queries [oq[b], oq[b+1]) and keys [ok[b], ok[b+1]); its Lq
// queries are the last of its Lk positions: query i stands at p = i + Lk - Lq
// and sees key j when 0 <= j < Lk, j <= p + right, and j >= p - left or
// j < sinks.  Per head (G query heads share a key head)
//   o = sum_j e^(s_j) v_j / sum_j e^(s_j),  s_j = scale q.k_j  over the seen j,
// and 0 where there is none.  The seen keys are two ranges:
//   [lo, hi) with lo = max(0, p - left), hi = min(Lk, p + right + 1), and
//   [0, min(sinks, lo, hi)).
// One pass over the keys with a running reference score m and the sum l of the
// exponentials (f32): a new reference rescales what is there by e^(m_old - m).
#pragma once

#include "sequence.hpp"

#include <algorithm>
#include <cmath>

namespace tsc {

struct AttendArgs {
  const void* q;
  int64_t q_row, q_head;
  const void* k;
  int64_t k_row, k_head;
  const void* v;
  int64_t v_row, v_head;
  const int32_t* off_q;
  const int32_t* off_k;
  int samples;
  int64_t n_q, n_k;
  int q_heads, k_heads, dim;
  int left, right, sinks;  // left, right: kNoLimit where there is none
  float scale_log2;        // |scale| * log2(e), 1 for a scale of 0
  float q_sign;            // the scale's sign, 0 for a scale of 0
  void* out;
  float* part;             // when the keys are split: [split][n_q * q_heads][m, l], then
                           // [split][n_q * q_heads][dim] sums from part_values() on
  __host__ __device__ int64_t rows() const { return n_q * q_heads; }
  __host__ __device__ int64_t part_values(int splits) const { return (splits * rows() * 2 + 3) / 4 * 4; }
};

constexpr int kNoLimit = 0x7fffffff;

// How a call is cut up: the rows of a workgroup and the parts its keys are
// split into.
struct Cut {
  int wave_rows;  // rows of a workgroup of four waves in 128s, 0: one wave, 32 rows
  int64_t tiles;
  int splits;
};

// Whether a wave may take 64 rows (two blocks of 32): halves the reads of K and
// V from LDS, but leaves room for two waves a SIMD instead of four.
constexpr bool can_pair(int dp, int elem) { return elem == 2 && dp <= 64; }
// Keys of a tile in 32s: two, unless four tiles of it would not fit the LDS.
template <typename T>
constexpr int key_blocks(int dp) { return dp * (int)sizeof(T) <= 512 ? 2 : 1; }

// Tiles of K and V in LDS: the one in use and those on their way.  A wave that
// is a workgroup of its own asks for three tiles at once, which is most of a
// split walk; every tile then waits for all that is on the way, so that over a
// longer walk four buffers hide no more than two.
template <typename T>
constexpr int tile_buffers(int dp, int waves) { return waves == 1 && dp * (int)sizeof(T) <= 128 ? 4 : 2; }
// Waves a SIMD that the registers and the LDS leave room for.
template <typename T>
constexpr int waves_per_simd(int dp, int row_blocks, int waves) {
  return dp * (int)sizeof(T) <= 128 && waves > 1 ? 4 / row_blocks : dp * (int)sizeof(T) <= 256 ? 2 : 1;
}

inline int padded_dim(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : 256; }

// The call on tensors of type T, cut as c says.
template <typename T>
int launch_attend(const AttendArgs& a, const Cut& c, hipStream_t s);

namespace {

// [offsets[b], offsets[b+1]) cut to [0, n]: no value of the offsets leads out
// of the tensors.
__device__ __forceinline__ void sample_range(const int32_t* off, int b, int64_t n, int64_t& at,
                                             int& len) {
  const int64_t lo = min(max((int64_t)off[b], (int64_t)0), n);
  const int64_t hi = min(max((int64_t)off[b + 1], lo), n);
  at = lo;
  len = static_cast<int>(hi - lo);
}

// The query rows [first, last) from the first sample's to the last one's; the
// others belong to no sample, and their outputs are 0.
__device__ __forceinline__ void sample_rows(const AttendArgs& a, int64_t& first, int64_t& last) {
  first = min(max((int64_t)a.off_q[0], (int64_t)0), a.n_q);
  last = min(max((int64_t)a.off_q[a.samples], first), a.n_q);
}

// Zeros for the rows outside [first, last), shared out over the grid.
template <typename T>
__device__ __noinline__ void zero_outside(T* out, int64_t row, int64_t first, int64_t last, int64_t n) {
  const int64_t before = first * row, all = before + (n - last) * row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x)
    out[i < before ? i : i - before + last * row] = from_f32<T>(0.f);
}

// The seen keys of position p among lk: [lo, hi) and [0, sink).
__device__ __forceinline__ void seen_keys(int p, int lk, int left, int right, int sinks, int& lo,
                                          int& hi, int& sink) {
  const int64_t h = (int64_t)p + right + 1, l = (int64_t)p - left;
  hi = static_cast<int>(max((int64_t)0, min(h, (int64_t)lk)));
  lo = static_cast<int>(min((int64_t)lk, max(l, (int64_t)0)));
  sink = min(sinks, min(lo, hi));
}

// One query and head by one wave: a lane scores every 64th key, then the lanes
// share out the D values and add the 64 keys' values one by one.  Reads no
// key it does not see, and of those only [s0, s1) among the sinks and [w0,
// w1) of the window's tiles.  Any size, stride and alignment; q_s: D floats of LDS
// for this wave.  Returns the running maximum (in units of log2) and sum;
// lane l holds the sums of values l, l + 64, ...
template <typename T>
__device__ void attend_row(const AttendArgs& a, const T* q, const T* k, const T* v, int lo, int hi,
                           int sink, int s0, int s1, int w0, int w1, float* q_s, float& m_out,
                           float& l_out, float o[4]) {
  const int lane = threadIdx.x % kWave;
  __builtin_amdgcn_wave_barrier();
  for (int d = lane; d < a.dim; d += kWave) q_s[d] = a.q_sign * to_f32(q[d]);
  __builtin_amdgcn_wave_barrier();
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int u = 0; u < 4; ++u) o[u] = 0.f;
  // sinks of the sink tiles, sinks that lie among the window's tiles, window
  for (int part = 0; part < 3; ++part) {
    const int from = part == 0 ? s0 : part == 1 ? w0 : max(lo, w0);
    const int to = part == 0 ? min(sink, s1) : part == 1 ? min(sink, w1) : min(hi, w1);
    for (int j0 = from; j0 < to; j0 += kWave) {
      const int j = j0 + lane;
      float s = -__builtin_inff();
      if (j < to) {
        float dot = 0.f;
        for (int d = 0; d < a.dim; ++d) dot += q_s[d] * to_f32(k[j * a.k_row + d]);
        s = dot * a.scale_log2;
      }
      float top = s;
#pragma unroll
      for (int x = 1; x < kWave; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, kWave));
      const float m_new = fmaxf(m, top);
      const float base = m_new == -__builtin_inff() ? 0.f : m_new;
      const float fix = exp2f(m - base), p = j < to ? exp2f(s - base) : 0.f;
      l *= fix;
      m = m_new;
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] *= fix;
      const int cnt = min(kWave, to - j0);
      for (int x = 0; x < cnt; ++x) {
        const float px = __shfl(p, x, kWave);
        l += px;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int d = lane + u * kWave;
          if (d < a.dim) o[u] += px * to_f32(v[(j0 + x) * a.v_row + d]);
        }
      }
    }
  }
  m_out = m;
  l_out = l;
}

// What 16-byte slot chunk c of row r of an LDS tile is stored in, so that the
// reads below find their pieces in different columns of the 256 bytes that LDS
// serves a cycle.  RB: bytes of a row.
template <int RB>
__device__ __forceinline__ int k_slot(int r, int c) {  // 16 rows, the same chunk: 16 bytes a lane
  return RB % 256 == 0 ? c ^ (r & 15) : RB % 128 == 0 ? c ^ ((r >> 1) & 7) : c ^ ((r >> 2) & 3);
}
template <int RB>
__device__ __forceinline__ int v_slot(int r, int c) {  // 4 rows, four chunks each: 8 bytes a lane
  return RB % 256 == 0 ? c ^ (4 * (r & 3)) : RB % 128 == 0 ? c ^ (2 * (r & 3)) : c;
}

// Brings tiles of rows [j0, j0 + 32 KB) of one key head's K or V into LDS,
// chunk by chunk in the order of the slots.  Rows from `end` on are not used
// by anyone: they are row end - 1 again, so nothing past the sample is read.
// Values from dim on stay the zeros that clear() put there.
template <typename T, int DP, int KB, int WAVES, bool ALIGNED, bool IS_V>
struct Stager {
  static constexpr int RB = DP * sizeof(T), CH = RB / 16, CHUNKS = 32 * KB * CH;
  static constexpr int THREADS = kWave * WAVES, ROUNDS = CHUNKS / THREADS;
  static_assert(CHUNKS % THREADS == 0, "whole instructions");
  // the slots of a thread's rounds hold the same chunk of rows a constant apart
  static constexpr bool SAME = THREADS % (16 * CH) == 0;
  const T* src;
  int64_t stride;
  int dim, lane, wave;
  uint32_t offset[SAME ? 1 : ROUNDS];  // bytes from row j0 to the thread's chunks

  __device__ static int row(int slot) { return slot / CH; }
  __device__ static int chunk(int slot) {
    return IS_V && kIs16<T> ? v_slot<RB>(slot / CH, slot % CH)
           : IS_V           ? slot % CH
                            : k_slot<RB>(slot / CH, slot % CH);
  }
  __device__ int slot(int i) const { return i * THREADS + wave * kWave + lane; }

  __device__ __forceinline__ void begin(const T* src_, int64_t stride_, int dim_, int wave_) {
    src = src_, stride = stride_, dim = dim_, wave = wave_, lane = threadIdx.x % kWave;
#pragma unroll
    for (int i = 0; i < (SAME ? 1 : ROUNDS); ++i)
      offset[i] = static_cast<uint32_t>(row(slot(i)) * stride * sizeof(T)) + chunk(slot(i)) * 16;
  }
  __device__ void clear(char* tile) const {
    if (dim >= DP) return;
    for (int i = 0; i < ROUNDS; ++i)
      if (chunk(slot(i)) * kPer16<T> >= dim) *reinterpret_cast<int4v*>(tile + slot(i) * 16) = int4v(0);
  }
  __device__ __forceinline__ void load(char* tile, int j0, int end) const {
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_address(tile) + wave * 1024);
    if constexpr (ALIGNED) {
      const T* base = src + j0 * stride;
      if (j0 + 32 * KB <= end && dim >= DP) {
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
          if (SAME) load_to_lds(base + i * (THREADS / CH) * stride, offset[0], at + i * WAVES * 1024);
          else load_to_lds(base, offset[SAME ? 0 : i], at + i * WAVES * 1024);
        }
      } else {
#pragma unroll 2
        for (int i = 0; i < ROUNDS; ++i) {
          const int r = min(row(slot(i)), end - 1 - j0);
          load_to_lds(base, static_cast<uint32_t>(r * stride * sizeof(T)) + chunk(slot(i)) * 16,
                      at + i * WAVES * 1024, in(i));
        }
      }
    } else {
#pragma unroll 2
      for (int i = 0; i < ROUNDS; ++i) {
        const int d = chunk(slot(i)) * kPer16<T>;
        const T* p = src + min(j0 + row(slot(i)), end - 1) * stride + d;
        const int4v x = d + kPer16<T> <= dim ? load16_unaligned(p) : load16_partial(p, dim - d);
        *reinterpret_cast<int4v*>(tile + slot(i) * 16) = x;
      }
    }
  }
  __device__ __forceinline__ bool in(int i) const { return dim >= DP || chunk(slot(i)) * kPer16<T> < dim; }
};

__device__ __forceinline__ float max_halves(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// Non-finite values of a V tile: replaced by 0, their keys' bits set in the
// KB words of LDS at `bad`.  Every thread of the workgroup calls it.
template <typename T, int DP, int KB, int WAVES>
__device__ void find_bad(char* vt, uint32_t* bad) {
  constexpr int RB = DP * sizeof(T), CH = RB / 16, CHUNKS = 32 * KB * CH;
  if (threadIdx.x < KB) bad[threadIdx.x] = 0u;
  __syncthreads();
  for (int slot = threadIdx.x; slot < CHUNKS; slot += kWave * WAVES) {
    T* e = reinterpret_cast<T*>(vt + slot * 16);
    bool any = false;
    for (int i = 0; i < kPer16<T>; ++i) {
      const float x = to_f32(e[i]) * 0.f;
      if (x != x) {
        e[i] = from_f32<T>(0.f);
        any = true;
      }
    }
    if (any) atomicOr(&bad[slot / CH / 32], 1u << (slot / CH % 32));
  }
  __syncthreads();
}

// The sample and the tile within it of the x-th tile of all: sample b has
// ceil(Lq * group / rows) of them.  Every wave finds it for itself, 64 samples
// at a time, the keys' offsets on the way so that nothing waits for them
// later.  false: past the last.
__device__ __forceinline__ bool find_tile(const AttendArgs& a, int group, int rows, int x, int64_t& q0,
                                          int& lq, int64_t& k0, int& lk, int& tile) {
  const int lane = threadIdx.x % kWave;
  for (int b0 = 0; b0 < a.samples; b0 += kWave) {
    int64_t at = 0, at_k = 0;
    int len = 0, len_k = 0;
    if (b0 + lane < a.samples) {
      sample_range(a.off_q, b0 + lane, a.n_q, at, len);
      sample_range(a.off_k, b0 + lane, a.n_k, at_k, len_k);
    }
    const uint32_t tiles = static_cast<uint32_t>(((int64_t)len * group + rows - 1) / rows);
    const uint32_t inc = wave_inclusive(tiles);
    const uint64_t past = __ballot(inc > static_cast<uint32_t>(x));
    if (past) {
      const int at_lane = __builtin_ctzll(past);
      tile = x - __builtin_amdgcn_readlane(inc - tiles, at_lane);
      lq = __builtin_amdgcn_readlane(len, at_lane);
      q0 = __builtin_amdgcn_readlane(static_cast<int>(at), at_lane);
      k0 = __builtin_amdgcn_readlane(static_cast<int>(at_k), at_lane);
      lk = __builtin_amdgcn_readlane(len_k, at_lane);
      return true;
    }
    x -= __builtin_amdgcn_readlane(inc, kWave - 1);
  }
  return false;
}

// What a workgroup computes: rows [row0, ...) of the `rows` (token, head of
// the group) rows of a sample and key head, against key tiles [t0, t1) of
// those that it walks: [0, sink_end) in sink_tiles of them, then [start, end).
struct Walk {
  int64_t q0;  // the sample's first query row
  uint32_t row0, rows;
  int group, hk, lk, shift;  // shift: position of the sample's first query
  int sink_end, sink_tiles, start, end, t0, t1;
  int split, splits;
  // (the host keeps n_q * group within 32 bits)
  __device__ int token(uint32_t r) const { return static_cast<int>(min(r, rows - 1) / static_cast<uint32_t>(group)); }
};

// The weight of a key at its row's reference score (in log2), and what a lane's 16
// weights may sum to before the reference moves: 2^7 times as much.  f16 needs
// the place below, and its values are too small for an f32 sum to overflow.  bf16
// and f32 reach as far as the sums: their weights are at most 1, so that sums of
// large values overflow no earlier than with the largest score as the reference.
template <typename T> constexpr float kLift = std::is_same_v<T, __half> ? 8.f : -7.f;
template <typename T> constexpr float kMostWeight = std::is_same_v<T, __half> ? 32768.f : 1.f;
constexpr float kFar = 0x1p24f;  // exponents from here on have no fractions in f32

// Tiles of 32 RB WAVES rows (a row: one query of one head; the heads that
// share a key head side by side) against tiles of 32 KB keys.
//
// A wave holds 32 RB rows as the columns of the transposed scores S^T = K Q^T:
// a lane has 16 KB keys of one row per 32, so the row's maximum and sum are a
// lane's own values and one exchange with the other half, and e^S^T is, as it
// stands, the right operand of O^T = V^T e^S^T: the product's sum runs over
// keys in the order that S^T's registers have them, and V is read in the same
// order (ds_read_b64_tr_b16 transposes it on the way from LDS).  K and V tiles
// have BUFFERS buffers: direct-to-LDS loads of the next ones fly while these
// are used, one barrier a tile.
//
// A row's reference m is the largest score of its first 32 keys; a key of that
// score has weight 2^kLift.  m moves (with a rescale of what is there, and the
// weights made again) only when a lane's 16 weights sum to over kMostWeight, so
// that most keys need no maximum at all.  m is a score of the row, so its largest
// weight is at least 2^kLift.  For f16, whose numbers end at 2^15 and are
// normal from 2^-14 on, that keeps weights down to 2^-22 of it normal, for long rows
// where many such keys make up a share of the sum.
//
// 16-bit tensors have their weights rounded to 16 bits for the product with V:
// on the f32 unit, or split into parts, that product would take several times
// as long.  It adds up to half a unit in the last place of the type to each
// weight (errors against 64 bits 1.4 times those with f32 weights); scores,
// references and both sums stay f32.
//
// The exponents are s c - mc with mc = m c rounded: a row's weights have a factor in
// common that the division takes out again, unless the rounding is of whole
// exponents.  Rows whose reference was ever that far from 0 are done key by key.
//
// A key that a row does not see has weight 0, and 0 times an infinite or NaN
// value would be NaN.  When a row of the workgroup comes out not finite, the
// keys are walked once more with such values replaced by 0, which leaves the
// bits of every row that sees none of them as they would have been; rows that
// see one are then done key by key.
template <typename T, int DP, int RB, int KB, int WAVES, bool ALIGNED>
__device__ __forceinline__ void attend_walk(const AttendArgs& a, const Walk& w, const T* k, const T* v,
                                            char* lds) {
  constexpr int KT = 32 * KB, ROW_BYTES = DP * sizeof(T);
  constexpr int BUFFERS = tile_buffers<T>(DP, WAVES), TILE = KT * ROW_BYTES, STEPS = DP * (int)sizeof(T) / 32, DB = DP / 32;
  const int lane = threadIdx.x % kWave, half = lane / 32, col = lane % 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int lo_first, hi_first, lo_last, hi_last, none;
  const uint32_t wave_row = w.row0 + wave * 32 * RB;
  seen_keys(w.token(wave_row) + w.shift, w.lk, a.left, a.right, a.sinks, lo_first, hi_first, none);
  seen_keys(w.token(wave_row + 32 * RB - 1) + w.shift, w.lk, a.left, a.right, a.sinks, lo_last, hi_last, none);
  int lo[RB], hi[RB];
  int4v qf[RB][STEPS];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const uint32_t r = wave_row + rb * 32 + col;
    const int t = w.token(r), g = static_cast<int>(min(r, w.rows - 1) - static_cast<uint32_t>(t) * w.group);
    seen_keys(t + w.shift, w.lk, a.left, a.right, a.sinks, lo[rb], hi[rb], none);
    if (r >= w.rows) hi[rb] = 0;
    const T* q = static_cast<const T*>(a.q) + (w.q0 + t) * a.q_row + (w.hk * w.group + g) * a.q_head;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int d = (2 * st + half) * kPer16<T>;
      int4v x;
      if (d + kPer16<T> <= a.dim) x = load16_unaligned(q + d);
      else x = load16_partial(q + d, a.dim - d);
      // the scale's sign (0 for a scale of 0) goes into q, exactly
      if (a.q_sign != 1.f) {
        T e[kPer16<T>];
        __builtin_memcpy(e, &x, 16);
#pragma unroll
        for (int i = 0; i < kPer16<T>; ++i) e[i] = from_f32<T>(to_f32(e[i]) * a.q_sign);
        __builtin_memcpy(&x, e, 16);
      }
      qf[rb][st] = x;
    }
  }

  auto tile_at = [&](int t, int& j0, int& end) {
    if (t < w.sink_tiles) {
      j0 = t * KT;
      end = w.sink_end;
    } else {
      j0 = w.start + (t - w.sink_tiles) * KT;
      end = w.end;
    }
  };
  Stager<T, DP, KB, WAVES, ALIGNED, false> k_stage;
  Stager<T, DP, KB, WAVES, ALIGNED, true> v_stage;
  k_stage.begin(k, a.k_row, a.dim, wave);
  v_stage.begin(v, a.v_row, a.dim, wave);
  for (int x = 0; x < BUFFERS; ++x) {
    k_stage.clear(lds + x * 2 * TILE);
    v_stage.clear(lds + x * 2 * TILE + TILE);
  }
  auto stage = [&](int j0, int end, int buf) {
    k_stage.load(lds + buf * 2 * TILE, j0, end);
    v_stage.load(lds + buf * 2 * TILE + TILE, j0, end);
  };

  f32x16 o[RB][DB];
  float m[RB], mc[RB], l[RB][2];  // reference score, its exponent, two partial sums
  int hit = 0;    // bit rb: the row is done key by key
  int clean = 0;  // the walk that replaces those values
  uint32_t* bad = reinterpret_cast<uint32_t*>(lds + 2 * BUFFERS * TILE + WAVES * DP * 4);
  const float c = a.scale_log2;
  // 32 keys from row kb * 32 of a tile; whole: every row of the wave sees all
  auto key_step = [&](bool whole, const char* kt, const char* vt, int kb, int j0, int end) {
    f32x16 s[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) s[rb] = f32x16(0.f);
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int4v x = *reinterpret_cast<const int4v*>(kt + (kb * 32 + col) * ROW_BYTES +
                                                      k_slot<ROW_BYTES>(col, 2 * st + half) * 16);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) s[rb] = mma32<T>(x, qf[rb][st], s[rb]);
    }
    if (!whole && j0 + kb * 32 < a.sinks) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = j0 + kb * 32 + 8 * (i / 4) + 4 * half + i % 4;
          const bool see = j < min(end, hi[rb]) && (j >= lo[rb] || j < a.sinks);
          s[rb][i] = see ? s[rb][i] : -__builtin_inff();
        }
    } else if (!whole) {
      // no sinks here: one comparison for both ends
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const uint32_t from = j0 + kb * 32 + 4 * half - lo[rb], span = max(0, min(end, hi[rb]) - lo[rb]);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[rb][i] = from + (8 * (i / 4) + i % 4) < span ? s[rb][i] : -__builtin_inff();
      }
    }
    // weights e^S^T with the rows' references, and their sums
    int p16[RB][8];     // 16 bits: two keys a register
    float p32[RB][16];  // f32
    float sum[RB][2];
    auto weights = [&] {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        sum[rb][0] = sum[rb][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][2 * i], c, -mc[rb]));
          const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][2 * i + 1], c, -mc[rb]));
          sum[rb][0] += x;
          sum[rb][1] += y;
          if constexpr (kIs16<T>) {
            p16[rb][i] = pack2<T>(x, y);
          } else {
            p32[rb][2 * i] = x;
            p32[rb][2 * i + 1] = y;
          }
        }
      }
    };
    weights();
    bool over = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) over |= m[rb] == -__builtin_inff() || sum[rb][0] + sum[rb][1] > kMostWeight<T>;
    if (__any(over)) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float top = fmaxf(s[rb][0], s[rb][1]);
#pragma unroll
        for (int i = 2; i < 16; i += 2) top = fmaxf(fmaxf(top, s[rb][i]), s[rb][i + 1]);
        const float m_new = fmaxf(m[rb], max_halves(top));
        const float mc_new = m_new == -__builtin_inff() ? 0.f : m_new * c - kLift<T>;
        const float fix = m[rb] == -__builtin_inff() ? 0.f : exp2f(mc[rb] - mc_new);
        m[rb] = m_new;
        mc[rb] = mc_new;
        hit |= (__builtin_fabsf(mc_new) >= kFar) << rb;
        l[rb][0] *= fix;
        l[rb][1] *= fix;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[rb][db] *= fix;
      }
      weights();
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      l[rb][0] += sum[rb][0];
      l[rb][1] += sum[rb][1];
    }
    // O^T += V^T e^S^T.  16 bits: 16 keys a step, of which the halves take
    // keys 0-3, 8-11 and 4-7, 12-15.  f32: two keys a step, 4 apart.
    if constexpr (kIs16<T>) {
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          int4v x;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = 16 * st + 8 * h + 4 * half + (lane & 15) / 4;
            const int d = 32 * db + (lane & 16) + 4 * (lane & 3);
            const char* p = vt + (kb * 32 + r) * ROW_BYTES + v_slot<ROW_BYTES>(r, d / 8) * 16 + (d % 8) * 2;
            const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) short4v*)p);
            const int2v z = __builtin_bit_cast(int2v, y);
            x[2 * h] = z[0];
            x[2 * h + 1] = z[1];
          }
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            const int4v p = {p16[rb][4 * st], p16[rb][4 * st + 1], p16[rb][4 * st + 2], p16[rb][4 * st + 3]};
            o[rb][db] = mma32<T>(x, p, o[rb][db]);
          }
        }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const int r = kb * 32 + 8 * (i / 4) + 4 * half + i % 4;
          const float x = *reinterpret_cast<const float*>(vt + r * ROW_BYTES + (32 * db + col) * 4);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
            o[rb][db] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p32[rb][i], o[rb][db], 0, 0, 0);
        }
    }
  };

  for (;;) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      // (rows past the last need none: their scores are all -inf)
      m[rb] = wave_row + rb * 32 + col < w.rows ? -__builtin_inff() : 0.f;
      mc[rb] = l[rb][0] = l[rb][1] = 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[rb][db] = f32x16(0.f);
    }

    // tile t is in buffer t - t0 modulo BUFFERS
    int j0 = 0, end = 0, buf = 0;
    tile_at(w.t0, j0, end);
    if (w.t0 < w.t1) stage(j0, end, 0);
    if constexpr (BUFFERS > 2) {
#pragma unroll 1
      for (int t = 1; t < BUFFERS - 1 && w.t0 + t < w.t1; ++t) {
        int j0_then, end_then;
        tile_at(w.t0 + t, j0_then, end_then);
        stage(j0_then, end_then, t);
      }
    }
    for (int t = w.t0; t < w.t1; ++t, buf = buf + 1 == BUFFERS ? 0 : buf + 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      const int j0_now = j0, end_now = end;
      if (t + 1 < w.t1) {
        j0 += KT;
        if (t + 1 == w.sink_tiles) j0 = w.start, end = w.end;
      }
      if constexpr (BUFFERS == 2) {
        if (t + 1 < w.t1) stage(j0, end, buf ^ 1);
      } else if (t + BUFFERS - 1 < w.t1) {
        int j0_then, end_then;
        tile_at(t + BUFFERS - 1, j0_then, end_then);
        stage(j0_then, end_then, buf == 0 ? BUFFERS - 1 : buf - 1);
      }
      const char* kt = lds + buf * 2 * TILE;
      const char* vt = kt + TILE;
      asm volatile("" : "+v"(clean));  // one loop for both walks
      if (__builtin_amdgcn_readfirstlane(clean)) {
        find_bad<T, DP, KB, WAVES>(lds + buf * 2 * TILE + TILE, bad);
        for (int x = 0; x < KT; ++x) {
          const int j = j0_now + x;
          if (!(bad[x / 32] >> (x % 32) & 1u)) continue;
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
            hit |= (j < min(end_now, hi[rb]) && (j >= lo[rb] || j < a.sinks)) << rb;
        }
      }
      // keys that no row of the wave sees, or that all of them see: by 32 keys,
      // or by the tile where a wave has so many rows that it sees nearly all
      // (the blocks of keys then follow each other without a branch)
      if constexpr (RB == 1) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const int jk = j0_now + kb * 32;
          if (jk >= min(hi_last, end_now) || (jk + 32 <= lo_first && jk >= a.sinks)) continue;
          const bool whole = jk + 32 <= min(end_now, hi_first) && (jk >= lo_last || jk + 32 <= a.sinks) &&
                             wave_row + 32 * RB <= w.rows;
          key_step(whole, kt, vt, kb, j0_now, end_now);
        }
      } else {
        if (j0_now >= hi_last || (j0_now + KT <= lo_first && j0_now >= a.sinks)) continue;
        const bool whole = j0_now + KT <= min(end_now, hi_first) &&
                           (j0_now >= lo_last || j0_now + KT <= a.sinks) && wave_row + 32 * RB <= w.rows;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) key_step(whole, kt, vt, kb, j0_now, end_now);
      }
    }

    if (__builtin_amdgcn_readfirstlane(clean)) break;
    float off = 0.f;  // NaN when one of the sums is not finite
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) off = __builtin_fmaf(o[rb][db][i], 0.f, off);
    clean = __syncthreads_or(off != off);
    if (!__builtin_amdgcn_readfirstlane(clean)) break;
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const float sum = sum_halves(l[rb][0] + l[rb][1]);
    const uint32_t r = wave_row + rb * 32 + col;
    const int t = w.token(r), g = static_cast<int>(min(r, w.rows - 1) - static_cast<uint32_t>(t) * w.group);
    const int64_t item = (w.q0 + t) * a.q_heads + w.hk * w.group + g;
    const bool odd = r < w.rows && (hit >> rb & 1);
    if (r < w.rows && !odd) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      if (w.splits > 1) {
        const int64_t at = w.split * a.rows() + item;
        float* part = a.part + a.part_values(w.splits) + at * a.dim;
        if (half == 0) {
          a.part[2 * at] = sum == 0.f ? -__builtin_inff() : mc[rb];
          a.part[2 * at + 1] = sum;
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int d = 32 * db + 8 * (i / 4) + 4 * half + i % 4;
            if (d < a.dim) part[d] = o[rb][db][i];
          }
      } else {
        T* out = static_cast<T*>(a.out) + item * a.dim;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 32 * db + 8 * i + 4 * half;
            T e[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) e[x] = from_f32<T>(o[rb][db][4 * i + x] * inv);
            if (d + 4 <= a.dim) {
              __builtin_memcpy(out + d, e, sizeof e);
            } else {
#pragma unroll
              for (int x = 0; x < 3; ++x)
                if (d + x < a.dim) out[d + x] = e[x];
            }
          }
      }
    }
    uint64_t redo = __ballot(odd && half == 0);  // rows done key by key
    if (redo) {
      // the tiles in LDS may still be read by other waves: each wave takes
      // its row's scratch from its own D floats behind them
      float* q_s = reinterpret_cast<float*>(lds + 2 * BUFFERS * TILE) + wave * DP;
      int j0 = 0, end = 0, sink_from = 0, sink_to = 0, from = 0, to = 0;
      // this split's keys: tiles [t0, t1)
      if (w.t0 < w.sink_tiles) {
        tile_at(w.t0, j0, end);
        sink_from = j0;
        sink_to = min(min(w.t1, w.sink_tiles) * KT, w.sink_end);
      }
      if (w.t1 > w.sink_tiles) {
        from = w.start + (max(w.t0, w.sink_tiles) - w.sink_tiles) * KT;
        to = min(w.start + (w.t1 - w.sink_tiles) * KT, w.end);
      }
      while (redo) {
        const int x = __builtin_ctzll(redo);
        redo &= redo - 1;
        const uint32_t rx = wave_row + rb * 32 + x;
        const int tx = w.token(rx), gx = static_cast<int>(rx - static_cast<uint32_t>(tx) * w.group);
        const int64_t ix = (w.q0 + tx) * a.q_heads + w.hk * w.group + gx;
        int lx, hx, sx;
        seen_keys(tx + w.shift, w.lk, a.left, a.right, a.sinks, lx, hx, sx);
        float mx, lsum, ox[4];
        attend_row(a, static_cast<const T*>(a.q) + (w.q0 + tx) * a.q_row + (w.hk * w.group + gx) * a.q_head, k, v,
                   lx, hx, sx, sink_from, sink_to, from, to, q_s, mx, lsum, ox);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int d = lane + u * kWave;
          if (d >= a.dim) continue;
          if (w.splits > 1) {
            const int64_t at = w.split * a.rows() + ix;
            a.part[a.part_values(w.splits) + at * a.dim + d] = ox[u];
            if (d == 0) {
              a.part[2 * at] = lsum == 0.f ? -__builtin_inff() : mx;
              a.part[2 * at + 1] = lsum;
            }
          } else {
            static_cast<T*>(a.out)[ix * a.dim + d] = from_f32<T>(lsum == 0.f ? 0.f : ox[u] / lsum);
          }
        }
      }
    }
  }
}

template <typename T, int DP, int RB, int KB, int WAVES, bool ALIGNED>
__global__ void __launch_bounds__(kWave * WAVES, waves_per_simd<T>(DP, RB, WAVES)) attend_kernel(AttendArgs a, int tiles_max, int splits) {
  constexpr int ROWS = 32 * RB * WAVES, KT = 32 * KB;
  extern __shared__ __align__(16) char lds[];  // K, V, K, V tiles; a row of q for each wave; KB words
  // tiles of one head next to each other on one XCD (workgroups go round the
  // eight in turn), so that neighbouring windows meet in its L2
  if (splits == 1) {  // (the join does it otherwise)
    int64_t first, last;
    sample_rows(a, first, last);
    if (first > 0 || last < a.n_q)
      zero_outside(static_cast<T*>(a.out), (int64_t)a.q_heads * a.dim, first, last, a.n_q);
  }
  const int64_t blocks = (int64_t)tiles_max * a.k_heads * splits, per = (blocks + 7) / 8;
  const int64_t id = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || id >= blocks) return;
  const int group = a.q_heads / a.k_heads;
  Walk w;
  w.split = static_cast<int>(id % splits);
  w.splits = splits;
  w.hk = static_cast<int>(id / splits / tiles_max);
  int64_t k0;
  int lq, tile;
  if (!find_tile(a, group, ROWS, static_cast<int>(id / splits % tiles_max), w.q0, lq, k0, w.lk, tile)) return;
  const T* k = static_cast<const T*>(a.k) + k0 * a.k_row + w.hk * a.k_head;
  const T* v = static_cast<const T*>(a.v) + k0 * a.v_row + w.hk * a.v_head;

  w.group = group;
  w.row0 = static_cast<uint32_t>(tile) * ROWS;
  w.rows = static_cast<uint32_t>(lq) * group;
  w.shift = w.lk - lq;
  int lo, hi, s, lo2, hi2;
  seen_keys(w.token(w.row0) + w.shift, w.lk, a.left, a.right, a.sinks, lo, hi, s);
  seen_keys(w.token(w.row0 + ROWS - 1) + w.shift, w.lk, a.left, a.right, a.sinks, lo2, hi2, s);
  w.sink_end = min(a.sinks, min(lo, hi2));
  w.start = lo;
  if (a.sinks >= lo) w.sink_end = w.start = 0;
  w.end = max(hi2, w.start);
  w.sink_tiles = (w.sink_end + KT - 1) / KT;
  const int tiles = w.sink_tiles + (w.end - w.start + KT - 1) / KT, each = (tiles + splits - 1) / splits;
  w.t0 = min(w.split * each, tiles);
  w.t1 = min(w.t0 + each, tiles);
  attend_walk<T, DP, RB, KB, WAVES, ALIGNED>(a, w, k, v, lds);
}

// Joins the splits of each row: sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s,
// m the largest m_s; always in the same order.  A workgroup per row: every
// wave works out the splits' weights for itself, then VALUES / 4 threads take
// four values each of every (1024 / VALUES)th split, and the groups' sums meet
// in LDS.
constexpr int kMostSplits = 512;  // two workgroups per CU (attend_cut)

template <typename T, int VALUES>
__global__ void __launch_bounds__(256) attend_join_kernel(AttendArgs a, int splits) {
  constexpr int LANES = VALUES / 4, GROUPS = 256 / LANES;
  __shared__ float weight[kMostSplits];
  __shared__ __align__(16) f32x4 sums[GROUPS][LANES];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t item = blockIdx.x, step = a.rows();
  const float* ml = a.part + 2 * item;
  float m = -__builtin_inff(), l = 0.f;
  for (int s = lane; s < splits; s += kWave) m = fmaxf(m, ml[2 * s * step]);
#pragma unroll
  for (int x = 1; x < kWave; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, kWave));
  const float base = m == -__builtin_inff() ? 0.f : m;
  for (int s = lane; s < splits; s += kWave) {
    const float ls = ml[2 * s * step + 1];
    // a part that saw nothing counts for nothing; NaN sums stay NaN
    const float f = ls == 0.f ? 0.f : exp2f(ml[2 * s * step] - base);
    if (wave == 0) weight[s] = f;
    l += f * ls;
  }
#pragma unroll
  for (int x = 1; x < kWave; x <<= 1) l += __shfl_xor(l, x, kWave);
  __syncthreads();
  const int c = threadIdx.x % LANES, g = threadIdx.x / LANES, d = 4 * c;
  const float* o = a.part + a.part_values(splits) + item * a.dim;
  f32x4 sum = f32x4(0.f);
  if (d < a.dim) {
#pragma unroll 2
    for (int s = g; s < splits; s += GROUPS) {
      const float f = weight[s];
      f32x4 x = f32x4(0.f);
      const float* p = o + s * step * a.dim + d;
      if (d + 4 <= a.dim) __builtin_memcpy(&x, p, 16);
      else
        for (int i = 0; i < 3; ++i) x[i] = d + i < a.dim ? p[i] : 0.f;
      if (f != 0.f) sum += f * x;
    }
  }
  sums[g][c] = sum;
  __syncthreads();
  if (threadIdx.x >= LANES) return;
  sum = f32x4(0.f);
  for (int x = 0; x < GROUPS; ++x) sum += sums[x][c];
  int64_t first, last;
  sample_rows(a, first, last);
  // (a row of no sample has no parts: what was read for it means nothing)
  const bool none = l == 0.f || item < first * a.q_heads || item >= last * a.q_heads;
  T* out = static_cast<T*>(a.out) + item * a.dim;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (d + i < a.dim) out[d + i] = from_f32<T>(none ? 0.f : sum[i] / l);
}

template <typename T>
int launch_join(const AttendArgs& a, int splits, hipStream_t s) {
  const unsigned blocks = static_cast<unsigned>(a.rows());
  if (a.dim <= 64) attend_join_kernel<T, 64><<<blocks, 256, 0, s>>>(a, splits);
  else if (a.dim <= 128) attend_join_kernel<T, 128><<<blocks, 256, 0, s>>>(a, splits);
  else attend_join_kernel<T, 256><<<blocks, 256, 0, s>>>(a, splits);
  TSC_LAUNCH_CHECK("window_attention_join");
  return 0;
}

template <typename T, int DP, int RB, int KB, int WAVES, bool ALIGNED>
int launch_tiles(const AttendArgs& a, const Cut& c, hipStream_t s) {
  constexpr int bytes = tile_buffers<T>(DP, WAVES) * 2 * 32 * KB * DP * (int)sizeof(T) + WAVES * DP * 4 + KB * 4;
  auto kernel = &attend_kernel<T, DP, RB, KB, WAVES, ALIGNED>;
  if (bytes > 65536)
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes)) return rc;
  const int64_t blocks = align_up(c.tiles * a.k_heads * c.splits, 8);
  TSC_REQUIRE(blocks * kWave * WAVES < (1ll << 32), "window_attention: too many tiles");
  kernel<<<static_cast<unsigned>(blocks), kWave * WAVES, bytes, s>>>(a, static_cast<int>(c.tiles), c.splits);
  TSC_LAUNCH_CHECK("window_attention");
  if (c.splits > 1) return launch_join<T>(a, c.splits, s);
  return 0;
}

template <typename T, int DP, bool ALIGNED>
int launch_dim(const AttendArgs& a, const Cut& c, hipStream_t s) {
  constexpr int KB = key_blocks<T>(DP);
  if constexpr (can_pair(DP, sizeof(T)))
    if (c.wave_rows == 2) return launch_tiles<T, DP, 2, KB, 4, ALIGNED>(a, c, s);
  return c.wave_rows ? launch_tiles<T, DP, 1, KB, 4, ALIGNED>(a, c, s)
                     : launch_tiles<T, DP, 1, KB, 1, ALIGNED>(a, c, s);
}

template <typename T, bool ALIGNED>
int launch_aligned(const AttendArgs& a, const Cut& c, hipStream_t s) {
  switch (padded_dim(a.dim)) {
    case 32: return launch_dim<T, 32, ALIGNED>(a, c, s);
    case 64: return launch_dim<T, 64, ALIGNED>(a, c, s);
    case 96: return launch_dim<T, 96, ALIGNED>(a, c, s);
    case 128: return launch_dim<T, 128, ALIGNED>(a, c, s);
    default: return launch_dim<T, 256, ALIGNED>(a, c, s);
  }
}

}  // namespace

template <typename T>
int launch_attend(const AttendArgs& a, const Cut& c, hipStream_t s) {
  const int64_t e = kPer16<T>;
  // 16-byte pieces at 16-byte addresses, rows of a tile within 32-bit offsets
  const bool aligned = a.k_row < (1 << 24) && a.v_row < (1 << 24) && a.dim % e == 0 && a.k_row % e == 0 && a.v_row % e == 0 && a.k_head % e == 0 &&
                       a.v_head % e == 0 && reinterpret_cast<uintptr_t>(a.k) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(a.v) % 16 == 0;
  return aligned ? launch_aligned<T, true>(a, c, s) : launch_aligned<T, false>(a, c, s);
}

}  // namespace tsc
