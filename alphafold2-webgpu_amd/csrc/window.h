// What the kernels of the windowed attention share (window.hip,
// window_backward.hip): the arguments, which keys a query sees, and tiles of
// rows in LDS with the fragments the MFMA takes from them.
#pragma once

#include "dma.h"
#include "heads.h"

namespace afhip {

constexpr float kWindowLog2e = 1.4426950408889634f;
constexpr float kWindowLn2 = 0.6931471805599453f;

struct WindowArgs {
  const char *q, *k, *v;
  char* out;
  float* lse;
  const int32_t *query_lengths, *key_lengths;
  // Split keys: [row][split] of head_dim sums, then of the reference point and the total. The way back: dk and dv of
  // each chunk of the tiles that may have several.
  float* partial;
  HeadStrides sq, sk, sv, so;
  int batch, queries, keys, query_heads, key_heads, group, head_dim;
  int left, right, sinks;
  float scale, scale_log2;
  int tiles, splits;
  // The way back.
  const char *o, *dout;
  HeadStrides sdo;
  char *dq, *dk, *dv;
  // [batch][key head][row]: the row's lse in base 2 and the sum of out * dout; the keys it sees, below and from.
  float2* rows;
  int2* limits;
  // dk and dv: tiles of keys that every row may see, and the most chunks of rows that one of them and of the others
  // has; the rows of a chunk, and of one where sinks are.
  int long_tiles, chunks, short_chunks, chunk_rows, sink_rows;
  int parts;  // chunks of a key head that leave partial sums
};

typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short window_short4 __attribute__((ext_vector_type(4)));
typedef short window_short8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) window_short4 lds_window_short4;

// Eight values along a product's inner axis, a lane's part of 16. f32 ones are held as three bf16 each, the first 8
// bits, the next 8 and the last 8, which is all of them: of the nine products of two such values the six that reach
// 2^-24 of the whole take 192 cycles of the bf16 MFMA, where one of inner length 16 takes 512 of the f32 MFMA.
struct Parts8 {
  bf16x8 high, mid, low;
};
template <typename T> struct Eight;
template <> struct Eight<half_t> { typedef half8 type; };
template <> struct Eight<float> { typedef Parts8 type; };

__device__ __forceinline__ Parts8 split_parts(floatx8 x) {
  Parts8 p;
  u32x4 part[3];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    uint32_t bits[3][2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      // Cut, not rounded: the rest is exact and has the value's sign. (An infinity's is NaN: products with it are.)
      const uint32_t first = __float_as_uint(x[j + i]) & 0xffff0000u;
      const float rest = x[j + i] - __uint_as_float(first);
      const uint32_t second = __float_as_uint(rest) & 0xffff0000u;
      bits[0][i] = first;
      bits[1][i] = second;
      bits[2][i] = __float_as_uint(rest - __uint_as_float(second));
    }
#pragma unroll
    for (int n = 0; n < 3; n++) part[n][j / 2] = __builtin_amdgcn_perm(bits[n][1], bits[n][0], 0x07060302u);
  }
  p.high = __builtin_bit_cast(bf16x8, part[0]);
  p.mid = __builtin_bit_cast(bf16x8, part[1]);
  p.low = __builtin_bit_cast(bf16x8, part[2]);
  return p;
}

// acc[32 x 32] += A[32 x 16] B[16 x 32]. Element j of the lane's eight pairs with element j of B's in the same half of
// the wave.
__device__ __forceinline__ floatx16 mma(half8 a, half8 b, floatx16 c) { return mfma_f16(a, b, c); }
__device__ __forceinline__ floatx16 mma(const Parts8& a, const Parts8& b, floatx16 c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.low, b.high, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.high, b.low, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b.mid, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b.high, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.high, b.mid, c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.high, b.high, c, 0, 0, 0);
}

// Rows of DP channels (zeros past head_dim) in LDS, their 16-byte chunks XORed with some of the row's bits, for the 64
// banks (256 bytes): sixteen rows that are read at one chunk (nat) lie in sixteen different places, and so do the four
// rows of four chunks of a transposing read (tr): the row's low bits move the groups of four chunks, the next ones the
// chunks of a group. In f32 a transposed value is read by itself, 32 channels of a row and 32 of the row 4 further on
// at once: bit 2 of the row moves the groups of eight.
template <typename T, int DP> struct Tile {
  typedef typename Eight<T>::type Frag;
  static constexpr int kRow = DP * (int)sizeof(T), kChunks = kRow / 16;

  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (sizeof(T) == 4) {
      return kChunks >= 16 ? (row & 3) | ((row & 4) << 1) | ((row & 8) >> 1) : (row >> 1) & 7;
    } else {
      const int low = (row >> 2) & 3;
      return kChunks >= 16 ? ((row & 3) << 2) | low : kChunks == 8 ? ((row & 2) << 1) | low : low;
    }
  }

  // Channels 16 kk + 8 (lane / 32) .. + 8 of row `row`.
  static __device__ __forceinline__ Frag nat(const unsigned char* t, int row, int kk, int hi) {
    const unsigned char* p = t + row * kRow;
    const int sw = swizzle(row);
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const half8*>(p + 16 * ((2 * kk + hi) ^ sw));
    } else {
      const floatx4 a = *reinterpret_cast<const floatx4*>(p + 16 * ((4 * kk + 2 * hi) ^ sw));
      const floatx4 b = *reinterpret_cast<const floatx4*>(p + 16 * ((4 * kk + 2 * hi + 1) ^ sw));
      return split_parts(floatx8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    }
  }

  // Channel 32 cb + lane % 32 of rows row0 + 4 (lane / 32) + {0..3} and those + 8: the rows that the lane's eight
  // accumulators 8 s .. of a product have (mfma_row), row0 = 16 s. In f16 two transposing reads.
  static __device__ __forceinline__ Frag tr(const unsigned char* t, int row0, int cb, int lane) {
    const int hi = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int row = 4 * hi + ((lane & 15) >> 2);  // row0 is a multiple of 16, which the swizzle does not see
      const int chunk = 4 * cb + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      const unsigned char* p = t + row0 * kRow + row * kRow + 8 * (lane & 1);
      const window_short4 x =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_window_short4*)(p + 16 * (chunk ^ swizzle(row))));
      const window_short4 y =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_window_short4*)(p + 8 * kRow + 16 * (chunk ^ swizzle(row + 8))));
      return __builtin_bit_cast(half8, window_short8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
    } else {
      const int ch = 32 * cb + (lane & 31);
      floatx8 f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int row = 4 * hi + (j & 3) + 8 * (j >> 2);
        f[j] = *reinterpret_cast<const float*>(t + row0 * kRow + row * kRow + 16 * ((ch >> 2) ^ swizzle(row)) +
                                               4 * (ch & 3));
      }
      return split_parts(f);
    }
  }
};

// The same tile of ROWS rows of f32 as three of bf16, one behind the other, made once a workgroup by split_two.
template <int DP, int ROWS> struct Planes {
  typedef Tile<half_t, DP> Half;
  static constexpr int kPlane = ROWS * Half::kRow, kBytes = 3 * kPlane;

  static __device__ __forceinline__ Parts8 nat(const unsigned char* t, int row, int kk, int hi) {
    Parts8 p;
    p.high = __builtin_bit_cast(bf16x8, Half::nat(t, row, kk, hi));
    p.mid = __builtin_bit_cast(bf16x8, Half::nat(t + kPlane, row, kk, hi));
    p.low = __builtin_bit_cast(bf16x8, Half::nat(t + 2 * kPlane, row, kk, hi));
    return p;
  }
  static __device__ __forceinline__ Parts8 tr(const unsigned char* t, int row0, int cb, int lane) {
    Parts8 p;
    p.high = __builtin_bit_cast(bf16x8, Half::tr(t, row0, cb, lane));
    p.mid = __builtin_bit_cast(bf16x8, Half::tr(t + kPlane, row0, cb, lane));
    p.low = __builtin_bit_cast(bf16x8, Half::tr(t + 2 * kPlane, row0, cb, lane));
    return p;
  }
  // Of two tiles, one behind the other, eight channels of a row at a time, by THREADS threads.
  template <int THREADS> static __device__ __forceinline__ void split_two(const unsigned char* raw, unsigned char* t) {
    constexpr int EIGHTS = DP / 8, RAW = Tile<float, DP>::kRow;
    static_assert(2 * ROWS * EIGHTS % THREADS == 0, "as many for each thread");
#pragma unroll 1
    for (int n = threadIdx.x; n < 2 * ROWS * EIGHTS; n += THREADS) {
      const int r = n / EIGHTS, e = n % EIGHTS, which = r / ROWS, row = r % ROWS;
      const unsigned char* from = raw + r * RAW;
      const int sw = Tile<float, DP>::swizzle(row);
      const floatx4 a = *reinterpret_cast<const floatx4*>(from + 16 * ((2 * e) ^ sw));
      const floatx4 b = *reinterpret_cast<const floatx4*>(from + 16 * ((2 * e + 1) ^ sw));
      const Parts8 p = split_parts(floatx8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
      unsigned char* to = t + which * kBytes + row * Half::kRow + 16 * (e ^ Half::swizzle(row));
      *reinterpret_cast<bf16x8*>(to) = p.high;
      *reinterpret_cast<bf16x8*>(to + kPlane) = p.mid;
      *reinterpret_cast<bf16x8*>(to + 2 * kPlane) = p.low;
    }
  }
};

// What a wave loads of a tile of ROWS rows of a tensor, shared among WAVES waves.
template <typename T, int DP, int ROWS, int WAVES> struct TileLoad {
  static constexpr int kChunks = Tile<T, DP>::kChunks, kCount = ROWS * kChunks / 64 / WAVES;
  static constexpr int kBytes = ROWS * DP * (int)sizeof(T);
  static_assert(ROWS * kChunks % (64 * WAVES) == 0, "whole instructions for each wave");

  static constexpr int kStep = 64 / kChunks;  // rows of an instruction
  // Offsets held for whole tiles, where they are few and registers are not.
  static constexpr bool kHeld = kCount <= 4 && DP * sizeof(T) <= 256;
  static constexpr int kUnroll = kHeld ? kCount : 2;
  int row, chunk, chunks;  // the lane's row and chunk in a wave's first instruction; a row's chunks
  uint32_t held[kHeld ? kCount : 1];

  __device__ __forceinline__ void init(int wave, int lane, int head_dim, int64_t token) {
    row = kStep * wave + lane / kChunks;
    chunk = lane % kChunks;
    chunks = head_dim * (int)sizeof(T) / 16;
    if constexpr (kHeld) {
#pragma unroll
      for (int n = 0; n < kCount; n++) held[n] = at(n, (uint32_t)token);
    }
  }
  __device__ __forceinline__ int row_of(int n) const { return row + kStep * WAVES * n; }
  // Offsets reach 127 rows, of token strides up to 2^24 bytes: those of a taller tile start anew at each instruction.
  static constexpr bool kTall = ROWS > 128;
  static_assert(kStep * WAVES <= 128, "an instruction's rows are in reach");
  __device__ __forceinline__ uint32_t at(int n, uint32_t token) const {
    const int r = row_of(n), c = chunk ^ Tile<T, DP>::swizzle(r);
    return c < chunks ? (uint32_t)(kTall ? row : r) * token + 16u * c : kOutOfRange;
  }

  // Rows row0 .. of the tensor at `base`: all of them where `whole`, else those that keep(row) holds for and zeros for
  // the others.
  template <typename Keep>
  __device__ __forceinline__ void issue(const char* base, int64_t token, int row0, uint32_t lds, int wave, bool whole,
                                        Keep keep) const {
    const char* first = base + (int64_t)row0 * token;
    int32x4_t rsrc = make_rsrc(first, 0x7ffffff0u);
    if (whole) {
#pragma unroll kUnroll
      for (int n = 0; n < kCount; n++) {
        if (kTall && n > 0) rsrc = make_rsrc(first + (int64_t)n * kStep * WAVES * token, 0x7ffffff0u);
        if constexpr (kHeld) {
          dma16(rsrc, lds + 1024 * (wave + WAVES * n), held[n]);
        } else {
          dma16(rsrc, lds + 1024 * (wave + WAVES * n), at(n, (uint32_t)token));
        }
      }
    } else {
#pragma unroll 1
      for (int n = 0; n < kCount; n++) {
        if (kTall && n > 0) rsrc = make_rsrc(first + (int64_t)n * kStep * WAVES * token, 0x7ffffff0u);
        dma16(rsrc, lds + 1024 * (wave + WAVES * n), keep(row0 + row_of(n)) ? at(n, (uint32_t)token) : kOutOfRange);
      }
    }
  }
};

// Eight channels of a row in global memory; zeros where there are none.
__device__ __forceinline__ half8 load_eight(const half_t* p, bool keep) {
  return keep ? *reinterpret_cast<const half8*>(p) : half8{};
}
__device__ __forceinline__ floatx8 load_eight(const float* p, bool keep) {
  return keep ? *reinterpret_cast<const floatx8*>(p) : floatx8{};
}
__device__ __forceinline__ half8 as_fragment(half8 x) { return x; }
__device__ __forceinline__ Parts8 as_fragment(floatx8 x) { return split_parts(x); }

// Eight accumulators as the second operand of the next product.
__device__ __forceinline__ half8 pack8(const float* x, half8*) {
  half8 f;
#pragma unroll
  for (int j = 0; j < 8; j++) f[j] = (half_t)x[j];
  return f;
}
__device__ __forceinline__ Parts8 pack8(const float* x, Parts8*) {
  return split_parts(floatx8{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]});
}

// Writes four channels.
__device__ __forceinline__ void put4(half_t* p, float a, float b, float c, float d) {
  *reinterpret_cast<half4*>(p) = half4{(half_t)a, (half_t)b, (half_t)c, (half_t)d};
}
__device__ __forceinline__ void put4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<floatx4*>(p) = floatx4{a, b, c, d};
}

// Of two waves on a SIMD one goes first wherever both could issue, so that its MFMAs run beside the other's vector
// instructions and not in step with them: the waves' slots tell them apart. (dk and dv of 4,096 tokens, 16 heads over
// 4 of 128 channels, window 1,024, f16: 97.0 us, and 99.2 without.)
__device__ __forceinline__ void prefer_one_of_two() {
  constexpr int kWaveSlot = 4 | (0 << 6) | (3 << 11);  // HW_ID, bits 0 to 3
  if (__builtin_amdgcn_s_getreg(kWaveSlot) & 1) __builtin_amdgcn_s_setprio(1);
}

// One sequence: its numbers of queries and keys, and where its queries start.
struct Sequence {
  int queries, keys, offset;
  __device__ __forceinline__ Sequence(const WindowArgs& a, int b) {
    queries = a.query_lengths ? min(max(a.query_lengths[b], 0), a.queries) : a.queries;
    keys = a.key_lengths ? min(max(a.key_lengths[b], 0), a.keys) : a.keys;
    offset = keys - queries;
  }
  // Keys [low, high) and those below min(sinks, high) are what query i sees.
  __device__ __forceinline__ int high(const WindowArgs& a, int i) const {
    return a.right < 0 ? keys : min(keys, max(0, offset + i + a.right + 1));
  }
  __device__ __forceinline__ int low(const WindowArgs& a, int i) const {
    return a.left < 0 ? 0 : max(0, offset + i - a.left);
  }
};

// Puts `fill` where a lane's row does not see its sixteen keys from `first` on (its accumulators' rows, mfma_row),
// seeing keys [low, high) and those below min(sinks, high). ends and starts: whether some row of the wave sees not all
// of the block for its end or its start, the same for every lane.
template <typename... X>
__device__ __forceinline__ void hide(int first, int lane, int low, int high, int sinks, bool ends, bool starts,
                                     float fill, X&... x) {
  const int key = first + 4 * (lane >> 5);
  if (ends) {
    const int to = high - key;
#pragma unroll
    for (int v = 0; v < 16; v++) {
      const bool hidden = 8 * (v >> 2) + (v & 3) >= to;
      ((x[v] = hidden ? fill : x[v]), ...);
      if (v == 7) __builtin_amdgcn_sched_barrier(0);  // sixteen masks would fill the scalar registers
    }
  }
  if (starts) {
    const int from = low - key, few = sinks - key;
#pragma unroll
    for (int v = 0; v < 16; v++) {
      // Of keys not yet hidden: below `low` and not below `sinks`.
      const int at = 8 * (v >> 2) + (v & 3);
      const bool hidden = min(from - at, at - few + 1) > 0;
      ((x[v] = hidden ? fill : x[v]), ...);
      if (v == 7) __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// The blocks of BK keys that queries first .. last of a sequence see: `sink_blocks` at the start, then `blocks` from
// `start` on.
struct KeyRange {
  int low, high, sinks, sink_blocks, start, total;
  __device__ __forceinline__ KeyRange(const WindowArgs& a, const Sequence& s, int first, int last, int BK) {
    high = s.high(a, last);
    low = min(s.low(a, first), high);
    sinks = a.left < 0 ? 0 : min(a.sinks, high);
    start = low / BK;
    sink_blocks = min((sinks + BK - 1) / BK, start);
    const int end = (high + BK - 1) / BK;
    total = sink_blocks + (low < high || sinks > start * BK ? end - start : 0);
  }
  __device__ __forceinline__ int block(int t) const { return t < sink_blocks ? t : start + t - sink_blocks; }
  __device__ __forceinline__ bool keeps(int key) const { return (key < high) & ((key >= low) | (key < sinks)); }
  __device__ __forceinline__ bool whole(int k0, int BK) const {
    return k0 + BK <= high && (k0 >= low || k0 + BK <= sinks);
  }
  // The parts t of [begin, end) that a wave computes, whose rows see keys from any_low to below any_high (and the
  // sinks): up to `sink_end`, and from `from` to `to`.
  struct Phases {
    int sink_end, from, to;
  };
  __device__ __forceinline__ Phases phases(int begin, int end, int BK, int any_low, int any_high, bool some) const {
    Phases p;
    p.sink_end = some ? min(end, max(begin, sink_blocks)) : begin;
    // The sinks may reach into the first block of the others.
    const int first = sinks > start * BK ? start : max(start, any_low / BK);
    p.from = some ? min(end, max(p.sink_end, first - start + sink_blocks)) : end;
    p.to = max(p.from, min(end, (any_high + BK - 1) / BK - start + sink_blocks));
    return p;
  }
};

int window_check(const afhip_window_desc* desc);
void window_fill(const afhip_window_desc& d, WindowArgs& a);

}  // namespace afhip
