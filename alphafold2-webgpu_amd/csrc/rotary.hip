// The norm of each query and key head and the rotation by its position, in one
// pass, and the way back:
//
//   n    = x, x / sqrt(mean(x^2) + eps) * w, or (x - mean) / sqrt(var + eps) * w + c  over a head's channels
//   y0   = s (n0 cos a - n1 sin a),  y1 = s (n1 cos a + n0 sin a)   for each pair, a = position * frequency
//
// Back, g the gradient turned by -a and times s: dw = sum g xhat, dc = sum g,
// and with u = g w and r the reciprocal root,
//   rms:   dx = r (u - xhat mean(u xhat))
//   layer: dx = r (u - mean(u) - xhat mean(u xhat)).
//
// Every value is read and written once: HBM bounds it. A head's row is held by
// a group of lanes, 8 channels each: four pairs that turn (4 low and 4 high
// channels in the half layout) or 8 that do not. The angles' cosines and sines
// are computed once for each token and pair (a product and its reduction in
// 64 bits: at position 10^6 a product of 32 bits is off by 0.06 rad) and kept
// in LDS for the token's heads. The first rows are loaded before the angles and
// the lengths: 2 x 4,096 tokens of 32 + 8 heads of 128 channels and the values,
// f16, take 38.6 us, 5.2 TB/s of the 5.33 of a large copy (a call 42, and 46 the
// other way round). Back, 4,096 such tokens take 31 us, 3.6 TB/s with the vectors' sums:
// a row more in flight a lane fills the registers.
#include "heads.h"

namespace afhip {

namespace {

constexpr int kThreads = 256;
constexpr int kInFlight = 4;      // rows a lane group loads before it works on the first
constexpr int kMostTokens = 16;   // a workgroup's, at once
constexpr int kRowsWanted = 128;  // a workgroup's, at once
constexpr int kBackGroups = 1024;  // workgroups of the way back, each with a row of partial sums

// The queries, the keys or the values: a workgroup has one of them.
struct Side {
  const char* x;
  const char* g;  // the way back: the gradient of what `out` is forwards
  char* out;
  const float *scale, *offset;
  float* partial;  // [workgroup][scale, offset][head_dim]
  HeadStrides sx, sg, so;
  int heads;
  int rows;                // the cache's, 0 where out is [batch][tokens]
  int tile_tokens, tiles;  // tokens at once; their number in a sequence
  int groups;              // workgroups
};

struct RotaryArgs {
  Side side[3];
  const int32_t *past, *lengths, *positions;
  const double* frequencies;
  int batch, tokens, head_dim, rotary_dim, layout;
  float epsilon, turn;
};

// The channels a lane has, of a row: four times two neighbours. Turned ones are four pairs, in the half layout two
// fours; where rotary_dim is an odd multiple of 4 (ODD), the last of them has two pairs, and in the half layout the
// four channels behind rotary_dim, two after its low and two after its high ones.
struct Channels {
  int first[4];
};
template <bool ODD> __device__ __forceinline__ Channels channels_of(int unit, int rotary_dim, bool half) {
  const int pairs = rotary_dim / 2;
  Channels c;
  c.first[0] = half && 8 * unit < rotary_dim ? 4 * unit : 8 * unit;
  c.first[2] = half && 8 * unit < rotary_dim ? pairs + 4 * unit : 8 * unit + 4;
  const bool last = ODD && half && 8 * unit < rotary_dim && 8 * unit + 4 == rotary_dim;
  c.first[1] = last ? rotary_dim : c.first[0] + 2;
  c.first[3] = last ? rotary_dim + 2 : c.first[2] + 2;
  return c;
}

template <typename T> struct Vector;
template <> struct Vector<half_t> {
  typedef half4 four;
  typedef half_t two __attribute__((ext_vector_type(2)));
};
template <> struct Vector<float> {
  typedef floatx4 four;
  typedef float two __attribute__((ext_vector_type(2)));
};

template <typename T, bool ODD> __device__ __forceinline__ void load8(const char* row, const Channels& c, float* x) {
  const T* p = reinterpret_cast<const T*>(row);
  if constexpr (ODD) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const auto v = *reinterpret_cast<const typename Vector<T>::two*>(p + c.first[i / 2]);
      x[i] = (float)v[0];
      x[i + 1] = (float)v[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const auto v = *reinterpret_cast<const typename Vector<T>::four*>(p + c.first[i / 2]);
#pragma unroll
      for (int j = 0; j < 4; j++) x[i + j] = (float)v[j];
    }
  }
}
template <typename T, bool ODD> __device__ __forceinline__ void store8(char* row, const Channels& c, const float* x) {
  T* p = reinterpret_cast<T*>(row);
  if constexpr (ODD) {
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      *reinterpret_cast<typename Vector<T>::two*>(p + c.first[i / 2]) =
          typename Vector<T>::two{(T)x[i], (T)x[i + 1]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      typename Vector<T>::four v;
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = (T)x[i + j];
      *reinterpret_cast<typename Vector<T>::four*>(p + c.first[i / 2]) = v;
    }
  }
}

// Sum over a row's lanes, each of them receiving it.
template <int LANES> __device__ __forceinline__ float row_sum(float x) {
  if constexpr (LANES >= 2) x += dpp<0xB1>(x);
  if constexpr (LANES >= 4) x += dpp<0x4E>(x);
  if constexpr (LANES >= 8) x += dpp<0x141>(x);
  if constexpr (LANES >= 16) x += dpp<0x140>(x);
  return x;
}

__device__ __forceinline__ float sum8(const float* x) {
  return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
}

// The sequence's live tokens.
__device__ __forceinline__ int live_tokens(const RotaryArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.tokens) : a.tokens;
}

// Cosines and sines, times the factor, of `count` tokens: [token][pair].
__device__ __forceinline__ void fill_turns(const RotaryArgs& a, int b, int first, int count, float2* turns) {
  const int pairs = a.rotary_dim / 2;
  const int64_t past = a.past ? a.past[b] : 0;
  for (int n = threadIdx.x; n < count * pairs; n += kThreads) {
    const int i = first + n / pairs;
    if (i >= a.tokens) break;
    const double position = a.positions ? (double)a.positions[(int64_t)b * a.tokens + i] : (double)(past + i);
    // In half turns, reduced to [-1, 1].
    double t = position * a.frequencies[n % pairs] * 0.31830988618379067154;
    t -= 2.0 * rint(0.5 * t);
    float c, s;
    sincospif((float)t, &s, &c);
    turns[n] = float2{c * a.turn, s * a.turn};
  }
}

// Turns a lane's four pairs, or where `two` the first two of them; sign -1 goes back.
template <int SIGN> __device__ __forceinline__ void turn4(const float2* turns, bool half, bool two, float* x) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float2 cs = turns[j];
    const float sn = SIGN * cs.y;
    float &x0 = half ? x[j] : x[2 * j], &x1 = half ? x[4 + j] : x[2 * j + 1];
    const float a = x0, b = x1;
    x0 = two && j >= 2 ? a : a * cs.x - b * sn;
    x1 = two && j >= 2 ? b : b * cs.x + a * sn;
  }
}

// The reciprocal root, x made xhat.
template <int LANES, int NORM> __device__ __forceinline__ float normalize(float* x, bool active, int dim, float eps) {
  const float per = 1.0f / (float)dim;
  if constexpr (NORM == AFHIP_HEAD_NORM_LAYER) {
    const float mean = row_sum<LANES>(sum8(x)) * per;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = active ? x[i] - mean : 0.0f;
  }
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; i++) s[i] = x[i] * x[i];
  const float r = 1.0f / sqrtf(row_sum<LANES>(sum8(s)) * per + eps);
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] *= r;
  return r;
}

// Which side a workgroup has, and its number there.
__device__ __forceinline__ int pick_side(const RotaryArgs& a, int& group) {
  group = blockIdx.x;
  if (group < a.side[0].groups) return 0;
  group -= a.side[0].groups;
  if (group < a.side[1].groups) return 1;
  group -= a.side[1].groups;
  return 2;
}

template <typename T, int LANES, int NORM, bool ODD>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  constexpr int GROUPS = kThreads / LANES;
  __shared__ float2 turns[kMostTokens * kMaxHeadDim / 2];
  int tile;
  const int which = pick_side(a, tile);
  const Side& s = a.side[which];
  const int b = tile / s.tiles, first = (tile % s.tiles) * s.tile_tokens;
  const int count = min(s.tile_tokens, a.tokens - first);
  const int unit = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int D = a.head_dim, pairs = a.rotary_dim / 2, heads = s.heads;
  const char* from = s.x + b * s.sx.batch + first * s.sx.token;
  const int token = (int)s.sx.token;  // at most 2^24, of at most 16 tokens
  const int total = count * heads;
  const bool active = 8 * unit < D, turned = 8 * unit < a.rotary_dim, half = a.layout == AFHIP_ROTARY_HALF;
  const bool two = ODD && 8 * unit + 4 == a.rotary_dim;
  const Channels at = channels_of<ODD>(unit, a.rotary_dim, half);
  // A token past the length is read all the same, and not used. The first rows are on their way before all else.
  float x[kInFlight][8];
  auto load = [&](int n0) {
#pragma unroll
    for (int r = 0; r < kInFlight; r++) {
      const int n = min(n0 + r * GROUPS, total - 1), t = n / heads, h = n % heads;
      if (!active) continue;
      const char* p = from + t * token + h * s.sx.head;
      load8<T, ODD>(p, at, x[r]);
    }
  };
  if (!active) {
#pragma unroll
    for (int r = 0; r < kInFlight; r++)
#pragma unroll
      for (int j = 0; j < 8; j++) x[r][j] = 0.0f;
  }
  if (which != 2) load(group);
  const int live = live_tokens(a, b);
  const int64_t past = a.past ? a.past[b] : 0;
  // Row of `out` that the tile's first token goes to; only those in [0, rows) of a cache are written.
  const int64_t row0 = s.rows ? past + first : first;
  char* to = s.out + b * s.so.batch + row0 * s.so.token;
  auto writes = [&](int t) {
    return s.rows == 0 || (first + t < live && row0 + t >= 0 && row0 + t < s.rows);
  };
  if (which == 2) {  // the values, bit for bit
    constexpr int PARTS = 8 * (int)sizeof(T) / 16;
    if (!active) return;
    for (int n0 = group; n0 < total; n0 += kInFlight * GROUPS) {
      u32x4 v[kInFlight][PARTS];
#pragma unroll
      for (int r = 0; r < kInFlight; r++) {
        const int n = min(n0 + r * GROUPS, total - 1);
        const u32x4* p = reinterpret_cast<const u32x4*>(from + n / heads * token + n % heads * s.sx.head);
#pragma unroll
        for (int j = 0; j < PARTS; j++) v[r][j] = p[PARTS * unit + j];
      }
#pragma unroll
      for (int r = 0; r < kInFlight; r++) {
        const int n = n0 + r * GROUPS, t = n / heads, h = n % heads;
        if (n >= total || !writes(t)) continue;
        u32x4* o = reinterpret_cast<u32x4*>(to + t * s.so.token + h * s.so.head);
#pragma unroll
        for (int j = 0; j < PARTS; j++) o[PARTS * unit + j] = v[r][j];
      }
    }
    return;
  }
  float w[8], c[8];
  if (NORM != AFHIP_HEAD_NORM_NONE && active) {
    load8<float, ODD>(reinterpret_cast<const char*>(s.scale), at, w);
    if (NORM == AFHIP_HEAD_NORM_LAYER) {
      load8<float, ODD>(reinterpret_cast<const char*>(s.offset), at, c);
    }
  }
  fill_turns(a, b, first, count, turns);
  __syncthreads();
  for (int n0 = group; n0 < total;) {
#pragma unroll
    for (int r = 0; r < kInFlight; r++) {
      const int n = n0 + r * GROUPS, t = n / heads, h = n % heads;
      if (n >= total) break;
      if constexpr (NORM != AFHIP_HEAD_NORM_NONE) {
        normalize<LANES, NORM>(x[r], active, D, a.epsilon);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          x[r][j] *= w[j];
          if (NORM == AFHIP_HEAD_NORM_LAYER) x[r][j] += c[j];
        }
      }
      if (turned) turn4<1>(turns + t * pairs + 4 * unit, half, two, x[r]);
      if (!active || !writes(t)) continue;
#pragma unroll
      for (int j = 0; j < 8; j++) x[r][j] = first + t < live ? x[r][j] : 0.0f;
      char* p = to + t * s.so.token + h * s.so.head;
      store8<T, ODD>(p, at, x[r]);
    }
    n0 += kInFlight * GROUPS;
    if (n0 < total) load(n0);
  }
}

// The way back. A workgroup takes every groups-th tile of its side's tokens and
// keeps its lanes' sums of the vectors' gradients in registers until the end:
// a row of partial sums each, which rotary_sums_kernel adds up.
template <typename T, int LANES, int NORM, bool ODD>
__global__ __launch_bounds__(kThreads) void rotary_backward_kernel(RotaryArgs a) {
  constexpr int GROUPS = kThreads / LANES, ROWS = 2;
  constexpr int VECTORS = NORM == AFHIP_HEAD_NORM_LAYER ? 2 : NORM == AFHIP_HEAD_NORM_RMS ? 1 : 0;
  __shared__ float2 turns[kMostTokens * kMaxHeadDim / 2];
  int mine;
  const Side& s = a.side[pick_side(a, mine)];
  const int unit = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int D = a.head_dim, pairs = a.rotary_dim / 2, heads = s.heads;
  const bool active = 8 * unit < D, turned = 8 * unit < a.rotary_dim, half = a.layout == AFHIP_ROTARY_HALF;
  const bool two = ODD && 8 * unit + 4 == a.rotary_dim;
  const Channels at = channels_of<ODD>(unit, a.rotary_dim, half);
  const float per = 1.0f / (float)D;
  float w[8], sums[VECTORS ? VECTORS : 1][8] = {};
  if (VECTORS && active) load8<float, ODD>(reinterpret_cast<const char*>(s.scale), at, w);
  for (int tile = mine; tile < a.batch * s.tiles; tile += s.groups) {
    const int b = tile / s.tiles, first = (tile % s.tiles) * s.tile_tokens;
    const int count = min(s.tile_tokens, a.tokens - first), total = count * heads;
    const int live = live_tokens(a, b);
    const char* xs = s.x + b * s.sx.batch + first * s.sx.token;
    const char* gs = s.g + b * s.sg.batch + first * s.sg.token;
    char* to = s.out + ((int64_t)b * a.tokens + first) * heads * D * sizeof(T);
    const int token_x = (int)s.sx.token, token_g = (int)s.sg.token;  // at most 2^24, of at most 16 tokens
    __syncthreads();  // the last tile's turns are read
    fill_turns(a, b, first, count, turns);
    __syncthreads();
    for (int n0 = group; n0 < total; n0 += ROWS * GROUPS) {
      float x[ROWS][8], g[ROWS][8];
      // A token past the length is read all the same, and counts as zeros.
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
        const int n = min(n0 + r * GROUPS, total - 1), t = n / heads, h = n % heads;
#pragma unroll
        for (int j = 0; j < 8; j++) x[r][j] = g[r][j] = 0.0f;
        if (!active) continue;
        const char* p = gs + t * token_g + h * s.sg.head;
        load8<T, ODD>(p, at, g[r]);
        if constexpr (VECTORS != 0) {
          p = xs + t * token_x + h * s.sx.head;
          load8<T, ODD>(p, at, x[r]);
        }
      }
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
        const int n = n0 + r * GROUPS, t = n / heads, h = n % heads;
        if (n >= total) break;
        const bool counts = active && first + t < live;
        if (turned) turn4<-1>(turns + t * pairs + 4 * unit, half, two, g[r]);
        if constexpr (VECTORS != 0) {
          const float root = normalize<LANES, NORM>(x[r], active, D, a.epsilon);
          float gx[8];
#pragma unroll
          for (int j = 0; j < 8; j++) {
            sums[0][j] += counts ? g[r][j] * x[r][j] : 0.0f;
            if constexpr (VECTORS == 2) sums[1][j] += counts ? g[r][j] : 0.0f;
            g[r][j] = active ? g[r][j] * w[j] : 0.0f;
            gx[j] = g[r][j] * x[r][j];
          }
          const float along = row_sum<LANES>(sum8(gx)) * per;
          const float mean = VECTORS == 2 ? row_sum<LANES>(sum8(g[r])) * per : 0.0f;
#pragma unroll
          for (int j = 0; j < 8; j++) g[r][j] = root * (g[r][j] - mean - x[r][j] * along);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) g[r][j] = counts ? g[r][j] : 0.0f;
        if (!active) continue;
        char* p = to + (t * heads + h) * D * (int)sizeof(T);
        store8<T, ODD>(p, at, g[r]);
      }
    }
  }
  if constexpr (VECTORS != 0) {
    __shared__ float rows[kThreads / 64][VECTORS][kMaxHeadDim];
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int v = 0; v < VECTORS; v++) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        float y = sums[v][j];
#pragma unroll
        for (int step = LANES; step < 64; step *= 2) y += __shfl_xor(y, step);
        if (active && (threadIdx.x & 63) < LANES) rows[wave][v][at.first[j / 2] + j % 2] = y;
      }
    }
    __syncthreads();
    float* to = s.partial + (int64_t)mine * VECTORS * D;
    for (int n = threadIdx.x; n < VECTORS * D; n += kThreads) {
      const int v = n / D, c = n % D;
      to[n] = (rows[0][v][c] + rows[1][v][c]) + (rows[2][v][c] + rows[3][v][c]);
    }
  }
}

// Sums the workgroups' rows, 8 columns a workgroup, in 64 bits and in order.
struct SumArgs {
  const float* partial[2];
  int groups[2];
  float* out[2][2];  // [side][scale, offset]
  int dim, columns;  // of a side
};

__global__ __launch_bounds__(kThreads) void rotary_sums_kernel(SumArgs a) {
  constexpr int SLICES = kThreads / 8;
  __shared__ double sums[SLICES][8];
  const int blocks = a.columns / 8, side = blockIdx.x >= blocks;
  const int column = (blockIdx.x - side * blocks) * 8 + threadIdx.x % 8, slice = threadIdx.x / 8;
  const float* partial = a.partial[side];
  double s = 0.0;
#pragma unroll 8
  for (int g = slice; g < a.groups[side]; g += SLICES) s += (double)partial[(int64_t)g * a.columns + column];
  sums[slice][threadIdx.x % 8] = s;
  __syncthreads();
  if (threadIdx.x >= 8) return;
  for (int n = 1; n < SLICES; n++) s += sums[n][threadIdx.x];
  a.out[side][column / a.dim][column % a.dim] = (float)s;
}

int check(const afhip_rotary_desc* desc) {
  AFHIP_REQUIRE(desc != nullptr, "descriptor is NULL");
  const afhip_rotary_desc& d = *desc;
  AFHIP_REQUIRE(d.batch > 0 && d.tokens > 0 && d.query_heads > 0 && d.key_heads > 0 && d.head_dim > 0,
                "rotary dimensions must be positive");
  AFHIP_REQUIRE(d.head_dim % 8 == 0 && d.head_dim <= kMaxHeadDim, "head dimension %d is not a multiple of 8 up to %d",
                d.head_dim, kMaxHeadDim);
  AFHIP_REQUIRE(d.rotary_dim >= 0 && d.rotary_dim % 4 == 0 && d.rotary_dim <= d.head_dim,
                "rotary dimension %d is not a multiple of 4 up to the head dimension %d", d.rotary_dim, d.head_dim);
  AFHIP_REQUIRE(d.query_heads <= 65536 && d.key_heads <= 65536, "more than 65,536 heads");
  AFHIP_REQUIRE(d.layout == AFHIP_ROTARY_HALF || d.layout == AFHIP_ROTARY_INTERLEAVED, "unknown rotary layout %d",
                d.layout);
  AFHIP_REQUIRE(d.norm >= AFHIP_HEAD_NORM_NONE && d.norm <= AFHIP_HEAD_NORM_LAYER, "unknown head norm %d", d.norm);
  AFHIP_REQUIRE(valid_float_dtype(d.dtype), "rotary dtype must be f32 or f16");
  AFHIP_REQUIRE(d.capacity >= 0, "cache capacity is negative");
  AFHIP_REQUIRE(d.epsilon >= 0.0f && d.epsilon < INFINITY, "epsilon must be finite and not negative");
  AFHIP_REQUIRE(fabsf(d.rotation_scale) < INFINITY, "rotation scale must be finite");
  AFHIP_REQUIRE((int64_t)d.batch * d.tokens < ((int64_t)1 << 29), "batch times tokens passes 2^29");
  int s;
  if ((s = check_strides("q", head_strides(d.q, d.tokens, d.query_heads, d.head_dim, d.dtype), d.batch, d.tokens,
                         d.query_heads, d.head_dim, d.dtype, false)) ||
      (s = check_strides("k", head_strides(d.k, d.tokens, d.key_heads, d.head_dim, d.dtype), d.batch, d.tokens,
                         d.key_heads, d.head_dim, d.dtype, false)))
    return s;
  return AFHIP_OK;
}

// What both ways have, and the sides' strides.
RotaryArgs fill(const afhip_rotary_desc& d, const int32_t* past, const int32_t* lengths, const int32_t* positions,
                const double* frequencies, const float* query_scale, const float* key_scale, int least) {
  RotaryArgs a{};
  const int kt = d.capacity ? d.capacity : d.tokens;
  a.side[0].sx = head_strides(d.q, d.tokens, d.query_heads, d.head_dim, d.dtype);
  a.side[1].sx = head_strides(d.k, d.tokens, d.key_heads, d.head_dim, d.dtype);
  a.side[2].sx = head_strides(d.v, d.tokens, d.key_heads, d.head_dim, d.dtype);
  a.side[0].so = head_strides(d.q_out, d.tokens, d.query_heads, d.head_dim, d.dtype);
  a.side[1].so = head_strides(d.k_out, kt, d.key_heads, d.head_dim, d.dtype);
  a.side[2].so = head_strides(d.v_out, kt, d.key_heads, d.head_dim, d.dtype);
  a.side[0].heads = d.query_heads;
  a.side[1].heads = a.side[2].heads = d.key_heads;
  a.side[1].rows = a.side[2].rows = d.capacity;
  a.side[0].scale = query_scale;
  a.side[1].scale = key_scale;
  a.past = past;
  a.lengths = lengths;
  a.positions = positions;
  a.frequencies = frequencies;
  a.batch = d.batch;
  a.tokens = d.tokens;
  a.head_dim = d.head_dim;
  a.rotary_dim = d.rotary_dim;
  a.layout = d.layout;
  a.epsilon = d.epsilon;
  a.turn = d.rotation_scale;
  // As many tokens at once as make kRowsWanted rows, fewer where that leaves
  // workgroups few: `least` of them are aimed at. 3 sequences of 1,021
  // tokens, 8 + 8 heads of 32, f32, take 7.4 us at 512 and 9.1 at 1024; back,
  // 4,096 tokens of 32 + 8 heads of 128, f16, take 36.7 at 512 and 34.9 at 1024.
  for (Side& s : a.side) {
    const int64_t tokens = (int64_t)d.batch * d.tokens;
    int64_t n = ceil_div(kRowsWanted, s.heads);
    if (n > kMostTokens) n = kMostTokens;
    if (n > tokens / least) n = tokens / least > 1 ? tokens / least : 1;
    s.tile_tokens = (int)n;
    s.tiles = (int)ceil_div(d.tokens, n);
    s.groups = d.batch * s.tiles;
  }
  return a;
}

template <typename T, int LANES, int NORM, bool ODD> int launch_way(const RotaryArgs& a, bool back, hipStream_t st) {
  const int64_t groups = (int64_t)a.side[0].groups + a.side[1].groups + a.side[2].groups;
  if (int s = check_grid(groups, kThreads)) return s;
  const dim3 grid((unsigned)groups);
  if (back)
    return launch("rotary.backward", rotary_backward_kernel<T, LANES, NORM, ODD>, grid, dim3(kThreads), 0, st, a);
  return launch("rotary", rotary_kernel<T, LANES, NORM, ODD>, grid, dim3(kThreads), 0, st, a);
}

template <typename T, int LANES, int NORM> int launch_odd(const RotaryArgs& a, bool back, hipStream_t st) {
  if constexpr (LANES > 1)
    if (a.rotary_dim % 8) return launch_way<T, LANES, NORM, true>(a, back, st);
  return launch_way<T, LANES, NORM, false>(a, back, st);
}

template <typename T, int LANES> int launch_norm(const RotaryArgs& a, int norm, bool back, hipStream_t st) {
  if (norm == AFHIP_HEAD_NORM_NONE) return launch_odd<T, LANES, AFHIP_HEAD_NORM_NONE>(a, back, st);
  if (norm == AFHIP_HEAD_NORM_RMS) return launch_odd<T, LANES, AFHIP_HEAD_NORM_RMS>(a, back, st);
  return launch_odd<T, LANES, AFHIP_HEAD_NORM_LAYER>(a, back, st);
}

template <typename T> int launch_lanes(const RotaryArgs& a, int norm, bool back, hipStream_t st) {
  // 4 turned channels of 8 take two lanes: where all lanes have the same channels scalar registers hold them, too many.
  if (a.head_dim <= 8 && a.rotary_dim % 8 == 0) return launch_norm<T, 1>(a, norm, back, st);
  if (a.head_dim <= 16) return launch_norm<T, 2>(a, norm, back, st);
  if (a.head_dim <= 32) return launch_norm<T, 4>(a, norm, back, st);
  if (a.head_dim <= 64) return launch_norm<T, 8>(a, norm, back, st);
  return launch_norm<T, 16>(a, norm, back, st);
}

int launch_any(const RotaryArgs& a, const afhip_rotary_desc& d, bool back, hipStream_t st) {
  return d.dtype == AFHIP_F16 ? launch_lanes<half_t>(a, d.norm, back, st) : launch_lanes<float>(a, d.norm, back, st);
}

int vectors(const afhip_rotary_desc& d) {  // of a side
  return d.norm == AFHIP_HEAD_NORM_LAYER ? 2 : d.norm == AFHIP_HEAD_NORM_RMS ? 1 : 0;
}

int check_side(const char* name, const HeadStrides& s, const void* p, int64_t tokens, int64_t heads,
               const afhip_rotary_desc& d, bool written) {
  if (int e = check_strides(name, s, d.batch, tokens, heads, d.head_dim, d.dtype, written)) return e;
  return check_address(name, p);
}

int check_vectors(const afhip_rotary_desc& d, const double* frequencies, const float* const* scales,
                  const float* const* offsets) {
  AFHIP_REQUIRE(d.rotary_dim == 0 || frequencies != nullptr, "frequencies are NULL");
  for (int i = 0; i < 2; i++) {
    if (d.norm != AFHIP_HEAD_NORM_NONE)
      if (int s = check_address(i ? "key scale" : "query scale", scales[i])) return s;
    if (d.norm == AFHIP_HEAD_NORM_LAYER && offsets)
      if (int s = check_address(i ? "key offset" : "query offset", offsets[i])) return s;
  }
  return AFHIP_OK;
}

}  // namespace

}  // namespace afhip

using namespace afhip;

extern "C" {

int afhip_rotary_run(const afhip_rotary_desc* desc, const void* q, const void* k, const void* v, const int32_t* past,
                     const int32_t* lengths, const int32_t* positions, const double* frequencies,
                     const float* query_scale, const float* query_offset, const float* key_scale,
                     const float* key_offset, void* q_out, void* k_out, void* v_out, void* stream) {
  int s;
  if ((s = require_open()) || (s = check(desc))) return s;
  const afhip_rotary_desc& d = *desc;
  const float* scales[] = {query_scale, key_scale};
  const float* offsets[] = {query_offset, key_offset};
  if ((s = check_vectors(d, frequencies, scales, offsets))) return s;
  RotaryArgs a = fill(d, past, lengths, positions, frequencies, query_scale, key_scale, 512);
  const int kt = d.capacity ? d.capacity : d.tokens;
  if ((s = check_address("q", q)) || (s = check_address("k", k)) ||
      (s = check_side("q_out", a.side[0].so, q_out, d.tokens, d.query_heads, d, true)) ||
      (s = check_side("k_out", a.side[1].so, k_out, kt, d.key_heads, d, true)))
    return s;
  AFHIP_REQUIRE((v != nullptr) == (v_out != nullptr), "v and v_out go together");
  AFHIP_REQUIRE(!v || d.capacity > 0, "v is taken where there is a cache");
  if (!v) a.side[2].groups = 0;
  if (v && ((s = check_side("v", a.side[2].sx, v, d.tokens, d.key_heads, d, false)) ||
            (s = check_side("v_out", a.side[2].so, v_out, kt, d.key_heads, d, true))))
    return s;
  a.side[0].x = (const char*)q;
  a.side[1].x = (const char*)k;
  a.side[2].x = (const char*)v;
  a.side[0].out = (char*)q_out;
  a.side[1].out = (char*)k_out;
  a.side[2].out = (char*)v_out;
  a.side[0].offset = query_offset;
  a.side[1].offset = key_offset;
  return launch_any(a, d, false, (hipStream_t)stream);
}

int afhip_rotary_backward_workspace_size(const afhip_rotary_desc* desc, size_t* bytes) {
  if (int s = check(desc)) return s;
  AFHIP_REQUIRE(bytes != nullptr, "output is NULL");
  *bytes = (size_t)2 * vectors(*desc) * desc->head_dim * kBackGroups * sizeof(float);
  return AFHIP_OK;
}

int afhip_rotary_backward(const afhip_rotary_desc* desc, const void* q, const void* k, const int32_t* past,
                          const int32_t* lengths, const int32_t* positions, const double* frequencies,
                          const float* query_scale, const float* key_scale, const void* dq_out, const void* dk_out,
                          void* dq, void* dk, float* dquery_scale, float* dquery_offset, float* dkey_scale,
                          float* dkey_offset, void* workspace, size_t workspace_bytes, void* stream) {
  int s;
  size_t need = 0;
  if ((s = require_open()) || (s = afhip_rotary_backward_workspace_size(desc, &need))) return s;
  const afhip_rotary_desc& d = *desc;
  AFHIP_REQUIRE(d.capacity == 0, "the way back takes no cache");
  const float* scales[] = {query_scale, key_scale};
  if ((s = check_vectors(d, frequencies, scales, nullptr))) return s;
  RotaryArgs a = fill(d, past, lengths, positions, frequencies, query_scale, key_scale, 1024);
  // The descriptor's q_out and k_out are the gradients' strides; dq and dk are packed.
  for (int i = 0; i < 2; i++) a.side[i].sg = a.side[i].so;
  if ((s = check_address("q", q)) || (s = check_address("k", k)) ||
      (s = check_side("dq_out", a.side[0].sg, dq_out, d.tokens, d.query_heads, d, false)) ||
      (s = check_side("dk_out", a.side[1].sg, dk_out, d.tokens, d.key_heads, d, false)) ||
      (s = check_address("dq", dq)) || (s = check_address("dk", dk)))
    return s;
  const int count = vectors(d);
  AFHIP_REQUIRE(count < 1 || (dquery_scale && dkey_scale), "the gradients of the norms' scales are NULL");
  AFHIP_REQUIRE(count < 2 || (dquery_offset && dkey_offset), "the gradients of the norms' offsets are NULL");
  if (need) {
    AFHIP_REQUIRE(workspace && workspace_bytes >= need, "workspace of %zu bytes is smaller than %zu", workspace_bytes,
                  need);
    if ((s = check_address("workspace", workspace))) return s;
  }
  SumArgs sums{};
  for (int i = 0; i < 2; i++) {
    if (a.side[i].groups > kBackGroups) a.side[i].groups = kBackGroups;
    a.side[i].partial = (float*)workspace + (size_t)i * count * d.head_dim * kBackGroups;
    sums.partial[i] = a.side[i].partial;
    sums.groups[i] = a.side[i].groups;
  }
  a.side[2].groups = 0;
  a.side[0].x = (const char*)q;
  a.side[1].x = (const char*)k;
  a.side[0].g = (const char*)dq_out;
  a.side[1].g = (const char*)dk_out;
  a.side[0].out = (char*)dq;
  a.side[1].out = (char*)dk;
  hipStream_t st = (hipStream_t)stream;
  if ((s = launch_any(a, d, true, st)) || !count) return s;
  sums.out[0][0] = dquery_scale;
  sums.out[0][1] = dquery_offset;
  sums.out[1][0] = dkey_scale;
  sums.out[1][1] = dkey_offset;
  sums.dim = d.head_dim;
  sums.columns = count * d.head_dim;
  return launch("rotary.sums", rotary_sums_kernel, dim3((unsigned)(2 * sums.columns / 8)), dim3(kThreads), 0, st, sums);
}

}  // extern "C"
