// The way back through the windowed attention (window.hip): with P = e^(s - lse), s = scale q . k, recomputed from
// what the forward pass left, and D = sum(out * dout) of each row,
//
//   dv = P^T dout,  ds = P (dout V^T - D),  dq = scale ds K,  dk = scale ds^T Q.
//
// Two kernels, seven products in place of the least five: one holds 32 rows a wave and passes over the keys (dq), one
// holds 32 keys a wave and passes over the rows that see them (dk and dv), all query heads of a key head among them. So
// every gradient is summed in registers, in one order, with no atomics. Both keep the held side in registers and
// stream the other through LDS; the probabilities and their gradients feed the next product from the registers they
// were computed in, as in the forward pass.
//
// In f16, P goes into its product times 2^13 (the smallest of a row of 10^6 equal ones is then a normal number), and
// ds, whose size nothing bounds, times a power of two that each held row (or key) lowers when a value would pass 2^15:
// the accumulators are rescaled with it.
//
// Rounded to f16 the row's out makes D, and with it a whole row of ds, wrong by as much as ds' own rounding does where
// a row sees few keys: dq 1.5 to 1.75 times as far from the truth as its own rounding to f16 alone, for 20 to 1,000
// tokens. So dq takes ds as two f16, the rounded one and the rest (an MFMA more for four; 1.1 to 1.4 then), and sums
// ds in f32: the sum is D's error, P having the sum 1, and dk and dv's kernel gets the D that is right.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "window.h"

namespace afhip {

namespace {

template <typename T> constexpr int kBlock = sizeof(T) == 2 ? 64 : 32;  // keys or rows of a streamed block

// The power of two (f16) that brings a held row's, or key's, largest ds of a block to [2^7, 2^8).
__device__ __forceinline__ float fitting(float top) {
  const float both = fmaxf(top, __shfl_xor(top, 32));
  return ldexpf(1.0f, min(126, 8 - __builtin_amdgcn_frexp_expf(both)));
}
__device__ __forceinline__ float largest(const float* ds) {
  float top = fabsf(ds[0]);
#pragma unroll
  for (int v = 1; v < 16; v++) top = fmaxf(top, fabsf(ds[v]));
  return top;
}
template <int BLOCKS> __device__ __forceinline__ void times(floatx16* acc, float f) {
#pragma unroll
  for (int c = 0; c < BLOCKS; c++)
#pragma unroll
    for (int v = 0; v < 16; v++) acc[c][v] *= f;
}

// dq, and each row's lse and D for the other kernel. ROWS waves of 32 rows each, and PARTS times as many where there
// are few rows: each part takes its WK keys of every block, and the parts' sums meet in LDS. MFMA and vector
// instructions bound it about alike: 4,096 tokens, 16 heads over 4 of 128 channels, window 1,024, f16, 85 us, 700
// TFLOP/s over its four products.
template <typename T, int DP, int ROWS, int PARTS, int WK> struct RowTile {
  static constexpr int kRows = 32 * ROWS, kThreads = 64 * ROWS * PARTS;
  static constexpr int kBlock = 2 * PARTS * WK * DP * (int)sizeof(T);  // K and V
  static constexpr int kStages = kBlock > 81920 ? 1 : 2, kLds = kStages * kBlock;
  // Workgroups a CU, for its LDS; the widest f32 takes more than 256 registers.
  static constexpr int kGroups = kLds > 81920 || DP * sizeof(T) > 256 ? 1 : 2;
  static_assert(PARTS == 1 || (PARTS - 1) * ROWS * (DP * 128 + 256) <= kLds, "the other parts' sums fit");
};

template <typename T, int DP, int ROWS, int PARTS, int WK>
__global__
__launch_bounds__((RowTile<T, DP, ROWS, PARTS, WK>::kThreads), (RowTile<T, DP, ROWS, PARTS, WK>::kGroups))
void window_dq_kernel(WindowArgs a) {
  constexpr int BK = WK * PARTS, STEPS = DP / 16, BLOCKS = DP / 32;
  constexpr int HELD = RowTile<T, DP, ROWS, PARTS, WK>::kRows, STAGES = RowTile<T, DP, ROWS, PARTS, WK>::kStages;
  constexpr bool F16 = sizeof(T) == 2;
  typedef TileLoad<T, DP, BK, ROWS * PARTS> Load;
  typedef typename Eight<T>::type Frag;
  typedef Tile<T, DP> Tl;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  prefer_one_of_two();
  const int lane = threadIdx.x & 63, hi = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wave % ROWS, part = wave / ROWS;
  const int heads = a.batch * a.key_heads;
  const int pair = blockIdx.x % heads, tile = a.tiles - 1 - blockIdx.x / heads;
  const int b = pair / a.key_heads, kv = pair % a.key_heads;
  const Sequence s(a, b);
  const int rows = a.queries * a.group;
  const int r0 = tile * HELD, row = r0 + 32 * rg + col;
  const int first = r0 / a.group, last = min(s.queries - 1, (r0 + HELD - 1) / a.group);
  const int i = row / a.group, h = kv * a.group + row % a.group;
  const bool live = i < s.queries;
  const int at = min(i, s.queries - 1), high = s.high(a, at), low = s.low(a, at);

  // The first keys are on their way before all else.
  const KeyRange range(a, s, first, last, BK);
  const int total = first < s.queries ? range.total : 0;
  const int wr0 = r0 + 32 * rg;
  const int wfirst = min(wr0 / a.group, s.queries - 1), wlast = min((wr0 + 31) / a.group, s.queries - 1);
  const int all_low = s.low(a, wlast), all_high = s.high(a, wfirst);
  const char* kb = a.k + b * a.sk.batch + kv * a.sk.head;
  const char* vb = a.v + b * a.sv.batch + kv * a.sv.head;
  const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>(smem);
  Load kload, vload;
  kload.init(wave, lane, a.head_dim, a.sk.token);
  vload.init(wave, lane, a.head_dim, a.sv.token);
  auto issue = [&](int t) {
    const int k0 = range.block(t) * BK;
    const uint32_t buffer = lds + (uint32_t)(t % STAGES) * 2 * Load::kBytes;
    const bool whole = range.whole(k0, BK);
    auto keep = [&](int key) { return range.keeps(key); };
    kload.issue(kb, a.sk.token, k0, buffer, wave, whole, keep);
    vload.issue(vb, a.sv.token, k0, buffer + Load::kBytes, wave, whole, keep);
  };
  auto arrive = [&](int t) {
    if (STAGES == 1 && t > 0) {
      block_barrier();  // block t - 1 is read
      issue(t);
    }
    wait_vmcnt<0>();
    block_barrier();
    if (STAGES == 2 && t + 1 < total) issue(t + 1);
  };
  if (total > 0) issue(0);

  Frag q[STEPS], g[STEPS];
  float delta = 0.0f;
  float* left_delta;
  float lse = INFINITY;
  {
    const int64_t src = live ? i : 0;
    const char* qp = a.q + b * a.sq.batch + src * a.sq.token + h * a.sq.head;
    const char* gp = a.dout + b * a.sdo.batch + src * a.sdo.token + h * a.sdo.head;
    const char* op = a.o + b * a.so.batch + src * a.so.token + h * a.so.head;
#pragma unroll
    for (int kk = 0; kk < STEPS; kk++) {
      const int ch = 16 * kk + 8 * hi;
      const bool keep = live && ch < a.head_dim;
      q[kk] = as_fragment(load_eight(reinterpret_cast<const T*>(qp) + ch, keep));
      const auto y = load_eight(reinterpret_cast<const T*>(gp) + ch, keep);
      const auto o = load_eight(reinterpret_cast<const T*>(op) + ch, keep);
      g[kk] = as_fragment(y);
#pragma unroll
      for (int j = 0; j < 8; j++) delta += (float)o[j] * (float)y[j];
    }
    delta += __shfl_xor(delta, 32);
    if (live) {
      lse = a.lse[((int64_t)b * a.query_heads + h) * a.queries + i] * kWindowLog2e;
      if (lse == -INFINITY) lse = INFINITY;  // nothing seen: probabilities of 0
    }
    left_delta = &a.rows[(int64_t)pair * rows + row].y;
    if (row < rows && !hi && part == 0) {
      a.rows[(int64_t)pair * rows + row] = float2{lse, delta};
      a.limits[(int64_t)pair * rows + row] = live ? int2{high, low} : int2{0, 0};
    }
  }
  // As a factor that the compiler does not see, it makes a difference and its rounding to f16 one instruction.
  float one = 1.0f;
  asm("" : "+s"(one));
  float rest = 0.0f;  // f16: the sum of the row's ds, which is what out's rounding put D off by
  // ds comes from the exponential with its power of two. The first holds the product of any f16 dout and v.
  int shift = F16 ? 60 : 0;
  float from = (float)shift - lse;
  floatx16 acc[BLOCKS];
#pragma unroll
  for (int c = 0; c < BLOCKS; c++) acc[c] = floatx16{};
  // As in window_rows_kernel.
  const auto phases =
      range.phases(0, total, BK, s.low(a, wfirst), s.high(a, wlast), wr0 < s.queries * a.group);
  int t = 0;
#pragma unroll 1
  for (int phase = 0; phase < 2; phase++) {
    const int work = phase ? phases.to : phases.sink_end, idle = phase ? total : phases.from;
    for (; t < work; t++) {
      arrive(t);
      const int at = WK * part, k0 = range.block(t) * BK + at;
      const bool ends = k0 + WK > all_high, starts = k0 < all_low && k0 + WK > range.sinks;
      const unsigned char* kt = smem + (t % STAGES) * 2 * Load::kBytes + at * Tl::kRow;
      const unsigned char* vt = kt + Load::kBytes;
#pragma unroll 1
      for (int sub = 0; sub < WK; sub += 32) {
        floatx16 x = floatx16{}, y = floatx16{};
#pragma unroll
        for (int kk = 0; kk < STEPS; kk++) {
          x = mma(Tl::nat(kt, sub + col, kk, hi), q[kk], x);
          y = mma(Tl::nat(vt, sub + col, kk, hi), g[kk], y);
        }
        float ds[16];
#pragma unroll
        for (int v = 0; v < 16; v++)
          ds[v] = __builtin_amdgcn_exp2f(fmaf(x[v], a.scale_log2, from)) * (y[v] - delta);
        if (ends | starts) hide(k0 + sub, lane, low, high, range.sinks, ends, starts, 0.0f, ds);
        if constexpr (F16) {
          const float top = largest(ds);
          if (__builtin_amdgcn_ballot_w64(top > 0x1p15f)) {
            const float f = fminf(fitting(top), 1.0f);
            times<BLOCKS>(acc, f);
            rest *= f;
#pragma unroll
            for (int v = 0; v < 16; v++) ds[v] *= f;
            const int by = __builtin_amdgcn_frexp_expf(f) - 1;
            shift += by;
            from += (float)by;
          }
          rest += (((ds[0] + ds[1]) + (ds[2] + ds[3])) + ((ds[4] + ds[5]) + (ds[6] + ds[7]))) +
                  (((ds[8] + ds[9]) + (ds[10] + ds[11])) + ((ds[12] + ds[13]) + (ds[14] + ds[15])));
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
          Frag f = pack8(ds + 8 * n, (Frag*)nullptr), g;
          if constexpr (F16) {
            asm("" : "+v"(f));  // else each half is rounded once more
#pragma unroll
            for (int j = 0; j < 8; j++) g[j] = (half_t)fmaf(ds[8 * n + j], one, -(float)f[j]);
          }
#pragma unroll
          for (int c = 0; c < BLOCKS; c++) {
            const Frag k = Tl::tr(kt, sub + 16 * n, c, lane);
            if constexpr (F16) acc[c] = mma(k, g, acc[c]);
            acc[c] = mma(k, f, acc[c]);
          }
        }
      }
    }
    for (; t < idle; t++) arrive(t);
  }
  times<BLOCKS>(acc, ldexpf(a.scale, -shift));
  if (F16) rest = ldexpf(rest, -shift);
  if constexpr (PARTS > 1) {
    constexpr int SUMS = (PARTS - 1) * ROWS * BLOCKS * 1024;  // then the rests
    float* shared = reinterpret_cast<float*>(smem) + rg * BLOCKS * 1024 + lane;
    float* rests = reinterpret_cast<float*>(smem) + SUMS + rg * 64 + lane;
    block_barrier();  // the last block is read
    if (part > 0) {
      rests[(part - 1) * ROWS * 64] = rest;
#pragma unroll
      for (int c = 0; c < BLOCKS; c++)
#pragma unroll
        for (int v = 0; v < 16; v++) shared[((part - 1) * ROWS * BLOCKS * 16 + 16 * c + v) * 64] = acc[c][v];
    }
    block_barrier();
    if (part > 0) return;
#pragma unroll 1
    for (int p = 0; p < PARTS - 1; p++) {
      rest += rests[p * ROWS * 64];
#pragma unroll
      for (int c = 0; c < BLOCKS; c++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[c][v] += shared[(p * ROWS * BLOCKS * 16 + 16 * c + v) * 64];
    }
  }
  if (F16) rest += __shfl_xor(rest, 32);
  if (row >= rows) return;
  if (F16 && !hi) *left_delta = delta + rest;
  T* to = reinterpret_cast<T*>(a.dq) + (((int64_t)b * a.queries + i) * a.query_heads + h) * a.head_dim;
#pragma unroll
  for (int c = 0; c < BLOCKS; c++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int ch = 32 * c + 8 * g + 4 * hi;
      if (ch >= a.head_dim) continue;
      const floatx16& x = acc[c];
      put4(to + ch, live ? x[4 * g] : 0.0f, live ? x[4 * g + 1] : 0.0f, live ? x[4 * g + 2] : 0.0f,
           live ? x[4 * g + 3] : 0.0f);
    }
}

// dk and dv of a tile of keys of a key head, over blocks of its rows: KEYS groups of 32 keys, each with ROWS waves that
// take 32 rows of a block in turn and meet in LDS at the end. Each wave reads every row of its part four times from
// LDS (for two products as it lies and for two transposed), which takes as long as its MFMAs: eight waves a CU let the
// one hide behind the other. What bounds it is each wave's own chain, MFMA to exponential to MFMA, with two waves a
// SIMD: 2.8 us a block of 64 rows over 128 channels in f16 (1.9 over 64, 0.9 over 32; f32 9, 4.5, 3.5).
//
// Tiles differ in how many rows see them (those of the sinks: all), and few sequences have few tiles: the rows are cut
// into chunks, and a tile of several leaves partial sums, joined by window_dkv_join_kernel.
template <typename T, int DP> struct KeyTile {
  // Values of three bf16 take more than the 256 registers that eight waves have each from 64 channels on.
  static constexpr int kKeyGroups = sizeof(T) == 4 && DP > 32 ? 2 : 4, kRowGroups = 2;
  static constexpr int kThreads = 64 * kKeyGroups * kRowGroups;
  static constexpr int kKeys = 32 * kKeyGroups, kRows = 32 * kRowGroups;
  static constexpr int kStats = 16 * kRows;  // the rows' statistics and limits
  static constexpr int kTileBytes = kRows * DP * (int)sizeof(T), kBuffer = 2 * kTileBytes + kStats;
  // Whether V is read from LDS at each block, a quarter more of LDS reads, where K, V and the sums would leave no
  // registers to read fragments ahead of their MFMAs.
  static constexpr bool kShareV = DP == 128 && sizeof(T) == 2;
  static constexpr int kVBytes = kShareV ? kKeys * DP * (int)sizeof(T) : 0, kLds = 2 * kBuffer + kVBytes;
};

// Rows that see any key of a tile, and its chunks of them.
struct TileRows {
  int begin, stop, chunk_rows, chunks;
  __device__ __forceinline__ TileRows(const WindowArgs& a, const Sequence& s, int from, int to) {
    int first, end;
    queries(a, s, from, to, first, end);
    begin = first * a.group;
    stop = max(begin, end * a.group);
    chunk_rows = from < a.sinks ? a.sink_rows : a.chunk_rows;
    chunks = (stop - begin + chunk_rows - 1) / chunk_rows;
  }
  // Queries [first, end) that see any of keys [from, to).
  static __device__ __forceinline__ void queries(const WindowArgs& a, const Sequence& s, int from, int to, int& first,
                                                 int& end) {
    to = min(to, s.keys);
    first = a.right < 0 ? 0 : max(0, from - a.right - s.offset);
    end = a.left < 0 || from < a.sinks ? s.queries : min(s.queries, max(0, to + a.left - s.offset));
    if (from >= to) end = 0;
  }
};

template <typename T, int DP> constexpr int kKeyTileThreads = KeyTile<T, DP>::kThreads;

template <typename T, int DP>
__global__ __launch_bounds__((kKeyTileThreads<T, DP>)) void window_dkv_kernel(WindowArgs a) {
  typedef KeyTile<T, DP> KT;
  typedef Tile<T, DP> Tl;
  typedef typename Eight<T>::type Frag;
  constexpr int BR = KT::kRows, STEPS = DP / 16, BLOCKS = DP / 32, WAVES = KT::kThreads / 64;
  constexpr int CHUNKS = Tl::kChunks, STEP = 64 / CHUNKS, COUNT = BR * CHUNKS / 64;
  constexpr int TILE = KT::kTileBytes;
  constexpr bool F16 = sizeof(T) == 2;
  constexpr float LIFT = F16 ? 13.0f : 0.0f;  // on P's exponent, and so on ds
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  prefer_one_of_two();
  const int lane = threadIdx.x & 63, hi = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave % KT::kKeyGroups, rg = wave / KT::kKeyGroups;
  const int heads = a.batch * a.key_heads;
  const int pair = blockIdx.x % heads, rest = blockIdx.x / heads, longs = a.long_tiles * a.chunks;
  const int tile = rest < longs ? rest / a.chunks : a.long_tiles + (rest - longs) / a.short_chunks;
  const int chunk = rest < longs ? rest % a.chunks : (rest - longs) % a.short_chunks;
  const int b = pair / a.key_heads, kv = pair % a.key_heads;
  const Sequence s(a, b);
  const int G = a.group, rows = a.queries * G;
  const int j0 = tile * KT::kKeys, wj0 = j0 + 32 * kg, key = wj0 + col;
  const bool live = key < s.keys;
  const TileRows range(a, s, j0, j0 + KT::kKeys);
  if (chunk > 0 && chunk >= range.chunks) return;
  const int begin = range.begin + chunk * range.chunk_rows, stop = min(range.stop, begin + range.chunk_rows);

  const unsigned char* vt = smem + 2 * KT::kBuffer;
  floatx16 dk[BLOCKS], dv[BLOCKS];
  float dk_scale = F16 ? 0x1p126f : 1.0f;
#pragma unroll
  for (int c = 0; c < BLOCKS; c++) dk[c] = dv[c] = floatx16{};

  if (begin < stop) {
    int wfirst, wend;
    TileRows::queries(a, s, wj0, wj0 + 32, wfirst, wend);
    const char* qb = a.q + b * a.sq.batch + (int64_t)kv * G * a.sq.head;
    const char* gb = a.dout + b * a.sdo.batch + (int64_t)kv * G * a.sdo.head;
    const float per = 1.0f / (float)G;
    const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>(smem);
    const int chunks = a.head_dim * (int)sizeof(T) / 16;
    // Of the block to load next: its first row's query and head. Where a block holds whole queries every block's rows
    // lie alike, and their offsets are kept.
    int i0 = begin / G, g0 = begin - i0 * G;
    const int step_i = BR / G, step_g = BR - step_i * G;
    // Row r of a block is query i0 + t / G, head t % G, with t = r + g0: below 2^17, where the rounded quotient of
    // t + 1/2 has the right whole part.
    auto offset = [&](int m, const HeadStrides& s) {
      const int r = STEP * m + lane / CHUNKS, c = (lane % CHUNKS) ^ Tl::swizzle(r);
      const int t = r + g0, i = (int)(((float)t + 0.5f) * per), g = t - i * G;
      return c < chunks ? (uint32_t)i * (uint32_t)s.token + (uint32_t)g * (uint32_t)s.head + 16u * c : kOutOfRange;
    };
    constexpr bool KEPT = COUNT % WAVES == 0 && COUNT / WAVES <= 2;
    uint32_t q_at[KEPT ? COUNT / WAVES : 1], g_at[KEPT ? COUNT / WAVES : 1];
    if constexpr (KEPT) {
#pragma unroll
      for (int j = 0; j < COUNT / WAVES; j++) {
        q_at[j] = offset(wave + WAVES * j, a.sq);
        g_at[j] = offset(wave + WAVES * j, a.sdo);
      }
    }
    auto issue = [&](int r0, int n) {
      const int32x4_t qr = make_rsrc(qb + (int64_t)i0 * a.sq.token, 0x7ffffff0u);
      const int32x4_t gr = make_rsrc(gb + (int64_t)i0 * a.sdo.token, 0x7ffffff0u);
      const uint32_t buffer = lds + (uint32_t)(n & 1) * KT::kBuffer;
      bool done = false;
      if constexpr (KEPT) {
        if (step_g == 0 && r0 + BR <= stop) {
#pragma unroll
          for (int j = 0; j < COUNT / WAVES; j++) {
            dma16(qr, buffer + 1024 * (wave + WAVES * j), q_at[j]);
            dma16(gr, buffer + TILE + 1024 * (wave + WAVES * j), g_at[j]);
          }
          done = true;
        }
      }
      if (!done) {
#pragma unroll 1
        for (int m = wave; m < COUNT; m += WAVES) {
          const bool ok = r0 + STEP * m + lane / CHUNKS < stop;
          dma16(qr, buffer + 1024 * m, ok ? offset(m, a.sq) : kOutOfRange);
          dma16(gr, buffer + TILE + 1024 * m, ok ? offset(m, a.sdo) : kOutOfRange);
        }
      }
      // The rows' statistics, 8 bytes each, 32 rows an instruction: lse and D, and the keys they see. Past the last
      // row zeros, whose rows of dout are zeros too.
      if (wave < 2 * KT::kRowGroups) {
        const int part = 32 * (wave >> 1);
        const int64_t at = (int64_t)pair * rows + r0 + part;
        const int32x4_t sr = make_rsrc(wave & 1 ? (const void*)(a.limits + at) : (const void*)(a.rows + at),
                                       8u * (uint32_t)max(0, min(32, stop - r0 - part)));
        dma4(sr, buffer + 2 * TILE + 8 * (wave & 1 ? BR : 0) + 8 * part, 4u * lane);
      }
      i0 += step_i;
      g0 += step_g;
      if (g0 >= G) g0 -= G, i0++;
    };
    if constexpr (KT::kShareV) {
      TileLoad<T, DP, KT::kKeys, WAVES> load;
      load.init(wave, lane, a.head_dim, a.sv.token);
      load.issue(a.v + b * a.sv.batch + kv * a.sv.head, a.sv.token, j0, lds + 2 * KT::kBuffer, wave, false,
                 [&](int key) { return key < s.keys; });
    }
    // Over 128 channels of f32 K and V are held as they are, and made three bf16 at each use, which costs a tenth of
    // the MFMAs' time: as parts they would not fit.
    constexpr bool RAW = sizeof(T) == 4 && DP == 128;
    typedef typename std::conditional<RAW, floatx8, Frag>::type Held;
    Held kf[STEPS], vf[KT::kShareV ? 1 : STEPS];
    auto held = [](Held& x) {
      if constexpr (RAW) {
        asm volatile("" : "+v"(x));  // not ahead of the loop
        return split_parts(x);
      } else {
        return x;
      }
    };
    {
      const int64_t src = live ? key : 0;
      const char* kp = a.k + b * a.sk.batch + src * a.sk.token + kv * a.sk.head;
      const char* vp = a.v + b * a.sv.batch + src * a.sv.token + kv * a.sv.head;
#pragma unroll
      for (int kk = 0; kk < STEPS; kk++) {
        const int ch = 16 * kk + 8 * hi;
        const bool keep = live && ch < a.head_dim;
        const auto x = load_eight(reinterpret_cast<const T*>(kp) + ch, keep);
        if constexpr (RAW) {
          kf[kk] = x;
          vf[kk] = load_eight(reinterpret_cast<const T*>(vp) + ch, keep);
        } else {
          kf[kk] = as_fragment(x);
          if constexpr (!KT::kShareV) vf[kk] = as_fragment(load_eight(reinterpret_cast<const T*>(vp) + ch, keep));
        }
      }
    }
    issue(begin, 0);
    int n = 0, r0 = begin;
    auto arrive = [&] {
      wait_vmcnt<0>();
      block_barrier();
      if (r0 + BR < stop) issue(r0 + BR, n + 1);
    };
    // Blocks with rows that see the wave's keys, between such that only see other waves'; its own 32 rows of the last
    // block may be past the end, and are zeros then.
    const int wbegin = wfirst * G, wstop = min(stop, wend * G);
    // Rows that see all of them.
    const int never = rows + 1;
    const int full_begin =
        wj0 + 32 > s.keys ? never : a.right < 0 ? 0 : min(s.queries, max(0, wj0 + 31 - a.right - s.offset)) * G;
    const int full_stop =
        a.left < 0 || wj0 + 32 <= a.sinks ? never : min(s.queries, max(0, wj0 + a.left - s.offset + 1)) * G;
#pragma unroll 1
    for (int phase = 0; phase < 2; phase++) {
      for (const int idle = phase ? stop : min(stop, wbegin - BR + 1); r0 < idle; r0 += BR, n++) arrive();
      for (; r0 < wstop; r0 += BR, n++) {
        arrive();
        const int w0 = r0 + 32 * rg;
        const bool partial = w0 < full_begin || min(w0 + 32, stop) > full_stop;
        const unsigned char* qt = smem + (n & 1) * KT::kBuffer;
        const unsigned char* gt = qt + TILE;
        const float2* stats = reinterpret_cast<const float2*>(gt + TILE) + 32 * rg;
        const int sub = 32 * rg;
        floatx16 x = floatx16{};
#pragma unroll
        for (int kk = 0; kk < STEPS; kk++) x = mma(Tl::nat(qt, sub + col, kk, hi), held(kf[kk]), x);
        float p[16];
#pragma unroll
        for (int v = 0; v < 16; v++)
          p[v] = __builtin_amdgcn_exp2f(fmaf(x[v], a.scale_log2, LIFT - stats[mfma_row(v, lane)].x));
        const int2* limits = reinterpret_cast<const int2*>(stats + BR);
        if (partial) {
#pragma unroll
          for (int v = 0; v < 16; v++) {
            const int2 lim = limits[mfma_row(v, lane)];
            // As one comparison: a block's sixteen would fill the scalar registers with masks.
            if (min(max(lim.y - key, key - lim.x + 1), key - min(a.sinks, lim.x) + 1) > 0) p[v] = 0.0f;
            if (sizeof(T) == 4 && v % 4 == 3) __builtin_amdgcn_sched_barrier(0);
          }
        }
        floatx16 y = floatx16{};
#pragma unroll
        for (int kk = 0; kk < STEPS; kk++) {
          if constexpr (KT::kShareV) {
            y = mma(Tl::nat(gt, sub + col, kk, hi), Tl::nat(vt, 32 * kg + col, kk, hi), y);
          } else {
            y = mma(Tl::nat(gt, sub + col, kk, hi), held(vf[kk]), y);
          }
        }
        float ds[16];
#pragma unroll
        for (int v = 0; v < 16; v++) ds[v] = p[v] * (y[v] - stats[mfma_row(v, lane)].y);
        if (partial) {  // what is not seen stays 0 whatever its gradient is
#pragma unroll
          for (int v = 0; v < 16; v++) ds[v] = p[v] == 0.0f ? 0.0f : ds[v];
        }
        if constexpr (F16) {
          const float top = largest(ds);
          if (__builtin_amdgcn_ballot_w64(top * dk_scale > 0x1p15f)) {
            const float next = fminf(fitting(top), dk_scale);
            times<BLOCKS>(dk, next / dk_scale);
            dk_scale = next;
          }
#pragma unroll
          for (int v = 0; v < 16; v++) ds[v] *= dk_scale;
        }
#pragma unroll
        for (int m = 0; m < 2; m++) {
          const Frag pf = pack8(p + 8 * m, (Frag*)nullptr), df = pack8(ds + 8 * m, (Frag*)nullptr);
#pragma unroll
          for (int c = 0; c < BLOCKS; c++) {
            dv[c] = mma(Tl::tr(gt, sub + 16 * m, c, lane), pf, dv[c]);
            dk[c] = mma(Tl::tr(qt, sub + 16 * m, c, lane), df, dk[c]);
          }
        }
      }
    }
  }
  // The row groups' sums, in their own magnitude, meet in LDS, one gradient at a time, and leave as whole rows.
  const float fv = F16 ? 0x1p-13f : 1.0f, fk = a.scale * fv / dk_scale;
  constexpr int PITCH = DP + 4;
  static_assert(KT::kKeys * PITCH * 4 <= KT::kLds, "a gradient of the tile fits");
  float* shared = reinterpret_cast<float*>(smem);
  float* own = shared + (32 * kg + col) * PITCH + 4 * hi;
  const bool whole = range.chunks <= 1;
  const int64_t part = (int64_t)pair * a.parts + rest;
  auto leave = [&](const floatx16* x, float f, int which) {
    for (int group = KT::kRowGroups - 1; group >= 0; group--) {
      block_barrier();
      if (rg != group) continue;
#pragma unroll
      for (int c = 0; c < BLOCKS; c++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          floatx4* at = reinterpret_cast<floatx4*>(own + 32 * c + 8 * g);
          floatx4 y{x[c][4 * g] * f, x[c][4 * g + 1] * f, x[c][4 * g + 2] * f, x[c][4 * g + 3] * f};
          if (group < KT::kRowGroups - 1) y += *at;
          *at = y;
        }
    }
    block_barrier();
    const int quads = a.head_dim / 4;
    for (int n = threadIdx.x; n < KT::kKeys * quads; n += KT::kThreads) {
      const int j = n / quads, ch = 4 * (n % quads);
      if (j0 + j >= a.keys) break;
      floatx4 y = *reinterpret_cast<const floatx4*>(shared + j * PITCH + ch);
      if (!whole) {
        *reinterpret_cast<floatx4*>(a.partial + ((2 * part + which) * KT::kKeys + j) * a.head_dim + ch) = y;
      } else {
        if (j0 + j >= s.keys) y = floatx4{};
        T* to = reinterpret_cast<T*>(which ? a.dv : a.dk) +
                (((int64_t)b * a.keys + j0 + j) * a.key_heads + kv) * a.head_dim + ch;
        put4(to, y[0], y[1], y[2], y[3]);
      }
    }
  };
  leave(dk, fk, 0);
  leave(dv, fv, 1);
}

// Adds up the chunks of the tiles that have several, in order: 1,024 values a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void window_dkv_join_kernel(WindowArgs a, int tile_keys, int parts) {
  const int heads = a.batch * a.key_heads;
  const int pair = blockIdx.x % heads, rest = blockIdx.x / heads, tile = rest / parts, part = rest % parts;
  const int b = pair / a.key_heads, kv = pair % a.key_heads, D = a.head_dim;
  const Sequence s(a, b);
  const TileRows range(a, s, tile * tile_keys, (tile + 1) * tile_keys);
  if (range.chunks <= 1) return;
  const int n = part * 1024 + 4 * (int)threadIdx.x, size = 2 * tile_keys * D;
  if (n >= size) return;
  const int which = n >= tile_keys * D, m = n - which * tile_keys * D, key = tile * tile_keys + m / D, ch = m % D;
  if (key >= a.keys) return;
  const int first = tile < a.long_tiles ? tile * a.chunks
                                        : a.long_tiles * a.chunks + (tile - a.long_tiles) * a.short_chunks;
  const float* from = a.partial + ((int64_t)pair * a.parts + first) * size + n;
  floatx4 x{};
#pragma unroll 4
  for (int c = 0; c < range.chunks; c++) x += *reinterpret_cast<const floatx4*>(from + (int64_t)c * size);
  if (key >= s.keys) x = floatx4{};
  T* to = reinterpret_cast<T*>(which ? a.dv : a.dk) + (((int64_t)b * a.keys + key) * a.key_heads + kv) * D + ch;
  put4(to, x[0], x[1], x[2], x[3]);
}

// The key tiles, and the rows of a chunk.
struct KeyPlan {
  int tile_keys, tiles, chunk_rows, sink_rows;
  int long_tiles, chunks, short_chunks;  // tiles that every row may see, the chunks of one, those of the others
  int64_t groups(int64_t heads) const {
    return heads * ((int64_t)long_tiles * chunks + (int64_t)(tiles - long_tiles) * short_chunks);
  }
  // Tiles, of the first, that may have several chunks, and those chunks.
  int joined() const { return chunks == 1 ? 0 : short_chunks == 1 ? long_tiles : tiles; }
  int64_t parts() const {
    return joined() == tiles ? groups(1) : (int64_t)joined() * chunks;
  }
};

KeyPlan key_plan(const afhip_window_desc& d) {
  KeyPlan p{};
  const bool f32 = d.dtype == AFHIP_F32, wide = d.head_dim > 32 && f32;
  p.tile_keys = wide ? KeyTile<float, 128>::kKeys : KeyTile<half_t, 128>::kKeys;
  p.tiles = (int)ceil_div(d.keys, p.tile_keys);
  const int64_t group = d.query_heads / d.key_heads, all = d.queries * group, heads = (int64_t)d.batch * d.key_heads;
  // Rows that see a tile, without sinks; without a window on both sides all, or half of them on average.
  const bool window = d.left >= 0 && d.right >= 0, half = !window && (d.left >= 0 || d.right >= 0);
  const int64_t span = window ? std::min<int64_t>(all, ((int64_t)d.left + d.right + p.tile_keys) * group) : all;
  const bool sinks = d.left >= 0 && d.sinks > 0;
  p.long_tiles = d.left < 0 ? p.tiles : (int)std::min<int64_t>(p.tiles, ceil_div(d.sinks, p.tile_keys));
  // The chunks that take the shortest by what they cost on MI355X in us, a CU having one workgroup at a time: a block
  // of 64 rows, a workgroup's start and end, the join and its sums at 4 TB/s. dk, dv and the join for 4,096 tokens, 16
  // heads over 4 of 128 channels, f16, window 1,024: 3 chunks of each tile 137, 2 102; with 4 sinks, whose tile every
  // row sees, 1 to 5 chunks 191, 166, 146, 169, 156.
  const int width = d.head_dim <= 32 ? 32 : d.head_dim <= 64 ? 64 : 128;
  const double block = f32 ? std::max(3.5, 0.07 * width) : 0.022 * width, ends = f32 && width == 128 ? 25 : 8;
  double best = INFINITY;
  for (int64_t chunks = 1; chunks <= 64; chunks++) {
    const int64_t rows = round_up(ceil_div(span, chunks), 64), each = ceil_div(span, rows);
    if (chunks > 1 && rows < 128) break;
    const int64_t sink_rows = std::max(rows, round_up(ceil_div(all, 64), 64));
    const int64_t most = sinks ? ceil_div(all, sink_rows) : each;
    const double one = ends + block * rows / 64;
    const double groups = (double)heads * (p.long_tiles * most + (p.tiles - p.long_tiles) * each);
    // Tiles of many lengths: what a CU has on average, and half a chunk for the end.
    const double work = (groups + heads * p.tiles) / 2 * ends + (double)heads * p.tiles * block * span / 128;
    double time = half ? std::max(one, work / 256 + one / 2) : std::ceil(groups / 256) * one;
    if (each > 1 || most > 1) time += 4 + groups * 4 * p.tile_keys * d.head_dim * 4 / 4e6;
    if (time >= best) continue;
    best = time;
    p.chunk_rows = (int)rows;
    p.sink_rows = (int)sink_rows;
    p.short_chunks = (int)each;
    p.chunks = (int)std::max(each, most);
  }
  return p;
}

size_t chunk_bytes(const afhip_window_desc& d, const KeyPlan& p) {
  return (size_t)d.batch * d.key_heads * p.parts() * 2 * p.tile_keys * d.head_dim * sizeof(float);
}

template <typename T, int DP, int ROWS, int PARTS, int WK>
int launch_dq(WindowArgs& a, int64_t heads, int64_t rows, hipStream_t st) {
  typedef RowTile<T, DP, ROWS, PARTS, WK> RT;
  a.tiles = (int)ceil_div(rows, RT::kRows);
  auto k = window_dq_kernel<T, DP, ROWS, PARTS, WK>;
  int s;
  if ((s = check_grid(heads * a.tiles, RT::kThreads)) || (s = allow_lds((const void*)k, RT::kLds))) return s;
  return launch("window.dq", k, dim3((unsigned)(heads * a.tiles)), dim3(RT::kThreads), RT::kLds, st, a);
}

// Tiles of 128 rows with four waves, or with eight where that would leave CUs with fewer, or of 32 rows where those
// would leave most CUs with nothing.
template <typename T, int DP> int launch_dq_any(WindowArgs& a, int64_t heads, int64_t rows, hipStream_t st) {
  constexpr int WK = kBlock<T>, EIGHT = DP * sizeof(T) > 256 ? 1 : 2;
  constexpr int FEW = DP * sizeof(T) > 64 ? 4 : 8;
  const int64_t groups = heads * ceil_div(rows, 128);
  if (groups < 128) return launch_dq<T, DP, 1, FEW, 32>(a, heads, rows, st);
  if (groups < 512) return launch_dq<T, DP, 4, EIGHT, WK>(a, heads, rows, st);
  return launch_dq<T, DP, 4, 1, WK>(a, heads, rows, st);
}

template <typename T, int DP> int launch_backward(WindowArgs& a, const KeyPlan& p, hipStream_t st) {
  typedef KeyTile<T, DP> KT;
  int s;
  const int64_t heads = (int64_t)a.batch * a.key_heads, rows = (int64_t)a.queries * a.group;
  AFHIP_REQUIRE(p.tile_keys == KT::kKeys, "key tiles of %d keys, not %d", KT::kKeys, p.tile_keys);
  const int parts = (int)ceil_div(2 * KT::kKeys * a.head_dim, 1024);
  if ((s = check_grid(p.groups(heads), KT::kThreads)) || (s = check_grid(heads * p.joined() * parts, 256))) return s;
  if ((s = launch_dq_any<T, DP>(a, heads, rows, st))) return s;
  a.tiles = p.tiles;
  a.chunks = p.chunks;
  a.chunk_rows = p.chunk_rows;
  a.sink_rows = p.sink_rows;
  a.long_tiles = p.long_tiles;
  a.short_chunks = p.short_chunks;
  a.parts = (int)p.parts();
  auto kkv = window_dkv_kernel<T, DP>;
  if ((s = allow_lds((const void*)kkv, KT::kLds))) return s;
  if ((s = launch("window.dkv", kkv, dim3((unsigned)p.groups(heads)), dim3(KT::kThreads), KT::kLds, st, a)))
    return s;
  return launch("window.dkv_join", window_dkv_join_kernel<T>, dim3((unsigned)(heads * p.joined() * parts)), dim3(256),
                0, st, a, KT::kKeys, parts);
}

template <typename T> int launch_width(WindowArgs& a, const KeyPlan& p, hipStream_t st) {
  if (a.head_dim <= 32) return launch_backward<T, 32>(a, p, st);
  if (a.head_dim <= 64) return launch_backward<T, 64>(a, p, st);
  return launch_backward<T, 128>(a, p, st);
}

size_t row_bytes(const afhip_window_desc& d) {
  return (size_t)round_up((int64_t)d.batch * d.queries * d.query_heads * 8, 256);
}

}  // namespace

}  // namespace afhip

using namespace afhip;

extern "C" {

int afhip_window_backward_workspace_size(const afhip_window_desc* desc, size_t* bytes) {
  if (int s = window_check(desc)) return s;
  AFHIP_REQUIRE(bytes != nullptr, "output is NULL");
  *bytes = 2 * row_bytes(*desc) + chunk_bytes(*desc, key_plan(*desc));
  return AFHIP_OK;
}

int afhip_window_backward(const afhip_window_desc* desc, const void* q, const void* k, const void* v, const void* out,
                          const float* lse, const void* dout, const afhip_strides* dout_strides,
                          const int32_t* query_lengths, const int32_t* key_lengths, void* dq, void* dk, void* dv,
                          void* workspace, size_t workspace_bytes, void* stream) {
  int s;
  size_t need = 0;
  if ((s = require_open()) || (s = afhip_window_backward_workspace_size(desc, &need))) return s;
  const afhip_window_desc& d = *desc;
  WindowArgs a{};
  window_fill(d, a);
  AFHIP_REQUIRE(dout_strides != nullptr, "the strides of dout are NULL");
  a.sdo = head_strides(*dout_strides, d.queries, d.query_heads, d.head_dim, d.dtype);
  if ((s = check_strides("dout", a.sdo, d.batch, d.queries, d.query_heads, d.head_dim, d.dtype, false)) ||
      (s = check_address("q", q)) || (s = check_address("k", k)) || (s = check_address("v", v)) ||
      (s = check_address("out", out)) || (s = check_address("dout", dout)) || (s = check_address("dq", dq)) ||
      (s = check_address("dk", dk)) || (s = check_address("dv", dv)))
    return s;
  // Rows of a block lie within a buffer's 2 GiB: 65 queries, and the group's heads beside them.
  for (const HeadStrides* x : {&a.sq, &a.sdo})
    AFHIP_REQUIRE(65 * x->token + (int64_t)a.group * x->head < ((int64_t)1 << 31),
                  "the heads of a group are more than 2 GiB apart");
  AFHIP_REQUIRE(lse != nullptr, "lse is NULL");
  AFHIP_REQUIRE(workspace && workspace_bytes >= need, "workspace of %zu bytes is smaller than %zu", workspace_bytes,
                need);
  if ((s = check_address("workspace", workspace))) return s;
  a.q = (const char*)q;
  a.k = (const char*)k;
  a.v = (const char*)v;
  a.o = (const char*)out;
  a.lse = const_cast<float*>(lse);
  a.dout = (const char*)dout;
  a.query_lengths = query_lengths;
  a.key_lengths = key_lengths;
  a.dq = (char*)dq;
  a.dk = (char*)dk;
  a.dv = (char*)dv;
  a.rows = (float2*)workspace;
  a.limits = (int2*)((char*)workspace + row_bytes(d));
  a.partial = (float*)((char*)workspace + 2 * row_bytes(d));
  const KeyPlan p = key_plan(d);
  hipStream_t st = (hipStream_t)stream;
  return d.dtype == AFHIP_F16 ? launch_width<half_t>(a, p, st) : launch_width<float>(a, p, st);
}

}  // extern "C"
