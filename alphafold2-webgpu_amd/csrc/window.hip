// Attention over a window of keys and the first few ("sinks"), for prompts and
// for single tokens against a cache:
//
//   p = key_length - query_length + i;  key j is seen iff j < key_length, j <= p + right, and j >= p - left or
//   j < sinks
//   out = sum_j e^(s_j - m) v_j / l,  l = sum_j e^(s_j - m),  lse = m + ln l,  s_j = scale q . k_j
//
// in one pass over the keys with a running reference point m. Query heads that
// share a key head are rows of one tile: row r of a key head is query r / group
// of head r % group, so that a tile reads each key once for all of them.
//
// Both products run on the MFMA as S^T = K Q^T and O^T = V^T P^T: a lane then
// holds one row's scores for 16 keys and the same row's output for 16 channels,
// the reference point and the sum stay inside the lane (and the lane 32 away),
// and the probabilities feed the second product from the registers they were
// computed in. K and V go to LDS by DMA; V^T comes from gfx950's transposing LDS
// read. f32 runs the same, its values as three bf16 each.
//
// Blocks of keys that no query of a workgroup sees are not visited, rows of one
// that none sees are loaded as zeros (whatever is there, infinities and NaN too),
// and the comparisons run only in blocks that some row sees in part.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "window.h"

namespace afhip {

namespace {

// A probability is held as 2^(x - m + kLift), in f16 within 2^-24 and 2^(kLift + kSlack): the reference point m moves
// only when a score passes it by more than kSlack, and small probabilities of long rows keep their bits.
template <typename T> constexpr float kLift = sizeof(T) == 2 ? 6.0f : 0.0f;
constexpr float kSlack = 8.0f;

// f32 over 128 channels just fits the 256 registers that each of eight waves has, where no fragments are read far
// ahead: two workgroups of four waves a CU. 2,000 tokens, 32 heads over 8, in 500 workgroups, us, two / one a CU: no
// mask 347 / 430, window 300 71 / 97; but 352 workgroups, causal, 97 / 86, since a CU gets its second before others
// have one.
template <typename T, int DP> constexpr bool kWide = DP * sizeof(T) > 256;

// One wave's 32 rows: Q, the running state and the output so far.
template <typename T, int DP> struct Rows {
  typedef typename Eight<T>::type Frag;
  static constexpr int kSteps = DP / 16, kBlocks = DP / 32;
  Frag q[kSteps];
  floatx16 o[kBlocks];
  float m, l;
  int high, low;  // what this lane's row sees

  __device__ __forceinline__ void init(const WindowArgs& a, const Sequence& s, int b, int kv, int row, int hi) {
    const int i = row / a.group, h = kv * a.group + row % a.group;
    const bool live = i < s.queries;
    const char* p = a.q + b * a.sq.batch + (int64_t)(live ? i : 0) * a.sq.token + h * a.sq.head;
#pragma unroll
    for (int kk = 0; kk < kSteps; kk++) {
      const int ch = 16 * kk + 8 * hi;
      q[kk] = as_fragment(load_eight(reinterpret_cast<const T*>(p) + ch, live && ch < a.head_dim));
    }
#pragma unroll
    for (int c = 0; c < kBlocks; c++) o[c] = floatx16{};
    m = -INFINITY;
    l = 0.0f;
    // A row past the length counts as the last one (its results are dropped), so that it makes no block partial.
    const int at = min(i, s.queries - 1);
    high = s.high(a, at);
    low = s.low(a, at);
  }

  // 32 NB keys from k0 on: K and V tiles at kt and vt; ends and starts: see hide().
  template <typename Read, int NB>
  __device__ __forceinline__ void step(const unsigned char* kt, const unsigned char* vt, int k0, bool ends, bool starts,
                                       int sinks, float scale, int lane) {
    const int col = lane & 31, hi = lane >> 5;
    floatx16 x[NB];
#pragma unroll
    for (int n = 0; n < NB; n++) {
      x[n] = floatx16{};
#pragma unroll
      for (int kk = 0; kk < kSteps; kk++) {
        x[n] = mma(Read::nat(kt, 32 * n + col, kk, hi), q[kk], x[n]);
        if (kWide<T, DP> && kk % 2) __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (ends | starts) {
#pragma unroll
      for (int n = 0; n < NB; n++) hide(k0 + 32 * n, lane, low, high, sinks, ends, starts, -INFINITY, x[n]);
    }
    float top = x[0][0];
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int v = 0; v < 16; v++) top = fmaxf(top, x[n][v]);
    top *= scale;
    if (__builtin_amdgcn_ballot_w64(top > m + kSlack)) {
      const float to = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
      const float f = to == m ? 1.0f : __builtin_amdgcn_exp2f(m - to);
      l *= f;
#pragma unroll
      for (int c = 0; c < kBlocks; c++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[c][v] *= f;
      m = to;
    }
    const float offset = kLift<T> - (m == -INFINITY ? 0.0f : m);
#pragma unroll
    for (int n = 0; n < NB; n++) {
      float p[16];
#pragma unroll
      for (int v = 0; v < 16; v++) p[v] = __builtin_amdgcn_exp2f(fmaf(x[n][v], scale, offset));
      // Before they are rounded: lse keeps 32 bits.
      l += (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]))) +
           (((p[8] + p[9]) + (p[10] + p[11])) + ((p[12] + p[13]) + (p[14] + p[15])));
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const Frag f = pack8(p + 8 * s, (Frag*)nullptr);
#pragma unroll
        for (int c = 0; c < kBlocks; c++) {
          o[c] = mma(Read::tr(vt, 32 * n + 16 * s, c, lane), f, o[c]);
          if (kWide<T, DP>) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
};

// The natural logarithm of a row's sum, from its reference point and total (both in base 2).
template <typename T> __device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.0f ? -INFINITY : (m - kLift<T> + log2f(l)) * kWindowLn2;
}

__device__ __forceinline__ int64_t lse_index(const WindowArgs& a, int b, int h, int i) {
  return ((int64_t)b * a.query_heads + h) * a.queries + i;
}

constexpr int kJoinRows = 8;  // of a workgroup of window_join_kernel, which takes up to 64 splits

// The reference points and totals of split keys, behind their sums.
__device__ __forceinline__ float2* part_totals(const WindowArgs& a) {
  return reinterpret_cast<float2*>(a.partial + (int64_t)a.batch * a.queries * a.query_heads * a.splits * a.head_dim);
}

// Four waves of 32 rows, or with PARTS = 2 eight, of which the second four take the second half of every block: where
// there are few tiles, twice the waves for the same reads of K and V, and their sums meet in LDS.
// MFMA bounds it, and the softmax's vector instructions, which a SIMD's two waves issue beside each other's MFMAs:
// 4,096 tokens, 32 heads over 8 of 128 channels, causal, f16, 150 us, 910 TFLOP/s of the 1,190 of a large product;
// window 1,024 over 16,384 tokens, 8 heads over 2, 87 us.
constexpr int kWaves = 4, kTileRows = 32 * kWaves;
template <typename T> constexpr int kBlockKeys = sizeof(T) == 2 ? 64 : 32;  // a wave's, of a block
// f32 blocks are loaded into one buffer and made three bf16 from there, once for all waves.
template <typename T, int DP, int PARTS>
constexpr int kRowsLds = (sizeof(T) == 2 ? 8 : 20) * PARTS * kBlockKeys<T> * DP;

template <typename T, int DP, bool SPLIT, int PARTS>
__global__ __launch_bounds__(64 * kWaves * PARTS, PARTS == 2 ? 1 : 2) void window_rows_kernel(
    WindowArgs a) {
  constexpr int WK = kBlockKeys<T>, BK = WK * PARTS;
  constexpr bool F32 = sizeof(T) == 4;
  typedef TileLoad<T, DP, BK, kWaves * PARTS> Load;
  typedef Planes<DP, BK> Split;
  typedef typename std::conditional<F32, Split, Tile<T, DP>>::type Read;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  prefer_one_of_two();
  const int lane = threadIdx.x & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wave % kWaves, part = wave / kWaves;
  // Neighbours are other key heads (with 8 of them or a multiple, a head's workgroups share an XCD's L2), the last
  // rows first: without a window they see the most keys.
  const int heads = a.batch * a.key_heads;
  const int pair = blockIdx.x % heads, rest = blockIdx.x / heads;
  const int b = pair / a.key_heads, kv = pair % a.key_heads;
  const int turn = rest % a.tiles, split = rest / a.tiles, half = (a.tiles + 1) / 2;
  // Where all run at once, two a CU, the second ones from the shortest on.
  const bool second = kWide<T, DP> && gridDim.x <= 512 && (SPLIT ? 2 * split >= a.splits : turn >= half);
  const int tile = second ? (SPLIT ? turn : turn - half) : a.tiles - 1 - turn;
  const Sequence s(a, b);
  const int rows = a.queries * a.group;
  const int r0 = tile * kTileRows;
  const int first = r0 / a.group, last = min(s.queries - 1, (r0 + kTileRows - 1) / a.group);

  const KeyRange range(a, s, first, last, BK);
  const int total = first < s.queries ? range.total : 0;
  const int begin = SPLIT ? (int)((int64_t)total * split / a.splits) : 0;
  const int end = SPLIT ? (int)((int64_t)total * (split + 1) / a.splits) : total;
  // What the wave's rows all see, and what any of them sees.
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
    const uint32_t buffer = lds + (F32 ? 0u : (uint32_t)((t - begin) & 1) * 2 * Load::kBytes);
    const bool whole = range.whole(k0, BK);
    auto keep = [&](int key) { return range.keeps(key); };
    kload.issue(kb, a.sk.token, k0, buffer, wave, whole, keep);
    vload.issue(vb, a.sv.token, k0, buffer + Load::kBytes, wave, whole, keep);
  };
  // Block t is the only one in flight; the barrier publishes it, and every wave is done with block t - 1.
  auto arrive = [&](int t) {
    wait_vmcnt<0>();
    block_barrier();
    if constexpr (F32) {
      Split::template split_two<64 * kWaves * PARTS>(smem, smem + 2 * Load::kBytes);
      block_barrier();  // written, and the buffer is read
    }
    if (t + 1 < end) issue(t + 1);
  };
  // The first keys are on their way before the queries.
  if (begin < end) issue(begin);
  Rows<T, DP> st;
  st.init(a, s, b, kv, r0 + 32 * rg + (lane & 31), hi);
  // Blocks that the wave's rows see, between such that only other waves' do. (A branch around the work of one loop
  // would have the compiler copy all sums at its end.)
  const auto phases = range.phases(begin, end, BK, s.low(a, wfirst), s.high(a, wlast), wr0 < s.queries * a.group);
  int t = begin;
#pragma unroll 1
  for (int phase = 0; phase < 2; phase++) {
    const int work = phase ? phases.to : phases.sink_end, idle = phase ? end : phases.from;
    for (; t < work; t++) {
      arrive(t);
      const int at = WK * part, k0 = range.block(t) * BK + at;
      const unsigned char* kt = F32 ? smem + 2 * Load::kBytes + at * DP * 2
                                    : smem + ((t - begin) & 1) * 2 * Load::kBytes + at * DP * 2;
      const unsigned char* vt = kt + (F32 ? Split::kBytes : Load::kBytes);
      st.template step<Read, WK / 32>(kt, vt, k0, k0 + WK > all_high, k0 < all_low && k0 + WK > range.sinks,
                                range.sinks, a.scale_log2, lane);
    }
    for (; t < idle; t++) arrive(t);
  }
  if constexpr (PARTS == 2) {
    constexpr int VALUES = 2 + DP / 2;
    static_assert(kWaves * VALUES * 256 <= kRowsLds<T, DP, PARTS>, "the second part's sums fit");
    float* shared = reinterpret_cast<float*>(smem) + rg * VALUES * 64 + lane;
    block_barrier();  // the last block is read
    if (part == 1) {
      shared[0] = st.m;
      shared[64] = st.l;
#pragma unroll
      for (int c = 0; c < DP / 32; c++)
#pragma unroll
        for (int v = 0; v < 16; v++) shared[(2 + 16 * c + v) * 64] = st.o[c][v];
    }
    block_barrier();
    if (part == 1) return;
    const float other = shared[0], m = fmaxf(st.m, other);
    const float f = st.m == m ? 1.0f : __builtin_amdgcn_exp2f(st.m - m);
    const float g = other == m ? 1.0f : __builtin_amdgcn_exp2f(other - m);
    st.m = m;
    st.l = st.l * f + shared[64] * g;
#pragma unroll
    for (int c = 0; c < DP / 32; c++)
#pragma unroll
      for (int v = 0; v < 16; v++) st.o[c][v] = st.o[c][v] * f + shared[(2 + 16 * c + v) * 64] * g;
  }
  const float l = st.l + __shfl_xor(st.l, 32);
  int row = threadIdx.x;
  asm volatile("" : "+v"(row));  // computed here, not held from the start
  row = r0 + 32 * rg + (row & 31);
  if (row >= rows) return;
  const int i = row / a.group, h = kv * a.group + row % a.group;
  if constexpr (SPLIT) {
    const int64_t n = ((int64_t)pair * rows + row) * a.splits + split;
    float* to = a.partial + n * a.head_dim;
#pragma unroll
    for (int c = 0; c < DP / 32; c++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int ch = 32 * c + 8 * g + 4 * hi;
        if (ch >= a.head_dim) continue;
        const floatx16& o = st.o[c];
        put4(to + ch, o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
      }
    if (!hi) part_totals(a)[n] = float2{st.m, l};
  } else {
    const bool live = i < s.queries && l != 0.0f;
    const float inv = 1.0f / l;
    T* to = reinterpret_cast<T*>(a.out + b * a.so.batch + i * a.so.token + h * a.so.head);
#pragma unroll
    for (int c = 0; c < DP / 32; c++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int ch = 32 * c + 8 * g + 4 * hi;
        if (ch >= a.head_dim) continue;
        const floatx16& o = st.o[c];
        if (live) {
          put4(to + ch, o[4 * g] * inv, o[4 * g + 1] * inv, o[4 * g + 2] * inv, o[4 * g + 3] * inv);
        } else {
          put4(to + ch, 0.0f, 0.0f, 0.0f, 0.0f);
        }
      }
    if (a.lse && !hi) a.lse[lse_index(a, b, h, i)] = live ? row_lse<T>(st.m, l) : -INFINITY;
  }
}

// 32 rows of a key head (single tokens, few of them, or where tiles of 128 rows would leave most CUs without work): its
// waves take blocks of 32 keys in turn, each through buffers of its own, with no barrier until the end, where their
// sums meet in LDS. For single tokens the cache's bytes bound it; a split adds workgroups until they fill the card. 4
// sequences of 32,768 keys, 8 heads of 128 channels, f16: 85 us, 4.95 TB/s; 16 of 1,028 visible ones, one workgroup on
// every second CU, 18.8 us, 3.6 TB/s.
template <typename T, int DP> struct Step {
  static constexpr int kBytes = 2 * 32 * DP * (int)sizeof(T);  // K and V of a block
  static constexpr int kWaves = 4;
  // Four waves with one buffer each where two fill the LDS with two: 16 sequences of 4,000 keys, 8 heads of 128
  // channels, f32, 131 us and 156; 2 of 195, 11 and 19.
  static constexpr int kStages = kBytes >= 32768 ? 1 : kBytes >= 16384 ? 2 : 4;
  static constexpr int kLds = kWaves * kStages * kBytes;
  static_assert(kLds >= kWaves * 32 * (DP + 2) * 4, "the waves' sums fit");
};

template <typename T, int DP> constexpr int kStepThreads = 64 * Step<T, DP>::kWaves;

template <typename T, int DP>
__global__ __launch_bounds__((kStepThreads<T, DP>)) void window_step_kernel(WindowArgs a) {
  typedef Step<T, DP> S;
  constexpr int W = S::kWaves, STAGES = S::kStages;
  typedef TileLoad<T, DP, 32, 1> Load;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x & 63, hi = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = a.batch * a.key_heads;
  const int pair = blockIdx.x % heads, rest = blockIdx.x / heads;
  const int tile = a.tiles - 1 - rest % a.tiles, split = rest / a.tiles;
  const int b = pair / a.key_heads, kv = pair % a.key_heads;
  const Sequence s(a, b);
  const int all = a.queries * a.group, r0 = 32 * tile, rows = min(32, all - r0);
  const int first = r0 / a.group, last = min(s.queries - 1, (r0 + rows - 1) / a.group);
  Rows<T, DP> st;
  st.init(a, s, b, kv, r0 + min(col, rows - 1), hi);
  const KeyRange range(a, s, first, last, 32);
  const int total = first < s.queries ? range.total : 0;
  const int begin = (int)((int64_t)total * split / a.splits);
  const int end = (int)((int64_t)total * (split + 1) / a.splits);
  const int all_low = s.low(a, last), all_high = s.high(a, first);
  const char* kb = a.k + b * a.sk.batch + kv * a.sk.head;
  const char* vb = a.v + b * a.sv.batch + kv * a.sv.head;
  const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>(smem) + wave * STAGES * S::kBytes;
  Load kload, vload;
  kload.init(0, lane, a.head_dim, a.sk.token);
  vload.init(0, lane, a.head_dim, a.sv.token);
  const int mine = begin + wave < end ? (end - begin - wave + W - 1) / W : 0;
  auto issue = [&](int n) {
    const int k0 = range.block(begin + wave + n * W) * 32;
    const uint32_t buffer = lds + (uint32_t)(n % STAGES) * S::kBytes;
    const bool whole = range.whole(k0, 32);
    auto keep = [&](int key) { return range.keeps(key); };
    kload.issue(kb, a.sk.token, k0, buffer, 0, whole, keep);
    vload.issue(vb, a.sv.token, k0, buffer + S::kBytes / 2, 0, whole, keep);
  };
#pragma unroll 1
  for (int n = 0; n < STAGES - 1 && n < mine; n++) issue(n);
  for (int n = 0; n < mine; n++) {
    // The buffer that block n + STAGES - 1 goes to was read by step n - 1, whose reads have returned.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (n + STAGES - 1 < mine) {
      issue(n + STAGES - 1);
      wait_vmcnt<2 * Load::kCount * (STAGES - 1)>();
    } else {
      wait_vmcnt<0>();
    }
    const int k0 = range.block(begin + wave + n * W) * 32;
    const unsigned char* kt = smem + (wave * STAGES + n % STAGES) * S::kBytes;
    st.template step<Tile<T, DP>, 1>(kt, kt + S::kBytes / 2, k0, k0 + 32 > all_high,
                                     k0 < all_low && k0 + 32 > range.sinks, range.sinks, a.scale_log2, lane);
  }
  // The waves' reference points, totals and sums: [wave][row][m, l, DP sums].
  float* sums = reinterpret_cast<float*>(smem);
  const float l = st.l + __shfl_xor(st.l, 32);
  block_barrier();  // every wave's loads have landed and been read
  constexpr int PITCH = DP + 2;
  float* own = sums + (wave * 32 + col) * PITCH;
  if (col < rows) {
    if (!hi) own[0] = st.m, own[1] = l;
#pragma unroll
    for (int c = 0; c < DP / 32; c++)
#pragma unroll
      for (int v = 0; v < 16; v++) own[2 + 32 * c + mfma_row(v, lane)] = st.o[c][v];
  }
  block_barrier();
  for (int n = threadIdx.x; n < rows * DP; n += 64 * W) {
    const int r = n / DP, ch = n % DP;
    if (ch >= a.head_dim) continue;
    float m = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) m = fmaxf(m, sums[(w * 32 + r) * PITCH]);
#pragma unroll
    for (int w = 0; w < W; w++) {
      const float* p = sums + (w * 32 + r) * PITCH;
      const float f = p[0] == m ? 1.0f : __builtin_amdgcn_exp2f(p[0] - m);
      sum += f * p[1];
      o += f * p[2 + ch];
    }
    const int i = (r0 + r) / a.group, h = kv * a.group + (r0 + r) % a.group;
    if (a.splits > 1) {
      const int64_t to = ((int64_t)pair * all + r0 + r) * a.splits + split;
      a.partial[to * a.head_dim + ch] = o;
      if (ch == 0) part_totals(a)[to] = float2{m, sum};
    } else {
      const bool live = i < s.queries;
      T* to = reinterpret_cast<T*>(a.out + b * a.so.batch + i * a.so.token + h * a.so.head);
      to[ch] = (T)(live && sum != 0.0f ? o / sum : 0.0f);
      if (ch == 0 && a.lse) a.lse[lse_index(a, b, h, i)] = live ? row_lse<T>(m, sum) : -INFINITY;
    }
  }
}

// Joins the splits of a row, half a wave a row and four channels a lane: 4 us, a launch's least, for single tokens;
// 4.8 for 8,192 rows of 4 parts, 17 MB.
template <typename T> __global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * kJoinRows + (threadIdx.x >> 5), rows = (int64_t)a.queries * a.group;
  if (n >= (int64_t)a.batch * a.key_heads * rows) return;
  const int pair = (int)(n / rows), row = (int)(n % rows);
  const int b = pair / a.key_heads, kv = pair % a.key_heads, i = row / a.group, h = kv * a.group + row % a.group;
  const Sequence s(a, b);
  // Two splits a lane; past the last one a total of 0.
  const float2* totals = part_totals(a) + n * a.splits;
  float2 mine[2];
#pragma unroll
  for (int j = 0; j < 2; j++) {
    mine[j] = totals[min(lane + 32 * j, a.splits - 1)];
    if (lane + 32 * j >= a.splits) mine[j] = float2{-INFINITY, 0.0f};
  }
  float m = fmaxf(mine[0].x, mine[1].x);
#pragma unroll
  for (int step = 1; step < 32; step *= 2) m = fmaxf(m, __shfl_xor(m, step));
  float f[2], total = 0.0f;
#pragma unroll
  for (int j = 0; j < 2; j++) {
    f[j] = lane + 32 * j >= a.splits ? 0.0f : mine[j].x == m ? 1.0f : __builtin_amdgcn_exp2f(mine[j].x - m);
    total += f[j] * mine[j].y;
  }
#pragma unroll
  for (int step = 1; step < 32; step *= 2) total += __shfl_xor(total, step);
  // Eight parts' loads at once; past the last part its own again, with a weight of 0.
  const int ch = min(4 * lane, a.head_dim - 4);
  const float* from = a.partial + n * a.splits * a.head_dim + ch;
  floatx4 o{};
  for (int k0 = 0; k0 < a.splits; k0 += 8) {
    floatx4 x[8];
#pragma unroll
    for (int k = 0; k < 8; k++)
      x[k] = *reinterpret_cast<const floatx4*>(from + (int64_t)min(k0 + k, a.splits - 1) * a.head_dim);
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const float w = __shfl(k0 < 32 ? f[0] : f[1], (k0 + k) & 31, 32);
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] += w * x[k][j];
    }
  }
  const bool live = i < s.queries && total != 0.0f;
  if (4 * lane < a.head_dim) {
    T* to = reinterpret_cast<T*>(a.out + b * a.so.batch + i * a.so.token + h * a.so.head) + ch;
    put4(to, live ? o[0] / total : 0.0f, live ? o[1] / total : 0.0f, live ? o[2] / total : 0.0f,
         live ? o[3] / total : 0.0f);
  }
  if (lane == 0 && a.lse) a.lse[lse_index(a, b, h, i)] = live ? row_lse<T>(m, total) : -INFINITY;
}

// Which kernel a call takes, and into how many parts its keys are split.
struct Plan {
  bool step;
  int parts;  // of a block of keys, in a workgroup: window_rows_kernel
  int tiles, splits;
};

Plan plan(const afhip_window_desc& d) {
  const bool f32 = d.dtype == AFHIP_F32;
  const int64_t group = d.query_heads / d.key_heads, rows = d.queries * group, heads = (int64_t)d.batch * d.key_heads;
  Plan p{};
  // Tiles of 32 rows also where those of 128 are few. Whole calls on MI355X, tiles of 128 / 32, us: f32 over 32
  // channels 128 tiles 15.9 / 10.1, 256 tiles 17.8 / 32; over 64 40 tiles 28 / 20, 64 tiles 35 / 37; over 128 40 tiles
  // 33 / 34, 112 tiles 33 / 43; f16 over 64 channels 2 tiles 10.5 / 8.9, 128 tiles 12.7 / 16.5; over 128 20 tiles
  // 12.2 / 13.6.
  const int64_t few = f32 ? (d.head_dim <= 32 ? 256 : 64) : d.head_dim <= 64 ? 64 : 0;
  p.step = rows <= 32 || heads * ceil_div(rows, kTileRows) < few;
  p.tiles = (int)ceil_div(rows, p.step ? 32 : kTileRows);
  const int64_t groups = heads * p.tiles;
  // Eight waves for every CU.
  p.parts = !p.step && groups < 1024 && !(f32 && d.head_dim > 64) ? 2 : 1;
  // The most keys that a tile's queries see.
  int64_t span = d.keys;
  if (d.left >= 0) {
    const int64_t queries = std::min<int64_t>(d.queries, ceil_div(p.step ? 32 : kTileRows, group) + 1);
    const int64_t right = d.right < 0 ? d.keys : d.right;
    span = std::min(span, (int64_t)d.left + right + queries + std::min<int64_t>(d.sinks, d.keys));
  }
  // Into how many parts the keys are split: the shortest of some, by what they take on MI355X in us. A block of 32 keys
  // takes a workgroup 0.4 (f16, 128 channels; f32 2.6, of four waves with keys of their own 1.2), a workgroup's start
  // and end 4, a CU having one of them at a time; the keys' bytes come at 5.3 TB/s where all CUs ask for them, at 4
  // where half do; the join takes 4.5, and its sums go out and in at 3.5 TB/s.
  const double block = std::max((!f32 ? 0.4 : p.step ? 1.2 : 2.6) * d.head_dim / 128, 0.15);
  const double bytes = 2.0 * heads * span * d.head_dim * dtype_size(d.dtype);
  double best = INFINITY;
  for (int64_t splits : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
    const int64_t blocks = ceil_div(span, 32), all = groups * splits;
    if (splits > 1 && (blocks < 4 * splits || all > 1024)) break;
    double time = ceil_div(all, p.parts == 2 || p.step ? 256 : 512) * (4 + block * ceil_div(blocks, splits));
    if (p.step) time = std::max(time, bytes / 5.3e6 * std::pow(std::max(1.0, 256.0 / all), 0.4));
    if (splits > 1) time += 4.5 + (double)heads * rows * splits * d.head_dim * 8 / 3.5e6;
    if (time < best) best = time, p.splits = (int)splits;
  }
  return p;
}

size_t partial_bytes(const afhip_window_desc& d, const Plan& p) {
  if (p.splits == 1) return 0;
  return (size_t)d.batch * d.queries * d.query_heads * p.splits * (d.head_dim + 2) * sizeof(float);
}

template <typename T, int DP, int PARTS>
int launch_rows(const WindowArgs& a, const Plan& p, int64_t groups, hipStream_t st) {
  // Half of the LDS and more: one a CU.
  const size_t lds = kRowsLds<T, DP, PARTS> + (kWide<T, DP> && groups < 448 ? 1024 : 0);
  auto k = p.splits > 1 ? window_rows_kernel<T, DP, true, PARTS> : window_rows_kernel<T, DP, false, PARTS>;
  int s;
  if ((s = check_grid(groups, 64 * kWaves * PARTS)) || (s = allow_lds((const void*)k, lds))) return s;
  return launch("window.rows", k, dim3((unsigned)groups), dim3(64 * kWaves * PARTS), lds, st, a);
}

template <typename T, int DP> int launch_forward(const WindowArgs& a, const Plan& p, hipStream_t st) {
  int s;
  const int64_t groups = (int64_t)a.batch * a.key_heads * p.tiles * p.splits;
  if (p.step) {
    typedef Step<T, DP> S;
    auto k = window_step_kernel<T, DP>;
    if ((s = check_grid(groups, 64 * S::kWaves)) || (s = allow_lds((const void*)k, S::kLds))) return s;
    s = launch("window.step", k, dim3((unsigned)groups), dim3(64 * S::kWaves), S::kLds, st, a);
  } else {
    s = p.parts == 2 ? launch_rows<T, DP, kWide<T, DP> ? 1 : 2>(a, p, groups, st)
                     : launch_rows<T, DP, 1>(a, p, groups, st);
  }
  if (s || p.splits == 1) return s;
  const int64_t rows = (int64_t)a.batch * a.queries * a.query_heads;
  if ((s = check_grid(ceil_div(rows, kJoinRows), 256))) return s;
  return launch("window.join", window_join_kernel<T>, dim3((unsigned)ceil_div(rows, kJoinRows)), dim3(256), 0, st, a);
}

template <typename T> int launch_width(const WindowArgs& a, const Plan& p, hipStream_t st) {
  if (a.head_dim <= 32) return launch_forward<T, 32>(a, p, st);
  if (a.head_dim <= 64) return launch_forward<T, 64>(a, p, st);
  return launch_forward<T, 128>(a, p, st);
}

}  // namespace

int window_check(const afhip_window_desc* desc) {
  AFHIP_REQUIRE(desc != nullptr, "descriptor is NULL");
  const afhip_window_desc& d = *desc;
  AFHIP_REQUIRE(d.batch > 0 && d.queries > 0 && d.keys > 0 && d.query_heads > 0 && d.key_heads > 0 && d.head_dim > 0,
                "attention dimensions must be positive");
  AFHIP_REQUIRE(d.head_dim % 8 == 0 && d.head_dim <= kMaxHeadDim, "head dimension %d is not a multiple of 8 up to %d",
                d.head_dim, kMaxHeadDim);
  AFHIP_REQUIRE(d.query_heads % d.key_heads == 0, "%d query heads over %d key heads", d.query_heads, d.key_heads);
  AFHIP_REQUIRE(d.left >= -1 && d.right >= -1 && d.sinks >= 0, "left and right are at least -1, sinks at least 0");
  AFHIP_REQUIRE(valid_float_dtype(d.dtype), "attention dtype must be f32 or f16");
  AFHIP_REQUIRE(d.scale > 0.0f && d.scale < INFINITY, "scale must be positive and finite");
  constexpr int64_t most = (int64_t)1 << 30;
  AFHIP_REQUIRE(d.keys < most && (int64_t)d.queries * d.query_heads < most && d.query_heads <= 65536,
                "more than 2^30 keys or queries of a sequence, or 65,536 heads");
  AFHIP_REQUIRE((int64_t)d.batch * d.key_heads < most, "batch times heads passes 2^30");
  WindowArgs a{};
  window_fill(d, a);
  int s;
  if ((s = check_strides("q", a.sq, d.batch, d.queries, d.query_heads, d.head_dim, d.dtype, false)) ||
      (s = check_strides("k", a.sk, d.batch, d.keys, d.key_heads, d.head_dim, d.dtype, false)) ||
      (s = check_strides("v", a.sv, d.batch, d.keys, d.key_heads, d.head_dim, d.dtype, false)) ||
      (s = check_strides("out", a.so, d.batch, d.queries, d.query_heads, d.head_dim, d.dtype, true)))
    return s;
  return AFHIP_OK;
}

void window_fill(const afhip_window_desc& d, WindowArgs& a) {
  constexpr int most = 1 << 30;  // more than any position: sums of two stay within 32 bits
  a.sq = head_strides(d.q, d.queries, d.query_heads, d.head_dim, d.dtype);
  a.sk = head_strides(d.k, d.keys, d.key_heads, d.head_dim, d.dtype);
  a.sv = head_strides(d.v, d.keys, d.key_heads, d.head_dim, d.dtype);
  a.so = head_strides(d.out, d.queries, d.query_heads, d.head_dim, d.dtype);
  a.batch = d.batch;
  a.queries = d.queries;
  a.keys = d.keys;
  a.query_heads = d.query_heads;
  a.key_heads = d.key_heads;
  a.group = d.query_heads / d.key_heads;
  a.head_dim = d.head_dim;
  a.left = d.left >= most ? -1 : d.left;
  a.right = d.right >= most ? -1 : d.right;
  a.sinks = std::min(d.sinks, most);
  a.scale = d.scale;
  a.scale_log2 = d.scale * kWindowLog2e;
}

}  // namespace afhip

using namespace afhip;

extern "C" {

int afhip_window_workspace_size(const afhip_window_desc* desc, size_t* bytes) {
  if (int s = window_check(desc)) return s;
  AFHIP_REQUIRE(bytes != nullptr, "output is NULL");
  *bytes = partial_bytes(*desc, plan(*desc));
  return AFHIP_OK;
}

int afhip_window_run(const afhip_window_desc* desc, const void* q, const void* k, const void* v,
                     const int32_t* query_lengths, const int32_t* key_lengths, void* out, float* lse, void* workspace,
                     size_t workspace_bytes, void* stream) {
  int s;
  if ((s = require_open()) || (s = window_check(desc))) return s;
  const afhip_window_desc& d = *desc;
  WindowArgs a{};
  window_fill(d, a);
  if ((s = check_address("q", q)) || (s = check_address("k", k)) || (s = check_address("v", v)) ||
      (s = check_address("out", out)))
    return s;
  const Plan p = plan(d);
  const size_t need = partial_bytes(d, p);
  if (need) {
    AFHIP_REQUIRE(workspace && workspace_bytes >= need, "workspace of %zu bytes is smaller than %zu", workspace_bytes,
                  need);
    if ((s = check_address("workspace", workspace))) return s;
  }
  a.q = (const char*)q;
  a.k = (const char*)k;
  a.v = (const char*)v;
  a.out = (char*)out;
  a.lse = lse;
  a.query_lengths = query_lengths;
  a.key_lengths = key_lengths;
  a.partial = (float*)workspace;
  a.tiles = p.tiles;
  a.splits = p.splits;
  hipStream_t st = (hipStream_t)stream;
  return d.dtype == AFHIP_F16 ? launch_width<half_t>(a, p, st) : launch_width<float>(a, p, st);
}

}  // extern "C"
