// The projection in 8-bit integers: y = act(s_m s_n sum_k q_mk w_nk + b_n) with whole numbers
// q = rint(x * (127 / m)) of each row of x, its scale s_m = m / 127 (m the row's largest
// magnitude), and a weight w with a scale s_n for each output channel.
//
// Sums of products are exact in 32-bit integers up to K = 131072 (127^2 K < 2^31), so neither the
// order of a sum nor its split changes a result: what is rounded is q, and the three float32
// operations of the last step.

#include <type_traits>

#include "lanes.h"

namespace {

using namespace spmi;

using i32x4 = int __attribute__((ext_vector_type(4)));
using i32x16 = int __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
// Operand of s_waitcnt: at most n vector memory operations outstanding, other counters free.
#define WAIT_LOADS(n) (((n) & 15) | ((n) >> 4 << 14) | (7 << 4) | (15 << 8))
// The same for LDS: all reads have returned.
#define WAIT_LDS (15 | (3 << 14) | (7 << 4))
constexpr int64_t kMaxGroups = 1 << 22;  // of kThreads: a grid holds less than 2^32 threads
constexpr int64_t kMaxThreads = 1ll << 32;  // of a grid, this not included
constexpr int64_t kMaxRows = (1ll << 31) - 512;  // with two threads a row (256 rows to a workgroup of 512) below that
constexpr int64_t kMaxInner = 131072;
constexpr int64_t kMaxStride = 1 << 24;  // of a row of x and of the output, in values
// Smallest row maximum that is divided by: 127 / 2^-120 is still finite.
constexpr float kTiny = 0x1p-120f;

// Largest magnitude of a row as a bit pattern: without the sign, patterns of float order like the
// numbers, infinity above them and NaN above infinity, so nothing that is not finite gets lost.
__device__ __forceinline__ unsigned top_of(unsigned m, const float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned a = __builtin_bit_cast(unsigned, v[i]) & 0x7fffffffu;
    m = a > m ? a : m;
  }
  return m;
}
template <int G>
__device__ __forceinline__ unsigned group_top(unsigned m) {
  return __builtin_bit_cast(unsigned, group_reduce<G>(__builtin_bit_cast(float, m), [](float a, float b) {
                              const unsigned x = __builtin_bit_cast(unsigned, a), y = __builtin_bit_cast(unsigned, b);
                              return x > y ? a : b;
                            }));
}
// inv = 127 / m and scale = m / 127; a row that is not finite comes out as NaN (and its q as 0).
__device__ __forceinline__ void row_scale(unsigned top, float& inv, float& scale) {
  const float t = __builtin_bit_cast(float, top);
  const float m = t > kTiny ? t : kTiny;
  const bool fine = top < 0x7f800000u;
  inv = fine ? 127.0f / m : 0.0f;
  scale = fine ? m / 127.0f : __builtin_nanf("");
}
// Four whole numbers in a word.  The product is rounded to float32 first and then, by adding 1.5 2^23,
// to the nearest whole number (ties to even), which the sum holds in its low bits.
__device__ __forceinline__ unsigned pack4(const float (&v)[4], float inv) {
#pragma clang fp contract(off)
  unsigned u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = v[i] * inv;
    u[i] = __builtin_bit_cast(unsigned, t + 12582912.0f);
  }
  const unsigned lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
  return inv == 0.0f ? 0u : lo | hi;
}

// q [M, width] (width >= K, zero past K) and the rows' scales.  W waves per row, which keep it in
// registers: R pieces of a lane each 16 bytes (four values of float32, eight of bfloat16).  R = 0: rows
// of any length, read twice.  Bound by memory: 8200 x 2048 in bfloat16 (50 MB) takes 13.2 us, 3.8 TB/s.
template <typename T, int R, int W>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t M, int K,
                                                            int8_t* __restrict__ q, int64_t ldq, int width,
                                                            float* __restrict__ scale) {
  constexpr int V = 16 / sizeof(T) / 4;  // fours of a lane
  constexpr int ROWS = kThreads / (64 * W), PIECE = 256 * V * W;
  static_assert(W == 1 || ROWS == 1, "the workgroup meets once a row");
  __shared__ unsigned tops[W > 1 ? 2 : 1][W];
  int turn = 0;
  const int lane = threadIdx.x % (64 * W);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / (64 * W); row < M;
       row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const T* const src = x + row * ldx;
    int8_t* const dst = q + row * ldq;
    unsigned top = 0;
    const auto fetch = [&](int c, held<T> (&raw)[V]) {
#pragma unroll
      for (int u = 0; u < V; ++u) raw[u] = hold_row<true>(src, c + 4 * u, K);
    };
    const auto look = [&](int c, const held<T> (&raw)[V], float (&v)[V][4]) {
#pragma unroll
      for (int u = 0; u < V; ++u) {
        widen_row<T>(raw[u], c + 4 * u, K, v[u]);
        top = top_of(top, v[u]);
      }
    };
    float inv, s;
    const auto agree = [&]() {
      top = group_top<64>(top);
      if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) tops[turn][threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; ++i) top = tops[turn][i] > top ? tops[turn][i] : top;
        turn ^= 1;
      }
      row_scale(top, inv, s);
    };
    const auto put = [&](int c, const float (&v)[V][4]) {
      unsigned w[V];
#pragma unroll
      for (int u = 0; u < V; ++u) w[u] = pack4(v[u], inv);
      if (c + 4 * V <= width) {
        __builtin_memcpy(dst + c, w, 4 * V);
      } else {
#pragma unroll
        for (int i = 0; i < 4 * V - 1; ++i)
          if (c + i < width) dst[c + i] = static_cast<int8_t>(w[i / 4] >> (8 * (i & 3)));
      }
    };
    if constexpr (R > 0) {
      held<T> raw[R][V];
      float v[R][V][4];
#pragma unroll
      for (int r = 0; r < R; ++r) fetch(r * PIECE + lane * 4 * V, raw[r]);
#pragma unroll
      for (int r = 0; r < R; ++r) look(r * PIECE + lane * 4 * V, raw[r], v[r]);
      agree();
#pragma unroll
      for (int r = 0; r < R; ++r) put(r * PIECE + lane * 4 * V, v[r]);
    } else {
      held<T> raw[V];
      float v[V][4];
#pragma unroll 4
      for (int c = lane * 4 * V; c < K; c += PIECE) {
        fetch(c, raw);
        look(c, raw, v);
      }
      agree();
#pragma unroll 4
      for (int c = lane * 4 * V; c < width; c += PIECE) {
        fetch(c, raw);
        look(c, raw, v);
        put(c, v);
      }
    }
    if (lane == 0) scale[row] = s;
  }
}

// The whole numbers k .. k + 15 of a row of K, zero from K on (k < K, a multiple of 16).  The last ones
// come with the 16 numbers that end the row, shifted into place; only a row shorter than 16 is read
// number by number.
__device__ __forceinline__ i32x4 load16(const int8_t* row, int k, int K) {
  i32x4 v;
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
    return v;
  }
  if (k) {
    unsigned __int128 w;
    __builtin_memcpy(&w, row + K - 16, 16);
    w >>= 8 * (k + 16 - K);
    return __builtin_bit_cast(i32x4, w);
  }
  unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; ++i)
    if (i < K) w[i >> 2] |= (static_cast<unsigned>(row[i]) & 255u) << (8 * (i & 3));
  return i32x4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
}

// Rows of whole numbers with another stride, zero from K to ldp (a multiple of 64).  A wave per row.
__global__ __launch_bounds__(kThreads) void pack_weight_kernel(const int8_t* __restrict__ w, int64_t ldw, int64_t N,
                                                               int K, int8_t* __restrict__ packed, int64_t ldp) {
  const int lane = threadIdx.x & 63;
  for (int64_t n = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 6; n < N;
       n += (static_cast<int64_t>(gridDim.x) * kThreads) >> 6)
    for (int64_t k = lane * 16; k < ldp; k += 1024) {
      i32x4 v = {0, 0, 0, 0};
      if (k < K) v = load16(w + n * ldw, static_cast<int>(k), K);
      *reinterpret_cast<i32x4*>(packed + n * ldp + k) = v;
    }
}

struct GemmArgs {
  const int8_t* a;  // [M, lda]: rows of whole numbers, zero from K to the next multiple of 64
  int64_t lda, M;
  const float* a_scale;
  const int8_t* w;  // [N, ldw]
  int64_t ldw, N;
  int K;
  const float* w_scale;
  const float* bias;
  int act;
  float slope;
  void* out;
  int64_t ldo;
};

// The fused form: x itself in the place of its whole numbers.
struct RowsArgs {
  const void* x;
  int64_t ldx, M;
  const int8_t* w;
  int64_t ldw;
  int K, N;
  const float* w_scale;
  const float* bias;
  int act;
  float slope;
  void* out;
  int64_t ldo;
};

// 32 rows of the output from a wave-uniform address on, row stride `ldo` (below 2^24: distances inside
// the block fit 32 bits).
template <typename OUT>
struct Block {
  __amdgpu_buffer_rsrc_t rsrc;
  int ld;  // bytes
  // The rows' 32 neighbouring outputs are whole 64-byte pieces of memory.  Only then are they stored as a
  // stream: pieces written in parts have to meet in the cache (58998 x 64 -> 431 in float32 takes 87 us
  // with the mark, 31 without).
  bool lines;
  // The address goes through the first lane: the compiler then knows it for a scalar and does not
  // loop over the lanes for each store.
  static __device__ OUT* scalar(OUT* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(a)));
    const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32)));
    return reinterpret_cast<OUT*>(hi << 32 | lo);
  }
  __device__ Block(OUT* base, int64_t ldo)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(scalar(base), 0, static_cast<int>(32 * ldo * sizeof(OUT)), 0x00027000)),
        ld(static_cast<int>(ldo * sizeof(OUT))),
        lines(((reinterpret_cast<uint64_t>(base) | static_cast<uint64_t>(ldo * sizeof(OUT))) & 63) == 0) {}
  // STREAM: marked as not read again soon (2 = nontemporal).
  template <bool STREAM>
  __device__ __forceinline__ void store(OUT v, unsigned lane_off, int row) const {
    if constexpr (sizeof(OUT) == 4)
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), rsrc, lane_off, row * ld, STREAM ? 2 : 0);
    else
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), rsrc, lane_off, row * ld, STREAM ? 2 : 0);
  }
};

// The last step for the 16 outputs a lane holds of a 32 x 32 block: column `lane % 32`, rows 8 (r / 4) +
// 4 (lane / 32) + r % 4, `sm[r]` the rows' scales, `sn` and `bias` the column's.  `to` describes the
// block's memory, `lane_off` is the lane's distance from its start in bytes and the rows' distances
// are scalars: with addresses of its own a lane would keep two registers for each of its rows.
//
// With scales from 2^-127 to 2^121 the product of a sum and both scales can leave float32's range
// half way although the result lies inside.  Where both scales are between 2^-60 and 2^60 (`is_plain`) it
// cannot; elsewhere it is formed from the scales' significands, and the powers are added and applied
// at the end.  Which of the two it is goes by the output's own scales, in every kernel: a result's bits
// depend neither on its neighbours nor on how many rows there are.  (`plain`: it holds for the whole wave.)
__device__ __forceinline__ bool is_plain(float s) { return s >= 0x1p-60f && s <= 0x1p60f; }

__device__ __forceinline__ float scaled(int acc, float sm, float sn, float bias) {
  return __builtin_fmaf(static_cast<float>(acc) * sn, sm, bias);
}
// The same of any scales; `y` is what `scaled` gives.
__device__ __forceinline__ float scaled_any(float y, int acc, float sm, float sn, float bias) {
  const float f = static_cast<float>(acc) * __builtin_amdgcn_frexp_mantf(sm) * __builtin_amdgcn_frexp_mantf(sn);
  const float wide = __builtin_amdgcn_ldexpf(f, __builtin_amdgcn_frexp_expf(sm) + __builtin_amdgcn_frexp_expf(sn)) + bias;
  return is_plain(sm) & is_plain(sn) ? y : wide;  // both at hand: no branch for each output
}

__device__ __forceinline__ float finish(int acc, float sm, float sn, float bias, int act, float slope) {
  const float y = scaled_any(scaled(acc, sm, sn, bias), acc, sm, sn, bias);
  if (act == SPMI_ACT_RELU) return y < 0.0f ? 0.0f : y;  // not a maximum: NaN stays
  if (act == SPMI_ACT_LEAKY_RELU) return y < 0.0f ? y * slope : y;
  return y;
}

template <typename OUT>
__device__ __forceinline__ void finish16(const i32x16& acc, const float (&sm)[16], float sn, float bias, bool plain,
                                         int act, float slope, Block<OUT> to, unsigned lane_off, int left) {
  float y[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) y[r] = scaled(acc[r], sm[r], sn, bias);
  if (!plain) {
#pragma unroll
    for (int r = 0; r < 16; ++r) y[r] = scaled_any(y[r], acc[r], sm[r], sn, bias);
  }
  if (act == SPMI_ACT_RELU) {
#pragma unroll
    for (int r = 0; r < 16; ++r) y[r] = y[r] < 0.0f ? 0.0f : y[r];
  } else if (act == SPMI_ACT_LEAKY_RELU) {
#pragma unroll
    for (int r = 0; r < 16; ++r) y[r] = y[r] < 0.0f ? y[r] * slope : y[r];
  }
  if (left >= 32 && to.lines) {
#pragma unroll
    for (int r = 0; r < 16; ++r) to.template store<true>(static_cast<OUT>(y[r]), lane_off, 8 * (r / 4) + r % 4);
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (8 * (r / 4) + r % 4 < left) to.template store<false>(static_cast<OUT>(y[r]), lane_off, 8 * (r / 4) + r % 4);
  }
}

// Tiles of BM x BN outputs, WM x WN waves, ST stages of 64 bytes of K in LDS.
//
// Rows go from global memory into LDS directly, 16 bytes a lane, ST - 1 stages ahead of the products;
// a stage is complete when the wave's own loads of it have landed (a counted wait) and a barrier
// has told so for all waves, and that barrier also frees the buffer the next loads go to: one
// barrier a stage.  Bound by the matrix instructions and the LDS reads that feed them: 8192 x 4096 -> 4096 in
// 140 us, 1964 x 10^12 operations a second.  An LDS row is 64 bytes, so a 16-lane group that reads 16 bytes of 16 rows meets
// each bank four times unless the four pieces of a row are turned by the row's number / 4: the loads
// fetch them in that order.  Rows past the end repeat the last one and are not stored.
template <typename OUT, int BM, int BN, int WM, int WN, int ST>
__global__ __launch_bounds__(WM * WN * 64) void tile_i8_kernel(GemmArgs p) {
  constexpr int MB = BM / WM / 32, NB = BN / WN / 32;
  constexpr int STAGE = (BM + BN) * 64;
  // loads of a wave per stage, 16 rows each; the first EXTRA waves have one more
  constexpr int LPW = (BM + BN) / 16 / (WM * WN), EXTRA = (BM + BN) / 16 % (WM * WN);
  extern __shared__ i32x4 smem[];
  char* const lds = reinterpret_cast<char*>(smem);

  // Workgroup b runs on XCD b % 8, which has an L2 of its own: give each XCD neighbouring tiles, four
  // tile rows at a time, so that the tiles in flight share rows of both operands.
  const int tm = static_cast<int>((p.M + BM - 1) / BM), tn = static_cast<int>((p.N + BN - 1) / BN);
  const int64_t tiles = static_cast<int64_t>(tm) * tn, per = (tiles + 7) / 8;
  const int64_t t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || t >= tiles) return;
  const int band = static_cast<int>(t / (4 * static_cast<int64_t>(tn)));
  const int in_band = static_cast<int>(t - static_cast<int64_t>(band) * 4 * tn);
  const int high = tm - band * 4 < 4 ? tm - band * 4 : 4;
  const int64_t m0 = static_cast<int64_t>(band * 4 + in_band % high) * BM, n0 = static_cast<int64_t>(in_band / high) * BN;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;

  const bool more = wave < EXTRA;
  const int first = wave * LPW + (more ? wave : EXTRA);
  const int8_t* src[LPW + (EXTRA > 0)];
#pragma unroll
  for (int i = 0; i < LPW + (EXTRA > 0); ++i) {
    const int row = (first + i) * 16 + lane / 4;  // of the BM rows of a, then the BN rows of w
    const int piece = ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
    if (row < BM) {
      const int64_t m = m0 + row < p.M ? m0 + row : p.M - 1;
      src[i] = p.a + m * p.lda + piece;
    } else {
      const int64_t n = n0 + row - BM < p.N ? n0 + row - BM : p.N - 1;
      src[i] = p.w + n * p.ldw + piece;
    }
  }
  // scales and bias for the last step, behind the stages
  float* const row_scale = reinterpret_cast<float*>(lds + ST * STAGE);
  float* const col_scale = row_scale + BM;
  float* const col_bias = col_scale + BN;
  for (int i = threadIdx.x; i < BM + BN; i += WM * WN * 64) {
    if (i < BM) {
      row_scale[i] = m0 + i < p.M ? p.a_scale[m0 + i] : 1.0f;
    } else {
      const int64_t n = n0 + i - BM;
      col_scale[i - BM] = n < p.N ? p.w_scale[n] : 1.0f;
      col_bias[i - BM] = p.bias && n < p.N ? p.bias[n] : 0.0f;
    }
  }
  const int stages = (p.K + 63) / 64;
  auto fetch = [&](int k) {
    char* const to = lds + (k % ST) * STAGE + first * 1024;
#pragma unroll
    for (int i = 0; i < LPW + (EXTRA > 0); ++i)
      if (i < LPW || more)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[i] + k * 64),
                                         (__attribute__((address_space(3))) void*)(to + i * 1024), 16, 0, 0);
  };
  // at most the loads of `n` stages of this wave outstanding
  auto wait = [&](auto n) {
    if (EXTRA > 0 && more) __builtin_amdgcn_s_waitcnt(WAIT_LOADS(decltype(n)::value * (LPW + 1)));
    else __builtin_amdgcn_s_waitcnt(WAIT_LOADS(decltype(n)::value * LPW));
  };

  i32x16 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = i32x16{0};

#pragma unroll
  for (int k = 0; k < ST - 1; ++k)
    if (k < stages) fetch(k);

  // Fragments of half a stage: while one half is multiplied the next one is on its way from LDS, also
  // over the barrier, which the matrix cores then do not notice.
  const int lr = lane & 31, lh = lane >> 5;
  const int at = lr * 64 + ((lh ^ ((lr >> 2) & 3)) << 4);
  i32x4 fa[2][MB], fw[2][NB];
  auto read = [&](int k, int h) {
    const int sa = (k % ST) * STAGE + wm * (MB * 2048) + at, sw = (k % ST) * STAGE + BM * 64 + wn * (NB * 2048) + at;
#pragma unroll
    for (int i = 0; i < MB; ++i) fa[h][i] = *reinterpret_cast<const i32x4*>(lds + ((sa + i * 2048) ^ (h * 32)));
#pragma unroll
    for (int j = 0; j < NB; ++j) fw[h][j] = *reinterpret_cast<const i32x4*>(lds + ((sw + j * 2048) ^ (h * 32)));
  };
  auto multiply = [&](int h) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[h][i], fw[h][j], acc[i][j], 0, 0, 0);
  };
  // Stage k complete for all waves.  (The empty asm keeps the compiler from moving LDS reads over it.)
  auto complete = [&](int k) {
    asm volatile("" ::: "memory");
    if (k + ST - 2 <= stages) wait(std::integral_constant<int, ST - 3>{});
    else wait(std::integral_constant<int, 0>{});
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  static_assert(ST >= 3, "the loads of a stage are waited for one stage early");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(WAIT_LDS);  // the scales are there for everyone after the barrier
  if (ST - 1 <= stages) wait(std::integral_constant<int, ST - 2>{});
  else wait(std::integral_constant<int, 0>{});
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  read(0, 0);
  for (int k = 0; k < stages; ++k) {
    // what the next products need has had the last products' time to arrive; waiting for it before
    // further reads are issued keeps those out of the wait
    __builtin_amdgcn_s_waitcnt(WAIT_LDS);
    read(k, 1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(0);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(WAIT_LDS);
    if (k + 1 < stages) {
      complete(k + 1);
      if (k + ST - 1 < stages) fetch(k + ST - 1);
      read(k + 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    multiply(1);
    __builtin_amdgcn_sched_barrier(0);
  }

  const int left = p.M - m0 < BM ? static_cast<int>(p.M - m0) : BM;
  const int cols_left = p.N - n0 < BN ? static_cast<int>(p.N - n0) : BN;
  OUT* const out = static_cast<OUT*>(p.out) + m0 * p.ldo + n0;
  const unsigned lane_off = static_cast<unsigned>(4 * lh * static_cast<int>(p.ldo) + lr) * sizeof(OUT);
  bool plain = true;
#pragma unroll
  for (int j = 0; j < NB; ++j) plain = plain && is_plain(col_scale[(wn * NB + j) * 32 + lr]);
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int m = (wm * MB + i) * 32 + 4 * lh;
    float sm[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) sm[r] = row_scale[m + 8 * (r / 4) + r % 4];
#pragma unroll
    for (int r = 0; r < 16; ++r) plain = plain && is_plain(sm[r]);
    const bool all_plain = __all(plain);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int n = (wn * NB + j) * 32 + lr;
      if (n < cols_left)
        finish16(acc[i][j], sm, col_scale[n], col_bias[n], all_plain, p.act, p.slope,
                 Block<OUT>(out + (wm * MB + i) * 32 * p.ldo + (wn * NB + j) * 32, p.ldo), lane_off,
                 left >= BM ? 32 : left - m);
    }
  }
}

// Rows of up to 512 values: one pass over x.  A wave takes 32 rows.  G lanes read a row in whole
// lines, find its largest magnitude among themselves and write its whole numbers into LDS rows of
// the wave's own, from where they come back as matrix operands (lane = row, 16 neighbouring k) and
// stay in registers; LDS is then free for the weight, which passes through it 32 columns at a time,
// the next slice on its way while one is multiplied: one barrier a slice.
//
// The kernel is bound by memory: x is read once, results are written once, 128 contiguous bytes of a
// row at a time, both marked as streams (10^5 x 512 -> 1024: 179 us without, 152 with), and the weight
// comes from L2 once per 256 rows: 10^6 x 128 -> 256 in float32 takes 290 us, 5.3 TB/s.  Workgroups are
// short (256 rows): handed out in order, they keep what is in flight close together in memory, which is worth
// a tenth against a resident grid that strides over the rows.  They begin at different columns: 96 us instead
// of 124 at 10^5 x 128 -> 1024.  LDS rows are padded by 16 bytes: 16 lanes that read 16 bytes of 16
// neighbouring rows then meet each bank once.
template <int KP>
struct RowsShape {
  static constexpr int NW = 8, SK = KP + 16;
  static constexpr int G = KP / 4 < 64 ? KP / 4 : 64, R = KP / 4 / G;  // lanes of a row, vectors of a lane
  static constexpr int RPL = 64 / G;                                  // rows of one load
  static constexpr int SROWS = KP > 256 ? 16 : 32;                    // rows in LDS at a time
  static constexpr int VECS = 16;                                     // vectors of a lane in flight
  static constexpr int BROWS = VECS / R * RPL < SROWS ? VECS / R * RPL : SROWS;  // rows of a batch of loads
  static constexpr int SLICE = 32 * SK + 256;                         // 32 columns, their scales and biases
  static constexpr int STAGING = SROWS * SK + 128;
  static constexpr int LDS = NW * STAGING > 2 * SLICE ? NW * STAGING : 2 * SLICE;
};

template <typename T, typename OUT, int KP>
__global__ __launch_bounds__(RowsShape<KP>::NW * 64, 2) void rows_i8_kernel(RowsArgs p) {
  using S = RowsShape<KP>;
  constexpr int SK = S::SK, KS = KP / 32, R = S::R, RPL = S::RPL, LOADS = S::BROWS / RPL;
  extern __shared__ i32x4 smem[];
  char* const lds = reinterpret_cast<char*>(smem);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* const stage = lds + wave * S::STAGING;
  float* const scales = reinterpret_cast<float*>(stage + S::SROWS * SK);

  const int c = lane % S::G * 4, sub = lane / S::G;
  const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * S::NW + wave) * 32;
  const bool full = row0 + 32 <= p.M;
  const T* const x0 = static_cast<const T*>(p.x) + row0 * p.ldx;
  const int last_row = full ? 31 : static_cast<int>(p.M - 1 - row0);  // may be negative: rows before the wave's
  float v[LOADS][R][4];
  auto fetch = [&](int r0) {  // rows r0 .. r0 + BROWS of the wave's 32
    // Loads without a condition around them, so that all are in flight together: rows past the end read
    // the last row again, and a lane whose four values pass the end of the row reads the row's last four
    // and moves them down.
    if (p.K >= 4) {
#pragma unroll
      for (int b = 0; b < LOADS; ++b) {
        int row = r0 + b * RPL + sub;
        row = row <= last_row ? row : last_row;
        const T* const src = x0 + row * p.ldx;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int k = r * 256 + c, from = k <= p.K - 4 ? k : p.K - 4, by = k - from;
          load4<true>(src + from, v[b][r]);
          float (&t)[4] = v[b][r];
          if (p.K % 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = (by & 2) ? (i < 2 ? t[i + 2] : 0.0f) : t[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = (by & 1) ? (i < 3 ? t[i + 1] : 0.0f) : t[i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) t[i] = by < 4 ? t[i] : 0.0f;
        }
      }
    } else {
#pragma unroll
      for (int b = 0; b < LOADS; ++b)
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[b][r][i] = 0.0f;
          const int k = r * 256 + c;
          if (r0 + b * RPL + sub <= last_row && k < p.K)
            load4_upto(x0 + (r0 + b * RPL + sub) * p.ldx + k, p.K - k, 0.0f, v[b][r]);
        }
    }
  };
  // a slice of the weight: thread = 16-byte pieces; and one of the 32 scales and 32 biases
  constexpr int PIECES = (32 * KP / 16 + S::NW * 64 - 1) / (S::NW * 64);
  i32x4 w[PIECES];
  float of_col = 0.0f;
  auto fetch_slice = [&](int n0) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = i * (S::NW * 64) + tid, n = n0 + at / (KP / 16), k = at % (KP / 16) * 16;
      w[i] = i32x4{0, 0, 0, 0};
      if (at < 32 * KP / 16 && n < p.N && k < p.K) w[i] = load16(p.w + n * p.ldw, k, p.K);
    }
    if (tid < 64) {
      const int n = n0 + (tid & 31);
      of_col = tid < 32 ? (n < p.N ? p.w_scale[n] : 1.0f) : (p.bias && n < p.N ? p.bias[n] : 0.0f);
    }
  };
  auto put_slice = [&](char* to) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = i * (S::NW * 64) + tid;
      if (at < 32 * KP / 16) *reinterpret_cast<i32x4*>(to + at / (KP / 16) * SK + at % (KP / 16) * 16) = w[i];
    }
    if (tid < 64) reinterpret_cast<float*>(to + 32 * SK)[tid] = of_col;
  };

  const int lr = lane & 31, lh = lane >> 5;
  i32x4 xa[KS];
  float sm[16];
  fetch(0);
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += S::BROWS) {
    if (r0) fetch(r0);
#pragma unroll
    for (int b = 0; b < LOADS; ++b) {
      unsigned top = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) top = top_of(top, v[b][r]);
      top = group_top<S::G>(top);
      float inv, s;
      row_scale(top, inv, s);
      const int at = (r0 + b * RPL + sub) % S::SROWS;
#pragma unroll
      for (int r = 0; r < R; ++r) *reinterpret_cast<unsigned*>(stage + at * SK + r * 256 + c) = pack4(v[b][r], inv);
      if (c == 0) scales[at] = s;
    }
    if ((r0 + S::BROWS) % S::SROWS == 0) {
      // the wave's own LDS rows: no other wave touches them
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      const int h0 = r0 + S::BROWS - S::SROWS;  // first of the rows that are there
      if (S::SROWS == 32 || (lr & 16) == h0) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
          xa[k] = *reinterpret_cast<const i32x4*>(stage + (lr - h0) * SK + k * 32 + lh * 16);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int m = 8 * (r / 4) + r % 4;
        if (m >= h0 && m < h0 + S::SROWS) sm[r] = scales[m - h0 + 4 * lh];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  }
  bool plain = true;
#pragma unroll
  for (int r = 0; r < 16; ++r) plain = plain && is_plain(sm[r]);
  const bool rows_plain = __all(plain);

  // The workgroup's share of the slices.  It begins at a slice of its own: rows of a power-of-two
  // length would otherwise have all workgroups write to the same few memory channels at a time.
  const int slices = (p.N + 31) / 32, share = (slices + gridDim.y - 1) / gridDim.y;
  const int first = blockIdx.y * share, count = slices - first < share ? slices - first : share;
  if (count <= 0) return;
  const int turned = blockIdx.x % count;
  const auto column = [&](int i) { return (first + (i + turned) % count) * 32; };
  fetch_slice(column(0));
  __syncthreads();  // every wave has its operands: LDS is free
  put_slice(lds);
  const int left = full ? 32 : static_cast<int>(p.M - row0) - 4 * lh;
  OUT* const out = static_cast<OUT*>(p.out) + row0 * p.ldo;
  const unsigned lane_off = static_cast<unsigned>(4 * lh * static_cast<int>(p.ldo) + lr) * sizeof(OUT);
  for (int i = 0; i < count; ++i) {
    const int n0 = column(i);
    const bool more = i + 1 < count;
    if (more) fetch_slice(column(i + 1));
    __syncthreads();
    const char* const slice = lds + (i & 1) * S::SLICE;
    i32x16 acc = {0};
#pragma unroll
    for (int k = 0; k < KS; ++k)
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(
          xa[k], *reinterpret_cast<const i32x4*>(slice + lr * SK + k * 32 + lh * 16), acc, 0, 0, 0);
    if constexpr (KS > 8) {
      // Four operands ahead of the products that take them.  Left to itself the compiler reads each of the 16 when
      // it is needed: 100003 x 512 -> 1024 takes 156 us so, and 148 with the reads ahead.  The shorter rows' kernels
      // have more waves to cover the wait, and the order costs them (20863 x 182 -> 3265 in bfloat16 98 us, 91 without).
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int k = 0; k < KS - 4; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    }
    const float sn = reinterpret_cast<const float*>(slice + 32 * SK)[lr];
    const float bias = reinterpret_cast<const float*>(slice + 32 * SK)[32 + lr];
    const bool all_plain = rows_plain && __all(is_plain(sn));
    if (n0 + lr < p.N) finish16(acc, sm, sn, bias, all_plain, p.act, p.slope, Block<OUT>(out + n0, p.ldo), lane_off, left);
    if (more) put_slice(lds + (~i & 1) * S::SLICE);
  }
}

// Few rows (up to 16 MT): reading the weight is the work.  A workgroup owns 16 columns; its eight
// waves take turns at the 64-byte pieces of K, reading them from memory straight into the operand
// layout (16 rows, 16 neighbouring k a lane), and add their sums up in LDS at the end.  The rows are
// brought to whole numbers in LDS by every workgroup for itself (T float or bfloat16: a launch less,
// and a small x comes from L2), or come from a matrix made before (T int8_t: larger x).  Four loads a
// wave are ahead of the products (eight: 8 x 8192 -> 8192 takes 30 us, not 21).
struct FewArgs {
  const void* x;         // [M, K] values, or whole numbers zero from K to the next multiple of 64
  int64_t ldx;
  const float* x_scale;  // of the whole numbers
  int M;
  const int8_t* w;
  int64_t ldw, N;
  int K;
  const float* w_scale;
  const float* bias;
  int act;
  float slope;
  void* out;
  int64_t ldo;
};
constexpr int kFewWaves = 8;
constexpr int kFewRows = 64;

// Pieces of a workgroup's width that M rows of K values take, and how many of them it holds: the rows are
// loaded at once and stay in registers.  By 4096 columns in bfloat16, 16 rows of 2048 take 11.1 us a call so
// and 14.4 with a launch of their own for the whole numbers, 8 of 4096 13.2 and 15.8; but twice the pieces in
// two turns, 16 of 4096, took 21.1 where the launch takes 15.9.
constexpr int kFewPiece = kFewWaves * 256;
constexpr int kFewPieces = 16;

// P: pieces held (T float or bfloat16); MT: rows, in sixteens.
template <typename T, typename OUT, int MT, int P>
__global__ __launch_bounds__(kFewWaves * 64) void few_i8_kernel(FewArgs p) {
  constexpr bool MAKE = sizeof(T) > 1;
  constexpr int NW = kFewWaves, U = 4;
  static_assert(MAKE ? P > 0 && P <= kFewPieces && MT == 1 : P == 0, "pieces");
  __shared__ i32x4 sums[NW][MT][64];
  __shared__ float row_scale_of[16 * MT];
  __shared__ unsigned tops[MAKE ? P : 1][NW];
  __shared__ float inv_of[16];
  extern __shared__ i32x4 smem[];
  char* const q = reinterpret_cast<char*>(smem);  // MAKE: rows of KP + 16 bytes
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int KP = (p.K + 63) & ~63, SK = KP + 16;
  const int steps = KP / 64;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 16 + (lane & 15);
  const int part = (lane >> 4) * 16;
  const int8_t* const w = p.w + (n < p.N ? n : p.N - 1) * p.ldw;
  auto piece = [&](int s) {
    const int k = s * 64 + part;
    return k < p.K ? load16(w, k, p.K) : i32x4{0, 0, 0, 0};
  };
  i32x4 fw[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (wave + u * NW < steps) fw[u] = piece(wave + u * NW);  // on the way while the rows are prepared

  const T* const x = static_cast<const T*>(p.x);
  if constexpr (MAKE) {
    const int per = (p.K + kFewPiece - 1) / kFewPiece;  // pieces of a row; those of all rows are on the way together
    held<T> raw[P];
    {
      int r = 0, i = 0;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        raw[k] = hold_row<false>(x + r * p.ldx, i * kFewPiece + tid * 4, p.K);
        if (++i == per) {
          i = 0;
          r = r + 1 < p.M ? r + 1 : r;  // past the last row: it again, not used
        }
      }
      i = 0;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        float v[4];
        widen_row<T>(raw[k], i * kFewPiece + tid * 4, p.K, v);
        const unsigned top = group_top<64>(top_of(0, v));
        if (lane == 0) tops[k][wave] = top;
        i = i + 1 < per ? i + 1 : 0;
      }
    }
    __syncthreads();
    if (tid < p.M) {
      unsigned top = 0;
      for (int k = tid * per; k < tid * per + per; ++k)
#pragma unroll
        for (int i = 0; i < NW; ++i) top = tops[k][i] > top ? tops[k][i] : top;
      row_scale(top, inv_of[tid], row_scale_of[tid]);
    }
    __syncthreads();
    int r = 0, i = 0;
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const int c = i * kFewPiece + tid * 4;
      float v[4];
      widen_row<T>(raw[k], c, p.K, v);
      if (r < p.M && c < KP) *reinterpret_cast<unsigned*>(q + r * SK + c) = pack4(v, inv_of[r]);
      if (++i == per) {
        i = 0;
        ++r;
      }
    }
    __syncthreads();
  } else {
    if (tid < 16 * MT) row_scale_of[tid] = tid < p.M ? p.x_scale[tid] : 1.0f;
  }

  i32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = i32x4{0, 0, 0, 0};
  for (int s0 = wave; s0 < steps; s0 += U * NW) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * NW;
      if (s < steps) {
        const i32x4 f = fw[u];
        if (s + U * NW < steps) fw[u] = piece(s + U * NW);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          int r = t * 16 + (lane & 15);
          r = r < p.M ? r : p.M - 1;  // rows past the end repeat the last one and are not stored
          i32x4 a;
          if constexpr (MAKE) a = *reinterpret_cast<const i32x4*>(q + r * SK + s * 64 + part);
          else a = *reinterpret_cast<const i32x4*>(reinterpret_cast<const char*>(x) + r * p.ldx + s * 64 + part);
          acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, f, acc[t], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) sums[wave][t][lane] = acc[t];
  __syncthreads();
  // lane l of a block holds column l % 16, rows 4 (l / 16) + 0..3
  for (int i = tid; i < MT * 256; i += NW * 64) {
    const int t = i >> 8, row = (i >> 4) & 15, col = i & 15;
    const int l = (row >> 2) * 16 + col;
    int sum = 0;
#pragma unroll
    for (int v = 0; v < NW; ++v) sum += reinterpret_cast<const int*>(&sums[v][t][l])[row & 3];
    const int m = t * 16 + row;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 16 + col;
    if (m < p.M && c < p.N)
      static_cast<OUT*>(p.out)[m * p.ldo + c] =
          static_cast<OUT>(finish(sum, row_scale_of[m], p.w_scale[c], p.bias ? p.bias[c] : 0.0f, p.act, p.slope));
  }
}

// Sizes for rows_i8_kernel.  Rows of up to 256 values always; of up to 512 where there are enough for
// one pass over x to pay (65 us against 69 for two launches at 10^5 rows of 512 by 256 columns in
// bfloat16, 177 against 224 by 1024 in float32, but 35 against 27 at 20000 rows by 512) and the
// padding to 512 is small (120 against 98 at 10^5 rows of 300).
bool rows_take(int64_t M, int64_t K) {
  return M > kFewRows && (K <= 256 || (K > 384 && K <= 512 && M >= 65536));
}

template <typename T, typename OUT>
int launch_rows(const RowsArgs& a, hipStream_t st) {
  const auto go = [&](auto kp) {
    using S = RowsShape<decltype(kp)::value>;
    const auto kernel = rows_i8_kernel<T, OUT, decltype(kp)::value>;
    SPMI_RAISE_LDS_LIMIT(kernel, static_cast<size_t>(S::LDS));
    // Few rows: the columns are shared out until there is a workgroup for each CU (more of them cost
    // more than they hide, since each makes the whole numbers of its rows again).
    const int64_t groups = (a.M + 32 * S::NW - 1) / (32 * S::NW), slices = (a.N + 31) / 32;
    int64_t shares = 256 / groups;
    shares = shares < 1 ? 1 : shares < slices ? shares : slices;
    kernel<<<dim3(static_cast<unsigned>(groups), static_cast<unsigned>(shares)), S::NW * 64, S::LDS, st>>>(a);
    return SPMI_OK;
  };
  if (a.K <= 32) return go(std::integral_constant<int, 32>{});
  if (a.K <= 64) return go(std::integral_constant<int, 64>{});
  if (a.K <= 128) return go(std::integral_constant<int, 128>{});
  if (a.K <= 256) return go(std::integral_constant<int, 256>{});
  return go(std::integral_constant<int, 512>{});
}

int64_t padded(int64_t K) { return (K + 63) / 64 * 64; }

template <typename OUT, int BM, int BN, int WM, int WN, int ST>
int launch_tile(const GemmArgs& a, hipStream_t st) {
  constexpr size_t lds = static_cast<size_t>(ST) * (BM + BN) * 64 + (BM + 2 * BN) * sizeof(float);
  const auto kernel = tile_i8_kernel<OUT, BM, BN, WM, WN, ST>;
  const int64_t tiles = ((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN);
  SPMI_REQUIRE((tiles + 7) / 8 * 8 < kMaxThreads / (WM * WN * 64), SPMI_ERR_UNSUPPORTED,
               "spmi_linear_i8: %lld x %lld outputs are too many", (long long)a.M, (long long)a.N);
  SPMI_RAISE_LDS_LIMIT(kernel, lds);
  kernel<<<static_cast<unsigned>((tiles + 7) / 8 * 8), WM * WN * 64, lds, st>>>(a);
  return SPMI_OK;
}
// A CU's share of the work with tiles of an area: how many of them the busiest CU gets.  Tiles of
// 256 x 256 move the least through LDS and L2, smaller ones leave fewer CUs idle at the end: the product
// of 8200 x 2048 -> 4096 takes 107 us in tiles of 256 x 256 (a third round for 16 of 528 tiles), 101 of
// 128 x 128 and 94 of 192 x 256.  The weights are what the smaller tiles cost more per output.
template <typename OUT>
int launch_tiles(const GemmArgs& a, hipStream_t st) {
  const auto share = [&](int64_t bm, int64_t bn, double weight) {
    const int64_t tiles = ((a.M + bm - 1) / bm) * ((a.N + bn - 1) / bn);
    return static_cast<double>((tiles + 255) / 256) * static_cast<double>(bm * bn) * weight;
  };
  const double big = share(256, 256, 1.0), high = share(192, 256, 1.0), mid = share(128, 128, a.K <= 512 ? 1.0 : 1.2),
               low = share(64, 64, 2.0);
  if (low < mid && low < big && low < high) return launch_tile<OUT, 64, 64, 2, 2, 4>(a, st);
  if (mid < big && mid < high) return launch_tile<OUT, 128, 128, 2, 4, 3>(a, st);
  if (high < big) return launch_tile<OUT, 192, 256, 3, 4, 4>(a, st);
  return launch_tile<OUT, 256, 256, 2, 4, 4>(a, st);
}

int64_t few_pieces(int64_t M, int64_t K) { return M * ((K + kFewPiece - 1) / kFewPiece); }

template <typename T, typename OUT>
int launch_few(const FewArgs& a, hipStream_t st) {
  const unsigned grid = static_cast<unsigned>((a.N + 15) / 16);
  const auto go = [&](auto mt, auto pieces) {
    constexpr int MT = decltype(mt)::value;
    const size_t lds = sizeof(T) > 1 ? static_cast<size_t>(a.M) * (((a.K + 63) & ~63) + 16) : 0;
    const auto kernel = few_i8_kernel<T, OUT, MT, decltype(pieces)::value>;
    SPMI_RAISE_LDS_LIMIT(kernel, lds);
    kernel<<<grid, kFewWaves * 64, lds, st>>>(a);
    return SPMI_OK;
  };
  using One = std::integral_constant<int, 1>;
  if constexpr (sizeof(T) > 1) {
    const int64_t pieces = few_pieces(a.M, a.K);
    if (pieces <= 1) return go(One{}, One{});
    if (pieces <= 4) return go(One{}, std::integral_constant<int, 4>{});
    return go(One{}, std::integral_constant<int, kFewPieces>{});
  } else {
    using None = std::integral_constant<int, 0>;
    if (a.M <= 16) return go(One{}, None{});
    if (a.M <= 32) return go(std::integral_constant<int, 2>{}, None{});
    return go(std::integral_constant<int, 4>{}, None{});
  }
}
// Rows that every workgroup of few_i8_kernel brings to whole numbers for itself: as many as it holds, and not so
// many columns that the repetition costs more than a launch (16 x 1024 in bfloat16 to 8192 columns 12.0 us
// against 14.7, to 16384 20.9 against 14.8; 4 x 1024 to 50000 26.4 against 18.5; one row to 50000 17.4
// against 17.7).
bool few_made(int64_t M, int64_t K, int64_t N) {
  const int64_t pieces = few_pieces(M, K);
  return pieces == 1 || (pieces <= kFewPieces && pieces * N <= 131072);
}

int check_rows(const char* what, int dtype, int64_t M, int64_t K) {
  SPMI_REQUIRE(dtype == SPMI_DTYPE_F32 || dtype == SPMI_DTYPE_BF16, SPMI_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  SPMI_REQUIRE(M >= 0 && K >= 1, SPMI_ERR_INVALID_ARG, "%s: M=%lld K=%lld", what, (long long)M, (long long)K);
  SPMI_REQUIRE(K <= kMaxInner && M <= kMaxRows, SPMI_ERR_UNSUPPORTED,
               "%s: %lld rows of %lld values (at most %lld rows of %lld)", what, (long long)M, (long long)K,
               (long long)kMaxRows, (long long)kMaxInner);
  return SPMI_OK;
}

template <typename T>
void launch_quantize(const void* x, int64_t ldx, int64_t M, int64_t K, int8_t* q, int64_t ldq, int64_t width,
                     float* scale, hipStream_t st) {
  const auto go = [&](auto r, auto w) {
    constexpr int W = decltype(w)::value, ROWS = kThreads / (64 * W);
    const int64_t groups = (M + ROWS - 1) / ROWS;
    quantize_kernel<T, decltype(r)::value, W>
        <<<static_cast<unsigned>(groups < kMaxGroups ? groups : kMaxGroups), kThreads, 0, st>>>(
            static_cast<const T*>(x), ldx, M, static_cast<int>(K), q, ldq, static_cast<int>(width), scale);
  };
  using One = std::integral_constant<int, 1>;
  using Four = std::integral_constant<int, 4>;
  // Rows of up to four pieces go to one wave each, longer ones to four (the projection of 64 x 8192 to 2048
  // columns in bfloat16 takes 25.7 us so and 33.5 with one, 8200 x 4096 to 512 in float32 64 and 68).
  const int64_t pieces = (width * static_cast<int64_t>(sizeof(T)) + 1023) / 1024;  // of a wave
  if (pieces <= 1) go(std::integral_constant<int, 1>{}, One{});
  else if (pieces <= 2) go(std::integral_constant<int, 2>{}, One{});
  else if (pieces <= 4) go(std::integral_constant<int, 4>{}, One{});
  else if (pieces <= 8) go(std::integral_constant<int, 2>{}, Four{});
  else if (pieces <= 16) go(std::integral_constant<int, 4>{}, Four{});
  else if (pieces <= 32) go(std::integral_constant<int, 8>{}, Four{});
  else go(std::integral_constant<int, 0>{}, Four{});
}
void launch_quantize(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, int8_t* q, int64_t ldq,
                     int64_t width, float* scale, hipStream_t st) {
  if (dtype == SPMI_DTYPE_F32) launch_quantize<float>(x, ldx, M, K, q, ldq, width, scale, st);
  else launch_quantize<bf16>(x, ldx, M, K, q, ldq, width, scale, st);
}

}  // namespace

extern "C" {

int spmi_quantize_rows_i8(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, int8_t* q, int64_t ldq,
                          float* scale, void* stream) {
  if (int rc = check_rows("spmi_quantize_rows_i8", dtype, M, K)) return rc;
  if (M == 0) return SPMI_OK;
  SPMI_REQUIRE(x && q && scale && ldx >= 0 && ldq >= K, SPMI_ERR_INVALID_ARG,
               "spmi_quantize_rows_i8: null pointer or row stride too small");
  launch_quantize(x, dtype, ldx, M, K, q, ldq, K, scale, as_stream(stream));
  SPMI_CHECK_LAUNCH("spmi_quantize_rows_i8");
  return SPMI_OK;
}

size_t spmi_linear_i8_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  if (few_made(M, K, N) || rows_take(M, K)) return 0;
  // whole numbers of x, their scales, the weight in rows of whole stages (not needed if it has them)
  return align_up(static_cast<size_t>(M) * padded(K), 256) + align_up(static_cast<size_t>(M) * sizeof(float), 256) +
         (static_cast<size_t>(N) * padded(K));
}

int spmi_linear_i8(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, const int8_t* weight, int64_t ldw,
                   const float* w_scale, int64_t N, const float* bias, int act, float slope, void* out, int out_dtype,
                   int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_rows("spmi_linear_i8", dtype, M, K)) return rc;
  SPMI_REQUIRE(N >= 0 && N < (1ll << 31), SPMI_ERR_INVALID_ARG, "spmi_linear_i8: N=%lld", (long long)N);
  SPMI_REQUIRE(out_dtype == SPMI_DTYPE_F32 || out_dtype == SPMI_DTYPE_BF16, SPMI_ERR_INVALID_ARG,
               "spmi_linear_i8: out_dtype %d", out_dtype);
  SPMI_REQUIRE(act >= SPMI_ACT_NONE && act <= SPMI_ACT_LEAKY_RELU, SPMI_ERR_INVALID_ARG, "spmi_linear_i8: act %d", act);
  SPMI_REQUIRE(ldx < kMaxStride && ldo < kMaxStride, SPMI_ERR_UNSUPPORTED,
               "spmi_linear_i8: row strides of %lld and %lld values (below %lld)", (long long)ldx, (long long)ldo,
               (long long)kMaxStride);
  if (M == 0 || N == 0) return SPMI_OK;
  SPMI_REQUIRE(x && weight && w_scale && out && ldx >= 0 && ldw >= 0 && ldo >= N, SPMI_ERR_INVALID_ARG,
               "spmi_linear_i8: null pointer or row stride too small");
  hipStream_t st = as_stream(stream);
  const bool f32 = dtype == SPMI_DTYPE_F32, of32 = out_dtype == SPMI_DTYPE_F32;
  if (few_made(M, K, N) || rows_take(M, K)) {  // one launch
    int rc;
    if (M <= kFewRows) {
      const FewArgs a{x, ldx, nullptr, static_cast<int>(M), weight, ldw, N, static_cast<int>(K), w_scale, bias, act, slope,
                      out, ldo};
      rc = f32 ? (of32 ? launch_few<float, float>(a, st) : launch_few<float, bf16>(a, st))
               : (of32 ? launch_few<bf16, float>(a, st) : launch_few<bf16, bf16>(a, st));
    } else {
      const RowsArgs a{x, ldx, M, weight, ldw, static_cast<int>(K), static_cast<int>(N), w_scale, bias, act, slope, out,
                       ldo};
      rc = f32 ? (of32 ? launch_rows<float, float>(a, st) : launch_rows<float, bf16>(a, st))
               : (of32 ? launch_rows<bf16, float>(a, st) : launch_rows<bf16, bf16>(a, st));
    }
    if (rc) return rc;
    SPMI_CHECK_LAUNCH("spmi_linear_i8");
    return SPMI_OK;
  }
  SPMI_REQUIRE(ws && ws_bytes >= spmi_linear_i8_workspace_bytes(M, K, N) && (reinterpret_cast<uintptr_t>(ws) & 15) == 0,
               SPMI_ERR_WORKSPACE, "spmi_linear_i8: workspace of %zu bytes is too small or not aligned to 16", ws_bytes);
  int8_t* q = static_cast<int8_t*>(ws);
  float* scale = reinterpret_cast<float*>(q + align_up(static_cast<size_t>(M) * padded(K), 256));
  launch_quantize(x, dtype, ldx, M, K, q, padded(K), padded(K), scale, st);
  SPMI_CHECK_LAUNCH("spmi_linear_i8");
  if (M <= kFewRows) {
    const FewArgs a{q, padded(K), scale, static_cast<int>(M), weight, ldw, N, static_cast<int>(K), w_scale, bias, act, slope,
                    out, ldo};
    if (int rc = of32 ? launch_few<int8_t, float>(a, st) : launch_few<int8_t, bf16>(a, st)) return rc;
    SPMI_CHECK_LAUNCH("spmi_linear_i8");
    return SPMI_OK;
  }
  // the tiles load 16 bytes of a weight row at a time, whole stages of 64
  if (K % 64 || ldw % 16 || (reinterpret_cast<uintptr_t>(weight) & 15)) {
    int8_t* const packed = reinterpret_cast<int8_t*>(scale) + align_up(static_cast<size_t>(M) * sizeof(float), 256);
    pack_weight_kernel<<<static_cast<unsigned>((N + 3) / 4 < 4096 ? (N + 3) / 4 : 4096), kThreads, 0, st>>>(
        weight, ldw, N, static_cast<int>(K), packed, padded(K));
    SPMI_CHECK_LAUNCH("spmi_linear_i8");
    weight = packed;
    ldw = padded(K);
  }
  GemmArgs a{q, padded(K), M, scale, weight, ldw, N, static_cast<int>(K), w_scale, bias, act, slope, out, ldo};
  if (int rc = of32 ? launch_tiles<float>(a, st) : launch_tiles<bf16>(a, st)) return rc;
  SPMI_CHECK_LAUNCH("spmi_linear_i8");
  return SPMI_OK;
}

}  // extern "C"
