// The projection in 8-bit integers: y = act(s_m s_n sum_k q_mk w_nk + b_n) with whole numbers
// q = rint(x * (127 / m)) of each row of x, its scale s_m = m / 127 (m the row's largest
// magnitude), and a weight w with a scale s_n for each output channel.
//
// Sums of products are exact in 32-bit integers up to K = 131072 (127^2 K < 2^31), so neither the
// order of a sum nor its split changes a result: what is rounded is q, and the three float32
// operations of the last step.

#include "lanes.h"

namespace {

using namespace spmi;

using i32x4 = int __attribute__((ext_vector_type(4)));
using i32x16 = int __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int64_t kMaxInner = 131072;
// Smallest row maximum that is divided by: 127 / 2^-120 is still finite.
constexpr float kTiny = 0x1p-120f;

__device__ __forceinline__ float top_of(float m, float v) {
  // the larger magnitude; not-a-number stays
  const float a = __builtin_fabsf(v);
  return (a > m || a != a) ? a : m;
}
__device__ __forceinline__ void row_scale(float top, float& inv, float& scale) {
  const float m = top > kTiny ? top : (top != top ? top : kTiny);
  const bool fine = m <= 3.40282347e38f;
  inv = fine ? 127.0f / m : 0.0f;
  scale = fine ? m / 127.0f : __builtin_nanf("");  // a row that is not finite comes out as NaN
}
__device__ __forceinline__ int eight_bits(float v, float inv) {
  // inv is 0 for a row that is not finite: NaN (0 * inf) must not reach the conversion
  const float t = __builtin_rintf(v * inv);
  return inv == 0.0f ? 0 : static_cast<int>(t);
}
__device__ __forceinline__ unsigned pack4(const float (&v)[4], float inv) {
  unsigned r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= (static_cast<unsigned>(eight_bits(v[i], inv)) & 255u) << (8 * i);
  return r;
}

// q [M, width] (width >= K, zero past K) and the rows' scales.  A wave per row.
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t M, int K,
                                                            int8_t* __restrict__ q, int64_t ldq, int width,
                                                            float* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  for (int64_t row = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 6; row < M;
       row += (static_cast<int64_t>(gridDim.x) * kThreads) >> 6) {
    const T* src = x + row * ldx;
    float top = 0.0f;
    for (int c = lane * 4; c < K; c += 256) {
      float v[4];
      load4_upto(src + c, K - c, 0.0f, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) top = top_of(top, v[i]);
    }
    top = group_reduce<64>(top, [](float a, float b) { return top_of(a, b); });
    float inv, s;
    row_scale(top, inv, s);
    if (lane == 0) scale[row] = s;
    int8_t* dst = q + row * ldq;
    for (int c = lane * 4; c < width; c += 256) {
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (c < K) load4_upto(src + c, K - c, 0.0f, v);
      const unsigned w = pack4(v, inv);
      if (c + 4 <= width) {
        __builtin_memcpy(dst + c, &w, 4);
      } else {
        for (int i = 0; c + i < width; ++i) dst[c + i] = static_cast<int8_t>(w >> (8 * i));
      }
    }
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

// A scale as significand and power of two.  The sum of products times two scales is formed from the
// significands, the powers are added and applied at the end: with scales from 2^-127 to 2^121 a
// product of all three in any order could leave float32's range half way, although y lies inside.
struct Scale {
  float f;
  int e;
  __device__ Scale() = default;
  __device__ explicit Scale(float s) : f(__builtin_amdgcn_frexp_mantf(s)), e(__builtin_amdgcn_frexp_expf(s)) {}
};

__device__ __forceinline__ float finish(const GemmArgs& p, int acc, Scale sa, Scale sw, float bias) {
  float y = __builtin_amdgcn_ldexpf(static_cast<float>(acc) * sa.f * sw.f, sa.e + sw.e) + bias;
  if (p.act == SPMI_ACT_RELU) y = y < 0.0f ? 0.0f : y;
  if (p.act == SPMI_ACT_LEAKY_RELU) y = y < 0.0f ? y * p.slope : y;
  return y;
}

// Sixteen neighbouring whole numbers of a row of which `left` exist, the others zero.
__device__ __forceinline__ i32x4 load16_upto(const int8_t* src, int left) {
  i32x4 v = {0, 0, 0, 0};
  if (left >= 16) {
    __builtin_memcpy(&v, src, 16);
  } else {
    unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (i < left) w[i >> 2] |= (static_cast<unsigned>(src[i]) & 255u) << (8 * (i & 3));
    v = i32x4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
  }
  return v;
}

// 64 x 64 outputs per workgroup, 32 x 32 per wave.
template <typename OUT>
__global__ __launch_bounds__(kThreads) void gemm_i8_kernel(GemmArgs p) {
  __shared__ i32x4 sa[64 * 5], sw[64 * 5];  // rows of 64 bytes, padded to 80
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * 64, n0 = static_cast<int64_t>(blockIdx.y) * 64;
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  i32x16 acc = {0};
  const int row = tid >> 2, piece = tid & 3;
  for (int k0 = 0; k0 < p.K; k0 += 64) {
    const int k = k0 + piece * 16;
    i32x4 va = {0, 0, 0, 0}, vw = {0, 0, 0, 0};
    if (m0 + row < p.M) __builtin_memcpy(&va, p.a + (m0 + row) * p.lda + k, 16);
    if (n0 + row < p.N) vw = load16_upto(p.w + (n0 + row) * p.ldw + k, p.K - k);
    __syncthreads();
    sa[row * 5 + piece] = va;
    sw[row * 5 + piece] = vw;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const i32x4 fa = sa[(wm + (lane & 31)) * 5 + h * 2 + (lane >> 5)];
      const i32x4 fw = sw[(wn + (lane & 31)) * 5 + h * 2 + (lane >> 5)];
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa, fw, acc, 0, 0, 0);
    }
  }
  const int64_t n = n0 + wn + (lane & 31);
  if (n >= p.N) return;
  const Scale s_n(p.w_scale[n]);
  const float b = p.bias ? p.bias[n] : 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t m = m0 + wm + 8 * (r / 4) + 4 * (lane >> 5) + (r % 4);
    if (m < p.M) static_cast<OUT*>(p.out)[m * p.ldo + n] = static_cast<OUT>(finish(p, acc[r], Scale(p.a_scale[m]), s_n, b));
  }
}

int64_t padded(int64_t K) { return (K + 63) / 64 * 64; }

int check_rows(const char* what, int dtype, int64_t M, int64_t K) {
  SPMI_REQUIRE(dtype == SPMI_DTYPE_F32 || dtype == SPMI_DTYPE_BF16, SPMI_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  SPMI_REQUIRE(M >= 0 && K >= 1, SPMI_ERR_INVALID_ARG, "%s: M=%lld K=%lld", what, (long long)M, (long long)K);
  SPMI_REQUIRE(K <= kMaxInner && M < (1ll << 31), SPMI_ERR_UNSUPPORTED,
               "%s: %lld rows of %lld values (at most 2^31 - 1 rows of %lld)", what, (long long)M, (long long)K,
               (long long)kMaxInner);
  return SPMI_OK;
}

void launch_quantize(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, int8_t* q, int64_t ldq,
                     int64_t width, float* scale, hipStream_t st) {
  const int64_t need = (M + 3) / 4;
  const unsigned grid = static_cast<unsigned>(need < 8192 ? need : 8192);
  if (dtype == SPMI_DTYPE_F32)
    quantize_kernel<float><<<grid, kThreads, 0, st>>>(static_cast<const float*>(x), ldx, M, static_cast<int>(K), q,
                                                      ldq, static_cast<int>(width), scale);
  else
    quantize_kernel<bf16><<<grid, kThreads, 0, st>>>(static_cast<const bf16*>(x), ldx, M, static_cast<int>(K), q, ldq,
                                                     static_cast<int>(width), scale);
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
  return align_up(static_cast<size_t>(M) * padded(K), 256) + static_cast<size_t>(M) * sizeof(float);
}

int spmi_linear_i8(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, const int8_t* weight, int64_t ldw,
                   const float* w_scale, int64_t N, const float* bias, int act, float slope, void* out, int out_dtype,
                   int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_rows("spmi_linear_i8", dtype, M, K)) return rc;
  SPMI_REQUIRE(N >= 0 && N < (1ll << 31), SPMI_ERR_INVALID_ARG, "spmi_linear_i8: N=%lld", (long long)N);
  SPMI_REQUIRE(out_dtype == SPMI_DTYPE_F32 || out_dtype == SPMI_DTYPE_BF16, SPMI_ERR_INVALID_ARG,
               "spmi_linear_i8: out_dtype %d", out_dtype);
  SPMI_REQUIRE(act >= SPMI_ACT_NONE && act <= SPMI_ACT_LEAKY_RELU, SPMI_ERR_INVALID_ARG, "spmi_linear_i8: act %d", act);
  if (M == 0 || N == 0) return SPMI_OK;
  SPMI_REQUIRE(x && weight && w_scale && out && ldx >= 0 && ldw >= 0 && ldo >= N, SPMI_ERR_INVALID_ARG,
               "spmi_linear_i8: null pointer or row stride too small");
  SPMI_REQUIRE(ws && ws_bytes >= spmi_linear_i8_workspace_bytes(M, K, N) && (reinterpret_cast<uintptr_t>(ws) & 15) == 0,
               SPMI_ERR_WORKSPACE, "spmi_linear_i8: workspace of %zu bytes is too small or not aligned to 16", ws_bytes);
  SPMI_REQUIRE((N + 63) / 64 < 65536, SPMI_ERR_UNSUPPORTED, "spmi_linear_i8: N=%lld is too large", (long long)N);
  hipStream_t st = as_stream(stream);
  int8_t* q = static_cast<int8_t*>(ws);
  float* scale = reinterpret_cast<float*>(q + align_up(static_cast<size_t>(M) * padded(K), 256));
  launch_quantize(x, dtype, ldx, M, K, q, padded(K), padded(K), scale, st);
  SPMI_CHECK_LAUNCH("spmi_linear_i8");
  GemmArgs a{q, padded(K), M, scale, weight, ldw, N, static_cast<int>(K), w_scale, bias, act, slope, out, ldo};
  const dim3 grid(static_cast<unsigned>((M + 63) / 64), static_cast<unsigned>((N + 63) / 64));
  if (out_dtype == SPMI_DTYPE_F32) gemm_i8_kernel<float><<<grid, kThreads, 0, st>>>(a);
  else gemm_i8_kernel<bf16><<<grid, kThreads, 0, st>>>(a);
  SPMI_CHECK_LAUNCH("spmi_linear_i8");
  return SPMI_OK;
}

}  // extern "C"
