// Layer norm of the rows of a matrix, forward and backward:
//
//   mu = mean(x), v = mean((x - mu)^2), r = (v + eps)^-1/2, xh = (x - mu) r, y = xh w + b
//   dx = r (g w - mean(g w) - xh mean(g w xh)),  dw = sum over rows of g xh,  db = sum of g
//
// Both directions are bound by memory: forward reads x and writes y, backward reads x and g and
// writes dx.  A row therefore stays in registers between its load and its store, whatever is
// computed from it: the mean first and then the centred squares (a single pass over E[x^2] would
// cancel for rows whose mean is large against their deviation), all in float32 for either storage
// type.  G neighbouring lanes own a row, four values of R vectors each: G = 8..64 for widths up to
// 2048, a workgroup of 256 or 1024 threads beyond (16384 at most).
//
// The gradients of w and b are column sums over all rows.  A lane sees the same columns in every
// row its group visits, so it adds them up in registers; the groups of a workgroup meet in LDS,
// the workgroups in a second launch that adds their partial rows in a fixed order.  No atomics:
// the same call gives the same bits.

#include "lanes.h"

namespace {

using namespace spmi;

constexpr int kThreads = 256;
constexpr int64_t kMaxWidth = 16384;
// Workgroups of the backward pass, i.e. rows of partial sums.
constexpr int64_t kBwdBlocks = 1024;

struct FwdArgs {
  const void* x;
  int64_t ldx, M;
  int D;
  const float* w;   // nullable: ones
  const float* b;   // nullable: zeros
  float eps;
  void* y;
  int64_t ldy;
  float2* stats;    // nullable: mean and r of each row
};

struct BwdArgs {
  const void *x, *g;
  int64_t ldx, ldg, M;
  int D;
  const float* w;   // nullable: ones
  const float2* stats;
  void* dx;         // nullable
  int64_t lddx;
  float* part;      // nullable: [gridDim.x][2][D] sums of g xh and of g
};

// The sum over the G lanes (or the whole workgroup: WG) of a row.  `turn` alternates between two
// LDS rows, so that one barrier a call is enough.
template <int G, bool WG>
__device__ __forceinline__ float row_sum(float v, float* scratch, int& turn) {
  if constexpr (!WG) {
    return group_sum<G>(v);
  } else {
    constexpr int W = G / 64;
    v = group_sum<64>(v);
    float* s = scratch + turn * W;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = s[0];
#pragma unroll
    for (int i = 1; i < W; ++i) t += s[i];
    return t;
  }
}

// RU rows of a group are in flight together.
template <typename T, int G, int R, int RU>
__global__ __launch_bounds__(G > kThreads ? G : kThreads) void ln_fwd_kernel(FwdArgs p) {
  constexpr bool WG = G > 64;
  constexpr int THREADS = G > kThreads ? G : kThreads;
  constexpr int GROUPS = THREADS / G;
  __shared__ float scratch[WG ? 2 * (G / 64) : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, grp = threadIdx.x / G;
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  const float inv_d = 1.0f / static_cast<float>(p.D);

  float w[R][4], b[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = (r * G + lane) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[r][i] = (p.w && c + i < p.D) ? p.w[c + i] : 1.0f;
      b[r][i] = (p.b && c + i < p.D) ? p.b[c + i] : 0.0f;
    }
  }

  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * (GROUPS * RU); row0 < p.M;
       row0 += static_cast<int64_t>(gridDim.x) * (GROUPS * RU)) {
    float v[RU][R][4];
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int64_t row = row0 + u * GROUPS + grp;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int c = (r * G + lane) * 4;
        if (row < p.M && c < p.D) {
          load4_upto(x + row * p.ldx + c, p.D - c, 0.0f, v[u][r]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[u][r][i] = 0.0f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int64_t row = row0 + u * GROUPS + grp;
      float s = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r) s += (v[u][r][0] + v[u][r][1]) + (v[u][r][2] + v[u][r][3]);
      const float mu = row_sum<G, WG>(s, scratch, turn) * inv_d;
      float q = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int c = (r * G + lane) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[u][r][i] = c + i < p.D ? v[u][r][i] - mu : 0.0f;
          q = __builtin_fmaf(v[u][r][i], v[u][r][i], q);
        }
      }
      const float rs = 1.0f / sqrtf(row_sum<G, WG>(q, scratch, turn) * inv_d + p.eps);
      if (row < p.M) {
        if (p.stats && lane == 0) p.stats[row] = make_float2(mu, rs);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int c = (r * G + lane) * 4;
          if (c < p.D) {
            float o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(v[u][r][i] * rs, w[r][i], b[r][i]);
            store4_upto(y + row * p.ldy + c, p.D - c, o);
          }
        }
      }
    }
  }
}

template <typename T, int G, int R>
__global__ __launch_bounds__(G > kThreads ? G : kThreads) void ln_bwd_kernel(BwdArgs p) {
  constexpr bool WG = G > 64;
  constexpr int THREADS = G > kThreads ? G : kThreads;
  constexpr int GROUPS = THREADS / G;
  constexpr int COLS = G * R * 4;
  __shared__ float scratch[WG ? 2 * (G / 64) : GROUPS * COLS];
  int turn = 0;
  const int lane = threadIdx.x % G, grp = threadIdx.x / G;
  const T* x = static_cast<const T*>(p.x);
  const T* g = static_cast<const T*>(p.g);
  T* dx = static_cast<T*>(p.dx);
  const float inv_d = 1.0f / static_cast<float>(p.D);

  float w[R][4], dw[R][4], db[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = (r * G + lane) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[r][i] = (p.w && c + i < p.D) ? p.w[c + i] : 1.0f;
      dw[r][i] = db[r][i] = 0.0f;
    }
  }

  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * GROUPS; row0 < p.M; row0 += step) {
    const int64_t row = row0 + grp;
    const bool there = row < p.M;
    const float2 st = there ? p.stats[row] : make_float2(0.0f, 0.0f);
    float xh[R][4], gv[R][4];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int c = (r * G + lane) * 4;
      if (there && c < p.D) {
        load4_upto(x + row * p.ldx + c, p.D - c, st.x, xh[r]);
        load4_upto(g + row * p.ldg + c, p.D - c, 0.0f, gv[r]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { xh[r][i] = st.x; gv[r][i] = 0.0f; }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float h = (xh[r][i] - st.x) * st.y;
        xh[r][i] = h;
        dw[r][i] = __builtin_fmaf(gv[r][i], h, dw[r][i]);
        db[r][i] += gv[r][i];
        gv[r][i] *= w[r][i];
        s1 += gv[r][i];
        s2 = __builtin_fmaf(gv[r][i], h, s2);
      }
    }
    if (dx) {
      const float m1 = row_sum<G, WG>(s1, scratch, turn) * inv_d;
      const float m2 = row_sum<G, WG>(s2, scratch, turn) * inv_d;
      if (there) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int c = (r * G + lane) * 4;
          if (c < p.D) {
            float o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = st.y * (gv[r][i] - m1 - xh[r][i] * m2);
            store4_upto(dx + row * p.lddx + c, p.D - c, o);
          }
        }
      }
    }
  }

  if (!p.part) return;
  float* out = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.D;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int c = (r * G + lane) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < p.D) {
          out[c + i] = dw[r][i];
          out[p.D + c + i] = db[r][i];
        }
    }
  } else {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          scratch[grp * COLS + (r * G + lane) * 4 + i] = half ? db[r][i] : dw[r][i];
      __syncthreads();
      for (int c = threadIdx.x; c < p.D; c += THREADS) {
        float s = scratch[c];
#pragma unroll 8
        for (int q = 1; q < GROUPS; ++q) s += scratch[q * COLS + c];
        out[half * p.D + c] = s;
      }
    }
  }
}

// Column sums of the partial rows: out[c] = sum over k of part[k][c], c < 2 D (dw, then db).  A
// workgroup owns 16 columns; 16 strands of 4-row steps keep the loads independent.
__global__ __launch_bounds__(kThreads) void ln_bwd_reduce_kernel(const float* __restrict__ part, int n_part, int D,
                                                                 float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float s[16][17];
  const int col = threadIdx.x & 15, strand = threadIdx.x >> 4;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 16 + col;
  const int64_t ld = 2 * static_cast<int64_t>(D);
  float t = 0.0f;
  if (c < ld) {
#pragma unroll 8
    for (int k = strand; k < n_part; k += 16) t += part[k * ld + c];
  }
  s[strand][col] = t;
  __syncthreads();
  if (strand == 0 && c < ld) {
#pragma unroll
    for (int q = 1; q < 16; ++q) t += s[q][col];
    if (c < D) {
      if (dw) dw[c] = t;
    } else if (db) {
      db[c - D] = t;
    }
  }
}

int64_t fwd_grid(int64_t M, int rows) {
  const int64_t need = (M + rows - 1) / rows;
  return need < 2048 ? need : 2048;
}

template <typename T, int G, int R, int RU>
void launch_fwd(const FwdArgs& a, hipStream_t st) {
  constexpr int THREADS = G > kThreads ? G : kThreads;
  ln_fwd_kernel<T, G, R, RU><<<fwd_grid(a.M, THREADS / G * RU), THREADS, 0, st>>>(a);
}

template <typename T>
void dispatch_fwd(const FwdArgs& a, hipStream_t st) {
  if (a.D <= 32) launch_fwd<T, 8, 1, 2>(a, st);
  else if (a.D <= 64) launch_fwd<T, 16, 1, 2>(a, st);
  else if (a.D <= 128) launch_fwd<T, 32, 1, 2>(a, st);
  else if (a.D <= 256) launch_fwd<T, 64, 1, 2>(a, st);
  else if (a.D <= 512) launch_fwd<T, 64, 2, 1>(a, st);
  else if (a.D <= 1024) launch_fwd<T, 64, 4, 1>(a, st);
  else if (a.D <= 2048) launch_fwd<T, 64, 8, 1>(a, st);
  else if (a.D <= 4096) launch_fwd<T, 256, 4, 1>(a, st);
  else if (a.D <= 8192) launch_fwd<T, 256, 8, 1>(a, st);
  else launch_fwd<T, 1024, 4, 1>(a, st);
}

int64_t bwd_groups(int64_t D) {  // rows a workgroup works on at once
  return D <= 32 ? 32 : D <= 64 ? 16 : D <= 128 ? 8 : D <= 2048 ? 4 : 1;
}
int64_t bwd_grid(int64_t M, int64_t D) {
  const int64_t need = (M + bwd_groups(D) - 1) / bwd_groups(D);
  return need < kBwdBlocks ? need : kBwdBlocks;
}

template <typename T, int G, int R>
void launch_bwd(const BwdArgs& a, hipStream_t st) {
  ln_bwd_kernel<T, G, R><<<bwd_grid(a.M, a.D), G > kThreads ? G : kThreads, 0, st>>>(a);
}

template <typename T>
void dispatch_bwd(const BwdArgs& a, hipStream_t st) {
  if (a.D <= 32) launch_bwd<T, 8, 1>(a, st);
  else if (a.D <= 64) launch_bwd<T, 16, 1>(a, st);
  else if (a.D <= 128) launch_bwd<T, 32, 1>(a, st);
  else if (a.D <= 256) launch_bwd<T, 64, 1>(a, st);
  else if (a.D <= 512) launch_bwd<T, 64, 2>(a, st);
  else if (a.D <= 1024) launch_bwd<T, 64, 4>(a, st);
  else if (a.D <= 2048) launch_bwd<T, 64, 8>(a, st);
  else if (a.D <= 4096) launch_bwd<T, 256, 4>(a, st);
  else if (a.D <= 8192) launch_bwd<T, 256, 8>(a, st);
  else launch_bwd<T, 1024, 4>(a, st);
}

__global__ void zero_kernel(float* a, float* b, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) {
    if (a) a[i] = 0.0f;
    if (b) b[i] = 0.0f;
  }
}

int check_rows(const char* what, int dtype, int64_t M, int64_t D) {
  SPMI_REQUIRE(dtype == SPMI_DTYPE_F32 || dtype == SPMI_DTYPE_BF16, SPMI_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  SPMI_REQUIRE(M >= 0 && D >= 1, SPMI_ERR_INVALID_ARG, "%s: M=%lld D=%lld", what, (long long)M, (long long)D);
  SPMI_REQUIRE(D <= kMaxWidth, SPMI_ERR_UNSUPPORTED, "%s: rows of %lld values, at most %lld", what, (long long)D,
               (long long)kMaxWidth);
  return SPMI_OK;
}

}  // namespace

extern "C" {

int64_t spmi_layer_norm_max_width(void) { return kMaxWidth; }

int spmi_layer_norm_fwd(const void* x, int dtype, int64_t ldx, int64_t M, int64_t D, const float* weight,
                        const float* bias, float eps, void* y, int64_t ldy, float* stats, void* stream) {
  if (int rc = check_rows("spmi_layer_norm_fwd", dtype, M, D)) return rc;
  if (M == 0) return SPMI_OK;
  SPMI_REQUIRE(x && y && ldx >= 0 && ldy >= D && eps >= 0.0f, SPMI_ERR_INVALID_ARG,
               "spmi_layer_norm_fwd: null pointer, negative eps or row stride too small");
  FwdArgs a{x, ldx, M, static_cast<int>(D), weight, bias, eps, y, ldy, reinterpret_cast<float2*>(stats)};
  if (dtype == SPMI_DTYPE_F32) dispatch_fwd<float>(a, as_stream(stream));
  else dispatch_fwd<bf16>(a, as_stream(stream));
  SPMI_CHECK_LAUNCH("spmi_layer_norm_fwd");
  return SPMI_OK;
}

size_t spmi_layer_norm_bwd_workspace_bytes(int64_t M, int64_t D) {
  if (M <= 0 || D <= 0) return 0;
  return static_cast<size_t>(bwd_grid(M, D)) * 2 * static_cast<size_t>(D) * sizeof(float);
}

int spmi_layer_norm_bwd(const void* x, const void* g, int dtype, int64_t ldx, int64_t ldg, int64_t M, int64_t D,
                        const float* weight, const float* stats, void* dx, int64_t lddx, float* dweight,
                        float* dbias, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_rows("spmi_layer_norm_bwd", dtype, M, D)) return rc;
  hipStream_t st = as_stream(stream);
  const bool sums = dweight || dbias;
  if (M == 0) {
    if (sums) {
      zero_kernel<<<(D + 255) / 256, 256, 0, st>>>(dweight, dbias, static_cast<int>(D));
      SPMI_CHECK_LAUNCH("spmi_layer_norm_bwd");
    }
    return SPMI_OK;
  }
  SPMI_REQUIRE(x && g && stats && ldx >= 0 && ldg >= 0 && (!dx || lddx >= D), SPMI_ERR_INVALID_ARG,
               "spmi_layer_norm_bwd: null pointer or row stride too small");
  SPMI_REQUIRE(!sums || (ws && ws_bytes >= spmi_layer_norm_bwd_workspace_bytes(M, D)), SPMI_ERR_WORKSPACE,
               "spmi_layer_norm_bwd: workspace of %zu bytes is too small", ws_bytes);
  BwdArgs a{x, g, ldx, ldg, M, static_cast<int>(D), weight, reinterpret_cast<const float2*>(stats), dx, lddx,
            sums ? static_cast<float*>(ws) : nullptr};
  if (dtype == SPMI_DTYPE_F32) dispatch_bwd<float>(a, st);
  else dispatch_bwd<bf16>(a, st);
  SPMI_CHECK_LAUNCH("spmi_layer_norm_bwd");
  if (sums) {
    ln_bwd_reduce_kernel<<<static_cast<unsigned>((2 * D + 15) / 16), kThreads, 0, st>>>(
        a.part, static_cast<int>(bwd_grid(M, D)), a.D, dweight, dbias);
    SPMI_CHECK_LAUNCH("spmi_layer_norm_bwd");
  }
  return SPMI_OK;
}

}  // extern "C"
