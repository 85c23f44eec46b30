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
// 2048, a workgroup of 256 or 1024 threads beyond (16384 at most; the bfloat16 backward kernel of more than
// 8192 keeps four of its 132 registers in scratch).
//
// The gradients of w and b are column sums over all rows.  A lane sees the same columns in every
// row its group visits, so it adds them up in registers; the groups of a workgroup meet in LDS,
// the workgroups in a second launch that adds their partial rows in a fixed order.  No atomics:
// the same call gives the same bits.
//
// 10^6 x 128 in float32: 1.02 GB forward in 171-178 us (5.8-6.0 TB/s), 1.54 GB backward in 260-265 us and
// 11 us for the sums; a copy of that size in the same kind of grid reaches 6.7 TB/s.  12289 x 1031 in
// bfloat16 (rows that start at odd addresses): 51 MB in 17 us, 76 MB in 22.5 us and 4.

#include "lanes.h"

namespace {

using namespace spmi;

constexpr int kThreads = 256;
constexpr int64_t kMaxWidth = 16384;
constexpr int kGather = 64;    // partial rows that are added up in a step of their own
constexpr int kMaxLast = 512;  // partial rows that the last step takes
constexpr int64_t kMaxParts = 1 << 20;   // partial rows in all
constexpr int64_t kMaxGroups = 1 << 20;  // workgroups of a launch: a grid holds less than 2^32 threads

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
  int64_t rows;     // of a workgroup
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

// One row's values in registers: vectors r = 0 .. R - 1 of four values at column (r G + lane) 4.  LO is the
// width below which the kernel is not used, so the vectors below it exist without a question; the
// lanes of the others may lie past the row's end, entirely or in part.
template <int G, int R, int LO, bool STREAM, typename T>
__device__ __forceinline__ void hold_all(const T* src, int lane, int D, held<T> (&t)[R]) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = (r * G + lane) * 4;
    t[r] = (r + 1) * G * 4 <= LO ? hold4<STREAM>(src + c) : hold_row<STREAM>(src, c, D);
  }
}
template <int G, int R, int LO, typename T>
__device__ __forceinline__ void widen_all(const held<T> (&t)[R], int lane, int D, float (&v)[R][4]) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if ((r + 1) * G * 4 <= LO) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[r][i] = widen(t[r][i]);
    } else {
      widen_row<T>(t[r], (r * G + lane) * 4, D, v[r]);
    }
  }
}
template <int G, int R, int LO, bool STREAM, typename T>
__device__ __forceinline__ void load_row(const T* src, int lane, int D, float (&v)[R][4]) {
  held<T> t[R];
  hold_all<G, R, LO, STREAM>(src, lane, D, t);
  widen_all<G, R, LO, T>(t, lane, D, v);
}
template <int G, int R, int LO, bool STREAM, typename T>
__device__ __forceinline__ void store_row(T* dst, int lane, int D, const float (&v)[R][4]) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = (r * G + lane) * 4;
    if ((r + 1) * G * 4 <= LO) store4<STREAM>(dst + c, v[r]);
    else if (c < D) store4_upto<STREAM>(dst + c, D - c, v[r]);
  }
}

// A group works on RU rows at a time.  The grid covers the rows once (the loop is for more rows than a
// grid can hold): workgroups that are handed out in order keep the accesses in flight close together,
// where a resident grid that strides over the rows lets its workgroups drift apart.
template <typename T, int G, int R, int LO, int RU>
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
  if (p.w) {
    load_row<G, R, LO, false>(p.w, lane, p.D, w);
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[r][i] = 1.0f;
  }
  if (p.b) {
    load_row<G, R, LO, false>(p.b, lane, p.D, b);
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) b[r][i] = 0.0f;
  }
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * (GROUPS * RU); first < p.M;
       first += static_cast<int64_t>(gridDim.x) * (GROUPS * RU)) {
    const int64_t row0 = first + grp;
    held<T> raw[RU][R];
    float v[RU][R][4];
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int64_t row = row0 + u * GROUPS;  // past the end: the last row again, not stored
      hold_all<G, R, LO, true>(x + (row < p.M ? row : p.M - 1) * p.ldx, lane, p.D, raw[u]);
    }
#pragma unroll
    for (int u = 0; u < RU; ++u) widen_all<G, R, LO, T>(raw[u], lane, p.D, v[u]);
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int64_t row = row0 + u * GROUPS;
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
          v[u][r][i] -= mu;
          if ((r + 1) * G * 4 > LO && c + i >= p.D) v[u][r][i] = 0.0f;
          q = __builtin_fmaf(v[u][r][i], v[u][r][i], q);
        }
      }
      const float rs = 1.0f / sqrtf(row_sum<G, WG>(q, scratch, turn) * inv_d + p.eps);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[u][r][i] = __builtin_fmaf(v[u][r][i] * rs, w[r][i], b[r][i]);
      if (row < p.M) {
        if (p.stats && lane == 0) p.stats[row] = make_float2(mu, rs);
        store_row<G, R, LO, true>(y + row * p.ldy, lane, p.D, v[u]);
      }
    }
  }
}

// A workgroup takes `rows` neighbouring rows and leaves one row of partial sums for each of dw, db.
template <typename T, int G, int R, int LO>
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
  if (p.w) {
    load_row<G, R, LO, false>(p.w, lane, p.D, w);
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[r][i] = 1.0f;
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[r][i] = db[r][i] = 0.0f;

  const int64_t begin = static_cast<int64_t>(blockIdx.x) * p.rows;
  const int64_t end = begin + p.rows < p.M ? begin + p.rows : p.M;
  for (int64_t row0 = begin; row0 < end; row0 += GROUPS) {
    const int64_t row = row0 + grp;
    const bool there = row < end;  // else: a row's values with a gradient of zero
    const int64_t at = there ? row : end - 1;
    const float2 st = p.stats[at];
    float xh[R][4], gv[R][4];
    held<T> raw_x[R], raw_g[R];
    hold_all<G, R, LO, true>(x + at * p.ldx, lane, p.D, raw_x);
    hold_all<G, R, LO, true>(g + at * p.ldg, lane, p.D, raw_g);
    widen_all<G, R, LO, T>(raw_x, lane, p.D, xh);
    widen_all<G, R, LO, T>(raw_g, lane, p.D, gv);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float h = (xh[r][i] - st.x) * st.y;
        if ((r + 1) * G * 4 > LO && (r * G + lane) * 4 + i >= p.D) h = 0.0f;
        xh[r][i] = h;
        const float gi = there ? gv[r][i] : 0.0f;
        dw[r][i] = there ? __builtin_fmaf(gi, h, dw[r][i]) : dw[r][i];
        db[r][i] += gi;
        gv[r][i] = gi * w[r][i];
        s1 += gv[r][i];
        s2 = __builtin_fmaf(gv[r][i], h, s2);
      }
    }
    if (dx) {
      const float m1 = row_sum<G, WG>(s1, scratch, turn) * inv_d;
      const float m2 = row_sum<G, WG>(s2, scratch, turn) * inv_d;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) gv[r][i] = st.y * (gv[r][i] - m1 - xh[r][i] * m2);
      if (there) store_row<G, R, LO, true>(dx + row * p.lddx, lane, p.D, gv);
    }
  }

  if (!p.part) return;
  float* out = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.D;
  if constexpr (GROUPS == 1) {
    store_row<G, R, LO, false>(out, lane, p.D, dw);
    store_row<G, R, LO, false>(out + p.D, lane, p.D, db);
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

// Many partial rows: kGather of them into one, so that the last step has few to add.
__global__ __launch_bounds__(kThreads) void ln_bwd_gather_kernel(const float* __restrict__ part, int n_part, int64_t ld,
                                                                 float* __restrict__ out) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= ld) return;
  const int k0 = blockIdx.y * kGather, k1 = k0 + kGather < n_part ? k0 + kGather : n_part;
  float t = 0.0f;
#pragma unroll 8
  for (int k = k0; k < k1; ++k) t += part[k * ld + c];
  out[blockIdx.y * ld + c] = t;
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

// f(G, R, LO): lanes of a row, vectors of a lane, the width below which a narrower form is taken.
template <int G, int R, int LO>
struct Form {
  static constexpr int g = G, r = R, lo = LO;
};
template <typename F>
void with_form(int D, F f) {
  if (D <= 32) f(Form<8, 1, 0>{});
  else if (D <= 64) f(Form<16, 1, 32>{});
  else if (D <= 128) f(Form<32, 1, 64>{});
  else if (D <= 256) f(Form<64, 1, 128>{});
  else if (D <= 512) f(Form<64, 2, 256>{});
  else if (D <= 768) f(Form<64, 3, 512>{});
  else if (D <= 1024) f(Form<64, 4, 768>{});
  else if (D <= 1280) f(Form<64, 5, 1024>{});
  else if (D <= 1536) f(Form<64, 6, 1280>{});
  else if (D <= 2048) f(Form<64, 8, 1536>{});
  else if (D <= 4096) f(Form<256, 4, 2048>{});
  else if (D <= 8192) f(Form<256, 8, 4096>{});
  else f(Form<1024, 4, 8192>{});
}
constexpr int threads_of(int G) { return G > kThreads ? G : kThreads; }

template <typename T>
void launch_fwd(const FwdArgs& a, hipStream_t st) {
  with_form(a.D, [&](auto form) {
    using F = decltype(form);
    constexpr int RU = F::r == 1 ? 2 : 1, rows = threads_of(F::g) / F::g * RU;
    const int64_t groups = (a.M + rows - 1) / rows;
    ln_fwd_kernel<T, F::g, F::r, F::lo, RU>
        <<<static_cast<unsigned>(groups < kMaxGroups ? groups : kMaxGroups), threads_of(F::g), 0, st>>>(a);
  });
}

// Rows of a workgroup in the backward pass: enough workgroups for two on each CU, and up to 64 rows, so
// that the partial sums (8 D bytes a workgroup, written and read) stay small against the rows.
int64_t bwd_rows(int64_t M, int64_t D) {
  int64_t groups = 1;
  with_form(static_cast<int>(D), [&](auto form) { groups = threads_of(decltype(form)::g) / decltype(form)::g; });
  int64_t rows = (M + 511) / 512;
  rows = rows < 64 ? rows : 64;
  const int64_t least = (M + kMaxParts - 1) / kMaxParts;
  rows = rows > least ? rows : least;
  return (rows + groups - 1) / groups * groups;
}
int64_t bwd_parts(int64_t M, int64_t D) { return (M + bwd_rows(M, D) - 1) / bwd_rows(M, D); }

template <typename T>
void launch_bwd(const BwdArgs& a, hipStream_t st) {
  with_form(a.D, [&](auto form) {
    using F = decltype(form);
    ln_bwd_kernel<T, F::g, F::r, F::lo>
        <<<static_cast<unsigned>(bwd_parts(a.M, a.D)), threads_of(F::g), 0, st>>>(a);
  });
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
  if (dtype == SPMI_DTYPE_F32) launch_fwd<float>(a, as_stream(stream));
  else launch_fwd<bf16>(a, as_stream(stream));
  SPMI_CHECK_LAUNCH("spmi_layer_norm_fwd");
  return SPMI_OK;
}

size_t spmi_layer_norm_bwd_workspace_bytes(int64_t M, int64_t D) {
  if (M <= 0 || D <= 0 || D > kMaxWidth) return 0;
  const int64_t parts = bwd_parts(M, D);
  return static_cast<size_t>(parts + (parts > kMaxLast ? (parts + kGather - 1) / kGather : 0)) * 2 *
         static_cast<size_t>(D) * sizeof(float);
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
            bwd_rows(M, D), sums ? static_cast<float*>(ws) : nullptr};
  if (dtype == SPMI_DTYPE_F32) launch_bwd<float>(a, st);
  else launch_bwd<bf16>(a, st);
  SPMI_CHECK_LAUNCH("spmi_layer_norm_bwd");
  if (sums) {
    const float* part = a.part;
    int parts = static_cast<int>(bwd_parts(M, D));
    if (parts > kMaxLast) {
      float* const gathered = a.part + static_cast<int64_t>(parts) * 2 * D;
      const dim3 grid(static_cast<unsigned>((2 * D + kThreads - 1) / kThreads), (parts + kGather - 1) / kGather);
      ln_bwd_gather_kernel<<<grid, kThreads, 0, st>>>(part, parts, 2 * D, gathered);
      SPMI_CHECK_LAUNCH("spmi_layer_norm_bwd");
      part = gathered;
      parts = (parts + kGather - 1) / kGather;
    }
    ln_bwd_reduce_kernel<<<static_cast<unsigned>((2 * D + 15) / 16), kThreads, 0, st>>>(part, parts, a.D, dweight,
                                                                                        dbias);
    SPMI_CHECK_LAUNCH("spmi_layer_norm_bwd");
  }
  return SPMI_OK;
}

}  // extern "C"
