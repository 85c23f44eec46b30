// The gated linear recurrence over a sequence, forward and backward, and its single step on the
// node memory.  With gate logits z and candidates c (one projection's output, [.., 2H]):
//
//   a = sigmoid(z),  h_t = a_t h_{t-1} + (1 - a_t) c_t          per node and hidden unit
//   backward, with e = the gradient that arrives at h_t from later steps:
//   d = g_t + e,  dc = d (1 - a),  dz = d (h_{t-1} - c) a (1 - a),  e <- a d
//
// Nothing here depends on h but h itself, so both directions are a chain of maps v -> p v + q that
// can be joined pairwise: a stretch of steps is one such map (p = product of the a, q = what the
// stretch makes of zero).  Both are bound by memory (forward: two values in, one out per unit and
// step; backward: three in, two out, and a state for every group of steps), and the design is about
// having enough loads in flight while every value is read once:
//  * many channels: a thread owns four neighbouring units of one node and walks the steps; the
//    loads of several steps are issued together;
//  * few channels (a long sequence of one or a few nodes): a workgroup is 8 strands of 32 lanes.
//    A strand takes consecutive steps of a tile into registers, reduces them to its map, the maps
//    meet in LDS, and each strand replays its steps from the registers with the right start: the
//    inputs are still read once;
//  * very few channels: the steps are also split over workgroups.  A first launch leaves the map
//    of each split in a workspace (this reads the gates, and backward the gradients, a second
//    time: mostly from the caches, since a problem of few channels is a small one), a second
//    launch starts every split from the joined maps before it.  No workgroup waits for another.
//
// a and 1 - a are computed from exp(-|z|), so neither loses digits where it is small; the state, its
// gradient and the maps are float32 whatever the storage type, and a state is rounded only when it
// is stored for the caller.  dz takes the difference h_{t-1} - c, which cancels where a state follows its
// candidates, so the backward pass reads no rounded state: it makes the states of a group of steps again,
// by the forward pass's arithmetic, from the float32 state before the group.  That is the row of h itself
// in float32; for bfloat16 the forward pass leaves it beside h, one state for 4 steps walked (half a value
// of bfloat16 a step) and for 2 of a strand.
//
// Steps where a node is not active pass the state (and its gradient) on unchanged; what stands in the
// gates there is never used.

#include "lanes.h"

namespace {

using namespace spmi;

constexpr int kThreads = 256;
// Steps a thread holds in registers.  Walking, the loads of the next steps are sent before the stores of
// the present ones: 32 x 50000 x 128 takes 481 us forward and 1253 trained in float32, 238 and 668 in
// bfloat16 (with 2 steps backward 1319 and 767; forward in float32 without the loads ahead 494, with 2
// steps 488).  As one of the strands, other waves cover the wait better than registers do (1185 x 2255 x 30
// trained in bfloat16 takes 482 us with four waves to a SIMD; with six the registers spill, 1.4 times as
// long), and more steps pay less than they cost: 65536 x 1 x 128 42 us with 2 forward, 49 with 4;
// 1601 x 717 x 64 trained in float32 667 with 2 backward, 1.2 times as long with 4.
constexpr int kFwdSteps = 2;
constexpr int kFwdWalkSteps = 4;
constexpr int kBwdSteps = 2;
constexpr int kBwdWalkSteps = 4;
// Backward they are also a group: the states inside one are made again from the one before it.
template <bool WALK>
constexpr int kGroup = WALK ? kBwdWalkSteps : kBwdSteps;
constexpr int kLanes = 32;     // shape of a workgroup over few channels: lanes x strands
constexpr int kStrands = kThreads / kLanes;
// Threads (of four units) from which the steps are walked by one thread each: one wave per SIMD.
constexpr int64_t kManyLanes = 65536;
// Up to this many steps there is nothing to share among the strands.
constexpr int64_t kFewSteps = 16;
// Workgroups from which the steps are not split: two per CU (852 x 221 x 448 in bfloat16, 774 workgroups, takes
// 139 us unsplit and 188 in two, which read the gates twice).  Below, as many splits as make kTargetGroups
// (1601 x 717 x 64, 359 workgroups, trained in bfloat16 410 us in five, a sixth longer in two).
constexpr int64_t kEnoughGroups = 512;
constexpr int64_t kTargetGroups = 2048;
constexpr int64_t kMaxSplits = 512;

struct ScanArgs {
  const void* gates;   // [T, N, 2H]: z, then c
  int64_t gates_t, gates_n;
  const float* h0;     // nullable, [N, H]
  int64_t h0_n;
  const uint8_t* active;  // nullable, [T, N]
  int64_t active_t, active_n;
  void* h;             // forward: [T, N, H]
  int64_t h_t, h_n;
  float* last;         // forward: [N, H]
  float* states;       // forward, nullable, [groups - 1, N, H]: the state before each group but the first
  const float* before; // backward: the same, with strides before_g, before_n (null if there is one group)
  int64_t before_g, before_n;
  const void* g;       // backward, nullable: gradient of h
  int64_t g_t, g_n;
  const float* g_last; // backward, nullable, [N, H]
  int64_t gl_n;
  void* dgates;        // backward, nullable, strides dg_t, dg_n
  int64_t dg_t, dg_n;
  float* dh0;          // backward, nullable, [N, H]
  int64_t T, N;
  int H, Hq;           // Hq = groups of four units per node
  int64_t per_split;   // steps of a split
  int splits;
  float* maps;         // [splits][2][lanes][4]: p, then q
};

// e^-|z| to about one unit in the last place down to the smallest normal number, |z| = 87 (0 below it): what the
// float32 log2(e) and its product with the exponent leave out is put back.  (The constant's own error
// alone, 1.3e-8 |z|, is 18 half units at |z| = 80.)
__device__ __forceinline__ void gate_pair(float z, float& a, float& rest) {
  const float m = -__builtin_fabsf(z);
  const float y = m * 1.44269504f;
  const float err = __builtin_fmaf(m, 1.925963e-8f, __builtin_fmaf(m, 1.44269504f, -y));
  float e = __builtin_amdgcn_exp2f(y);
  // (the correction is below 10^-5 where e is not 0; kept finite where y has overflowed)
  e = __builtin_fmaf(e, __builtin_amdgcn_fmed3f(err * 0.693147181f, -1.0f, 1.0f), e);
  const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  a = z >= 0.0f ? big : small;
  rest = z >= 0.0f ? small : big;
}

// What a thread works on: four units of one node.  The last four of a row whose length is no multiple
// of four reach back into the units of the thread before: both compute the same bits from the same
// inputs and write them to the same places, and no access has an end to look at.  (Rows of fewer than
// four units do: `left`, the same for all.)
struct Place {
  bool there;
  int64_t n;
  int c, left;
  __device__ Place(const ScanArgs& p, int64_t lane) {
    there = lane < p.N * p.Hq;
    n = there ? lane / p.Hq : 0;
    c = there ? static_cast<int>(lane - n * p.Hq) * 4 : 0;
    if (p.H >= 4 && c > p.H - 4) c = p.H - 4;
    left = p.H < 4 ? p.H : 4;
  }
};

// TINY: rows of fewer than four units.
template <bool STREAM, bool TINY, typename T>
__device__ __forceinline__ held<T> take(const T* p, int left) {
  held<T> v;
  if constexpr (TINY) {
    const auto* q = reinterpret_cast<const std::conditional_t<sizeof(T) == 4, float, unsigned short>*>(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = q[k < left ? k : left - 1];
  } else {
    v = hold4<STREAM>(p);
  }
  return v;
}
template <bool TINY, typename T>
__device__ __forceinline__ void put(T* p, int left, const float (&v)[4]) {
  if constexpr (TINY) store4_upto(p, left, v);
  else store4<true>(p, v);
}

// Forward.  C lanes x S strands; MAPS: only the map of the split is wanted.
template <typename T, int C, int S, bool MAPS, bool TINY>
__global__ __launch_bounds__(kThreads, S > 1 ? 4 : 1) void scan_fwd_kernel(ScanArgs p) {
  constexpr int L = S == 1 ? kFwdWalkSteps : kFwdSteps;
  constexpr bool STREAM = S == 1;  // a split sequence is read twice, the second time from the caches
  static_assert(C * S == kThreads, "lanes x strands");
  __shared__ float4 meet[S > 1 ? 2 : 1][S][2][S > 1 ? C : 1];
  const int lane = threadIdx.x % C, strand = threadIdx.x / C;
  const int64_t channel = static_cast<int64_t>(blockIdx.x) * C + lane;
  const Place at(p, channel);
  const int split = blockIdx.y;
  const int64_t lanes4 = p.N * p.Hq * 4;
  const int64_t t_begin = split * p.per_split;
  const int64_t t_end = t_begin + p.per_split < p.T ? t_begin + p.per_split : p.T;
  const T* gates = static_cast<const T*>(p.gates) + at.n * p.gates_n + at.c;
  const uint8_t* active = p.active ? p.active + at.n * p.active_n : nullptr;

  // The loads of all steps are in flight together: steps past the end read the last one again, lanes past
  // the end the first node's; `on` says what counts.  Walking, a thread knows a tile ahead which steps are
  // active (`ahead`) and leaves out the rows of the others without a wait: 32 x 50000 x 128 with about a quarter
  // of them inactive, trained in float32, 1097 us instead of 1253 (in bfloat16 602 and 668).  As a strand it reads them (852 x 221 x 448
  // in bfloat16, ragged: 144 us, with the questions between the loads 171).
  held<T> raw_z[L], raw_c[L];
  unsigned act[L], ahead[L];
  auto look = [&](int64_t t0) {
    if (active) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int64_t t = t0 + strand * L + i;
        ahead[i] = active[(t < t_end ? t : t_end - 1) * p.active_t];
      }
    }
  };
  auto fetch = [&](int64_t t0) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      int64_t t = t0 + strand * L + i;
      t = t < t_end ? t : t_end - 1;
      if constexpr (S == 1) act[i] = active ? ahead[i] : 1u;
      if (S > 1 || act[i]) {
        raw_z[i] = take<STREAM, TINY>(gates + t * p.gates_t, at.left);
        raw_c[i] = take<STREAM, TINY>(gates + t * p.gates_t + p.H, at.left);
      }
    }
    look(S == 1 ? t0 + L : t0);
    if constexpr (S > 1) {
#pragma unroll
      for (int i = 0; i < L; ++i) act[i] = active ? ahead[i] : 1u;
    }
  };
  float a[L][4], b[L][4];
  // z, c -> the step's map (a, (1 - a) c)
  auto to_maps = [&](int64_t t0) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const bool on = t0 + strand * L + i < t_end && act[i] != 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // chosen before the arithmetic, not after: there is no branch around it then
        float rest;
        gate_pair(on ? widen(raw_z[i][k]) : __builtin_inff(), a[i][k], rest);
        b[i][k] = rest * (on ? widen(raw_c[i][k]) : 0.0f);
      }
    }
  };

  if (t_begin < t_end) {
    if (S == 1) look(t_begin);
    fetch(t_begin);
  }

  // the state the split starts from
  float h[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  float prod[4] = {1.0f, 1.0f, 1.0f, 1.0f};  // MAPS
  if constexpr (!MAPS) {
    if (p.h0 && at.there) load4_upto(p.h0 + at.n * p.h0_n + at.c, at.left, 0.0f, h);
    if constexpr (S > 1) {
      if (split > 0) {
        // each strand joins a share of the maps before this split, then the shares are joined
        const int share = (split + S - 1) / S;
        const int k0 = strand * share, k1 = k0 + share < split ? k0 + share : split;
        float4 P = make_float4(1, 1, 1, 1), Q = make_float4(0, 0, 0, 0);
        if (at.there) {
          const float* m = p.maps + channel * 4;
#pragma unroll 8
          for (int k = k0; k < k1; ++k) {
            const float4 pk = *reinterpret_cast<const float4*>(m + (2 * k) * lanes4);
            const float4 qk = *reinterpret_cast<const float4*>(m + (2 * k + 1) * lanes4);
            Q = make_float4(pk.x * Q.x + qk.x, pk.y * Q.y + qk.y, pk.z * Q.z + qk.z, pk.w * Q.w + qk.w);
            P = make_float4(P.x * pk.x, P.y * pk.y, P.z * pk.z, P.w * pk.w);
          }
        }
        meet[1][strand][0][lane] = P;
        meet[1][strand][1][lane] = Q;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const float4 ps = meet[1][s][0][lane], qs = meet[1][s][1][lane];
          h[0] = ps.x * h[0] + qs.x; h[1] = ps.y * h[1] + qs.y;
          h[2] = ps.z * h[2] + qs.z; h[3] = ps.w * h[3] + qs.w;
        }
        // the first tile writes meet[0], the second meet[1] after a barrier of its own
      }
    }
  }

  int turn = 0;
  for (int64_t t0 = t_begin; t0 < t_end; t0 += S * L) {
    if (S > 1 && t0 != t_begin) fetch(t0);
    to_maps(t0);
    if (S == 1 && t0 + L < t_end) fetch(t0 + L);  // the next steps' loads, before this one's stores
    float start[4];
    if constexpr (S > 1) {
      float P[4] = {1.0f, 1.0f, 1.0f, 1.0f}, Q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < L; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          P[k] *= a[i][k];
          Q[k] = __builtin_fmaf(a[i][k], Q[k], b[i][k]);
        }
      meet[turn][strand][0][lane] = make_float4(P[0], P[1], P[2], P[3]);
      meet[turn][strand][1][lane] = make_float4(Q[0], Q[1], Q[2], Q[3]);
      __syncthreads();
#pragma unroll 2
      for (int s = 0; s < S; ++s) {
        if (s == strand) {
#pragma unroll
          for (int k = 0; k < 4; ++k) start[k] = h[k];
        }
        const float4 ps = meet[turn][s][0][lane], qs = meet[turn][s][1][lane];
        h[0] = ps.x * h[0] + qs.x; h[1] = ps.y * h[1] + qs.y;
        h[2] = ps.z * h[2] + qs.z; h[3] = ps.w * h[3] + qs.w;
        if constexpr (MAPS) {
          prod[0] *= ps.x; prod[1] *= ps.y; prod[2] *= ps.z; prod[3] *= ps.w;
        }
      }
      turn ^= 1;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) start[k] = h[k];
    }
    if constexpr (!MAPS) {
      T* out = static_cast<T*>(p.h) + at.n * p.h_n + at.c;
      constexpr int GROUP = kGroup<S == 1>;
      static_assert(L % GROUP == 0, "a group begins with a thread's steps or inside them");
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int64_t t = t0 + strand * L + i;
        if (i % GROUP == 0 && p.states && at.there && t > 0 && t < t_end)
          put<TINY>(p.states + ((t / GROUP - 1) * p.N + at.n) * p.H + at.c, at.left, start);
#pragma unroll
        for (int k = 0; k < 4; ++k) start[k] = __builtin_fmaf(a[i][k], start[k], b[i][k]);
        if (at.there && t < t_end) put<TINY>(out + t * p.h_t, at.left, start);
      }
      if constexpr (S == 1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = start[k];
      }
    }
  }

  if (!at.there) return;
  if constexpr (MAPS) {
    if (strand == 0) {
      float* m = p.maps + channel * 4 + static_cast<int64_t>(2 * split) * lanes4;
      *reinterpret_cast<float4*>(m) = make_float4(prod[0], prod[1], prod[2], prod[3]);
      *reinterpret_cast<float4*>(m + lanes4) = make_float4(h[0], h[1], h[2], h[3]);
    }
  } else if (split == p.splits - 1 && strand == 0) {
    store4_upto(p.last + at.n * p.H + at.c, at.left, h);
  }
}

// Backward, from the last step down: strand 0 has the latest steps of a tile, split 0 the latest
// steps of all.  A thread's L steps are a group: they begin at a multiple of L, and the states before each
// of them come from the one before the group, by the forward pass's own arithmetic.
//
// Walking, the bfloat16 form takes 168 registers, which leaves room for three waves to a SIMD: what is the same for
// all steps of a tile (the address of the state before it) is therefore made again and not kept, and which steps
// are active is kept in scalar masks.  With 176 registers and two waves, 32 x 50000 x 128 with a quarter
// of the steps inactive takes 659 us trained, not 602.
template <typename T, int C, int S, bool MAPS, bool TINY>
__global__ __launch_bounds__(kThreads, S > 1 ? 4 : 1) void scan_bwd_kernel(ScanArgs p) {
  constexpr int L = kGroup<S == 1>;
  constexpr bool STREAM = S == 1;
  static_assert(C * S == kThreads, "lanes x strands");
  __shared__ float4 meet[S > 1 ? 2 : 1][S][2][S > 1 ? C : 1];
  const int lane = threadIdx.x % C, strand = threadIdx.x / C;
  const int64_t channel = static_cast<int64_t>(blockIdx.x) * C + lane;
  const Place at(p, channel);
  const int split = blockIdx.y;
  const int64_t lanes4 = p.N * p.Hq * 4;
  // steps counted from the end of the last group: u = groups L - 1 - t
  const int64_t steps = (p.T + L - 1) / L * L;
  const int64_t u_begin = split * p.per_split;
  const int64_t u_end = u_begin + p.per_split < steps ? u_begin + p.per_split : steps;
  const T* gates = static_cast<const T*>(p.gates) + at.n * p.gates_n + at.c;
  const T* g = static_cast<const T*>(p.g) + (p.g ? at.n * p.g_n + at.c : 0);
  const uint8_t* active = p.active ? p.active + at.n * p.active_n : nullptr;

  held<T> raw_z[L], raw_c[L], raw_g[L];
  held<float> raw_s;
  unsigned ahead[L];
  bool act[L];
  // The step at u, kept among those of the split: steps that are not there read a neighbour again.
  auto step_at = [&](int64_t u) {
    const int64_t t = steps - 1 - (u < u_end ? u : u_end - 1);
    return t < p.T ? t : p.T - 1;
  };
  auto look = [&](int64_t u0) {
    if (active) {
#pragma unroll
      for (int i = 0; i < L; ++i) ahead[i] = active[step_at(u0 + strand * L + i) * p.active_t];
    }
  };
  auto fetch = [&](int64_t u0) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int64_t t = step_at(u0 + strand * L + i);
      if constexpr (S == 1) act[i] = !active || ahead[i] != 0;
      if (S > 1 || act[i]) {
        raw_z[i] = take<STREAM, TINY>(gates + t * p.gates_t, at.left);
        if constexpr (!MAPS) raw_c[i] = take<STREAM, TINY>(gates + t * p.gates_t + p.H, at.left);
      }
    }
    if (p.g) {
#pragma unroll
      for (int i = 0; i < L; ++i) raw_g[i] = take<STREAM, TINY>(g + step_at(u0 + strand * L + i) * p.g_t, at.left);
    }
    if constexpr (!MAPS) {
      // (a strand past the end of its split reads what is before an earlier group, or h0, and does not use it)
      const int64_t group = (steps - 1 - (u0 + strand * L)) / L;
      const float* const src = group > 0 ? p.before + (group - 1) * p.before_g : p.h0;
      raw_s = held<float>{0.0f, 0.0f, 0.0f, 0.0f};
      if (src) raw_s = take<STREAM, TINY>(src + at.n * (group > 0 ? p.before_n : p.h0_n) + at.c, at.left);
    }
    look(S == 1 ? u0 + L : u0);
    if constexpr (S > 1) {
#pragma unroll
      for (int i = 0; i < L; ++i) act[i] = !active || ahead[i] != 0;
    }
  };

  if (u_begin < u_end) {
    if (S == 1) look(u_begin);
    fetch(u_begin);
  }

  float e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  float prod[4] = {1.0f, 1.0f, 1.0f, 1.0f};  // MAPS
  if constexpr (!MAPS) {
    if (p.g_last && at.there) load4_upto(p.g_last + at.n * p.gl_n + at.c, at.left, 0.0f, e);
    if constexpr (S > 1) {
      if (split > 0) {
        const int share = (split + S - 1) / S;
        const int k0 = strand * share, k1 = k0 + share < split ? k0 + share : split;
        float4 P = make_float4(1, 1, 1, 1), Q = make_float4(0, 0, 0, 0);
        if (at.there) {
          const float* m = p.maps + channel * 4;
#pragma unroll 8
          for (int k = k0; k < k1; ++k) {
            const float4 pk = *reinterpret_cast<const float4*>(m + (2 * k) * lanes4);
            const float4 qk = *reinterpret_cast<const float4*>(m + (2 * k + 1) * lanes4);
            Q = make_float4(pk.x * Q.x + qk.x, pk.y * Q.y + qk.y, pk.z * Q.z + qk.z, pk.w * Q.w + qk.w);
            P = make_float4(P.x * pk.x, P.y * pk.y, P.z * pk.z, P.w * pk.w);
          }
        }
        meet[1][strand][0][lane] = P;
        meet[1][strand][1][lane] = Q;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const float4 ps = meet[1][s][0][lane], qs = meet[1][s][1][lane];
          e[0] = ps.x * e[0] + qs.x; e[1] = ps.y * e[1] + qs.y;
          e[2] = ps.z * e[2] + qs.z; e[3] = ps.w * e[3] + qs.w;
        }
      }
    }
  }

  int turn = 0;
  for (int64_t u0 = u_begin; u0 < u_end; u0 += S * L) {
    if (S > 1 && u0 != u_begin) fetch(u0);
    float a[L][4], rest[L][4], gv[L][4], away[L][4];  // away: the state before the step, less c
    bool there[L], on[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int64_t u = u0 + strand * L + i;
      there[i] = u < u_end && steps - 1 - u < p.T;
      on[i] = there[i] && act[i];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        gate_pair(on[i] ? widen(raw_z[i][k]) : __builtin_inff(), a[i][k], rest[i][k]);  // 1, 0 for a step passed over
        // a step that is not there passes e on as it is
        gv[i][k] = p.g && there[i] ? widen(raw_g[i][k]) : 0.0f;
      }
    }
    if constexpr (!MAPS) {
      float state[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) state[k] = raw_s[k];
#pragma unroll
      for (int i = L - 1; i >= 0; --i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float c = on[i] ? widen(raw_c[i][k]) : 0.0f;
          away[i][k] = state[k] - c;
          state[k] = __builtin_fmaf(a[i][k], state[k], rest[i][k] * c);
        }
    }
    if (S == 1 && u0 + L < u_end) fetch(u0 + L);
    float start[4];
    if constexpr (S > 1) {
      float P[4] = {1.0f, 1.0f, 1.0f, 1.0f}, Q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < L; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          P[k] *= a[i][k];
          Q[k] = a[i][k] * (Q[k] + gv[i][k]);
        }
      meet[turn][strand][0][lane] = make_float4(P[0], P[1], P[2], P[3]);
      meet[turn][strand][1][lane] = make_float4(Q[0], Q[1], Q[2], Q[3]);
      __syncthreads();
#pragma unroll 2
      for (int s = 0; s < S; ++s) {
        if (s == strand) {
#pragma unroll
          for (int k = 0; k < 4; ++k) start[k] = e[k];
        }
        const float4 ps = meet[turn][s][0][lane], qs = meet[turn][s][1][lane];
        e[0] = ps.x * e[0] + qs.x; e[1] = ps.y * e[1] + qs.y;
        e[2] = ps.z * e[2] + qs.z; e[3] = ps.w * e[3] + qs.w;
        if constexpr (MAPS) {
          prod[0] *= ps.x; prod[1] *= ps.y; prod[2] *= ps.z; prod[3] *= ps.w;
        }
      }
      turn ^= 1;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) start[k] = e[k];
    }
    if constexpr (!MAPS) {
      T* out = static_cast<T*>(p.dgates) + at.n * p.dg_n + at.c;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int64_t u = u0 + strand * L + i, t = steps - 1 - u;
        float dz[4], dc[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float d = start[k] + gv[i][k];
          dc[k] = on[i] ? d * rest[i][k] : 0.0f;
          dz[k] = on[i] ? d * away[i][k] * (a[i][k] * rest[i][k]) : 0.0f;
          start[k] = a[i][k] * d;
        }
        if (p.dgates && at.there && there[i]) {
          put<TINY>(out + t * p.dg_t, at.left, dz);
          put<TINY>(out + t * p.dg_t + p.H, at.left, dc);
        }
      }
      if constexpr (S == 1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = start[k];
      }
    }
  }

  if (!at.there) return;
  if constexpr (MAPS) {
    if (strand == 0) {
      float* m = p.maps + channel * 4 + static_cast<int64_t>(2 * split) * lanes4;
      *reinterpret_cast<float4*>(m) = make_float4(prod[0], prod[1], prod[2], prod[3]);
      *reinterpret_cast<float4*>(m + lanes4) = make_float4(e[0], e[1], e[2], e[3]);
    }
  } else if (p.dh0 && split == p.splits - 1 && strand == 0) {
    store4_upto(p.dh0 + at.n * p.H + at.c, at.left, e);
  }
}

// How a problem is laid out; the same for both directions but for the steps of a tile.
struct Plan {
  bool walk;     // a thread walks the steps
  int splits;
  int64_t per_split;
};
Plan plan_for(int64_t T, int64_t N, int64_t H, int steps) {
  const int64_t lanes = N * ((H + 3) / 4);
  if (lanes >= kManyLanes || T <= kFewSteps) return {true, 1, T};
  const int64_t tile = static_cast<int64_t>(kStrands) * steps;
  const int64_t tiles = (T + tile - 1) / tile;
  const int64_t groups = (lanes + kLanes - 1) / kLanes;
  int64_t splits = groups >= kEnoughGroups ? 1 : kTargetGroups / groups;
  splits = splits > kMaxSplits ? kMaxSplits : splits;
  splits = splits < tiles ? splits : tiles;
  const int64_t per = (tiles + splits - 1) / splits * tile;
  return {false, static_cast<int>((T + per - 1) / per), per};
}
int64_t group_of(const Plan& q) { return q.walk ? kGroup<true> : kGroup<false>; }
size_t maps_bytes(int64_t T, int64_t N, int64_t H, int steps) {
  const Plan q = plan_for(T, N, H, steps);
  return q.splits > 1 ? static_cast<size_t>(q.splits) * 2 * N * ((H + 3) / 4) * 4 * sizeof(float) : 0;
}

template <typename T, bool TINY>
void launch_fwd(const ScanArgs& a, const Plan& q, hipStream_t st) {
  const int64_t lanes = a.N * a.Hq;
  if (q.walk) {
    scan_fwd_kernel<T, kThreads, 1, false, TINY><<<(lanes + kThreads - 1) / kThreads, kThreads, 0, st>>>(a);
    return;
  }
  const unsigned groups = static_cast<unsigned>((lanes + kLanes - 1) / kLanes);
  if (q.splits > 1)  // the last split's map starts nothing
    scan_fwd_kernel<T, kLanes, kStrands, true, TINY><<<dim3(groups, q.splits - 1), kThreads, 0, st>>>(a);
  scan_fwd_kernel<T, kLanes, kStrands, false, TINY><<<dim3(groups, q.splits), kThreads, 0, st>>>(a);
}
template <typename T, bool TINY>
void launch_bwd(const ScanArgs& a, const Plan& q, hipStream_t st) {
  const int64_t lanes = a.N * a.Hq;
  if (q.walk) {
    scan_bwd_kernel<T, kThreads, 1, false, TINY><<<(lanes + kThreads - 1) / kThreads, kThreads, 0, st>>>(a);
    return;
  }
  const unsigned groups = static_cast<unsigned>((lanes + kLanes - 1) / kLanes);
  if (q.splits > 1)
    scan_bwd_kernel<T, kLanes, kStrands, true, TINY><<<dim3(groups, q.splits - 1), kThreads, 0, st>>>(a);
  scan_bwd_kernel<T, kLanes, kStrands, false, TINY><<<dim3(groups, q.splits), kThreads, 0, st>>>(a);
}

int check_sizes(const char* what, int dtype, int64_t T, int64_t N, int64_t H) {
  SPMI_REQUIRE(dtype == SPMI_DTYPE_F32 || dtype == SPMI_DTYPE_BF16, SPMI_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  SPMI_REQUIRE(T >= 0 && N >= 0 && H >= 1, SPMI_ERR_INVALID_ARG, "%s: T=%lld N=%lld H=%lld", what, (long long)T,
               (long long)N, (long long)H);
  // a thread for each four units (a row has one at least), and a grid holds less than 2^32 threads
  SPMI_REQUIRE(H <= (1 << 24) && N <= ((1ll << 32) - kThreads) / ((H + 3) / 4), SPMI_ERR_UNSUPPORTED,
               "%s: N=%lld H=%lld is too large", what, (long long)N, (long long)H);
  return SPMI_OK;
}

// ---- the single step on the node memory ------------------------------------------------------

struct StepArgs {
  const void* gates;
  int64_t ldg;
  float* mem;          // [nodes, H]
  const int64_t* ids;  // nullable: row i of the gates belongs to node i
  int64_t M, nodes;
  int H, Hq;
  float* out;          // [M, H]
  float* before;       // nullable, [M, H]: the rows' old states
  bool write;          // ids == nullptr only: the new states go to the memory as well
  int32_t* owner;      // nullable, [nodes]: the entries of the named nodes are cleared
};

template <typename T>
__global__ __launch_bounds__(kThreads) void step_kernel(StepArgs p) {
  const int64_t total = p.M * p.Hq;
  for (int64_t j = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; j < total;
       j += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = j / p.Hq;
    const int c = static_cast<int>(j - row * p.Hq) * 4, left = p.H - c;
    const int64_t node = p.ids ? p.ids[row] : row;
    float z[4], cand[4], h[4];
    const T* gates = static_cast<const T*>(p.gates) + row * p.ldg + c;
    load4_upto(gates, left, 0.0f, z);
    load4_upto(gates + p.H, left, 0.0f, cand);
    const bool known = node >= 0 && node < p.nodes;
    if (known) {
      load4_upto(p.mem + node * p.H + c, left, 0.0f, h);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) h[k] = __builtin_nanf("");
    }
    if (p.before) store4_upto(p.before + row * p.H + c, left, h);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float a, rest;
      gate_pair(z[k], a, rest);
      h[k] = __builtin_fmaf(a, h[k], rest * cand[k]);
    }
    store4_upto(p.out + row * p.H + c, left, h);
    if (p.write && known) store4_upto(p.mem + node * p.H + c, left, h);
    if (p.owner && known && c == 0) p.owner[node] = -1;
  }
}

// The last of the rows that name a node.
__global__ void step_owner_kernel(const int64_t* ids, int64_t M, int64_t nodes, int32_t* owner) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i < M && ids[i] >= 0 && ids[i] < nodes) atomicMax(&owner[ids[i]], static_cast<int32_t>(i));
}

// New states to the memory: a row is copied if no later row names its node.  `owner` holds the
// last row of each named node, or is null and the wave looks through the later ids itself.
__global__ __launch_bounds__(kThreads) void step_write_kernel(StepArgs p) {
  const int lane = threadIdx.x & 63;
  for (int64_t row = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 6; row < p.M;
       row += (static_cast<int64_t>(gridDim.x) * kThreads) >> 6) {
    const int64_t node = p.ids[row];
    if (node < 0 || node >= p.nodes) continue;
    bool last = true;
    if (p.owner) {
      last = p.owner[node] == row;
    } else {
      for (int64_t i = row + 1 + lane; i < p.M; i += 64) last = last && p.ids[i] != node;
      last = __all(last);
    }
    if (!last) continue;
    for (int c = lane * 4; c < p.H; c += 256) {
      float h[4];
      load4_upto(p.out + row * p.H + c, p.H - c, 0.0f, h);
      store4_upto(p.mem + node * p.H + c, p.H - c, h);
    }
  }
}

// Up to this many rows the ids behind a row are looked through (one launch less, no workspace).
constexpr int64_t kLookRows = 1024;

}  // namespace

extern "C" {

size_t spmi_gated_scan_fwd_workspace_bytes(int64_t T, int64_t N, int64_t H) {
  return T > 0 && N > 0 && H > 0 ? maps_bytes(T, N, H, kFwdSteps) : 0;
}
size_t spmi_gated_scan_bwd_workspace_bytes(int64_t T, int64_t N, int64_t H) {
  return T > 0 && N > 0 && H > 0 ? maps_bytes(T, N, H, kBwdSteps) : 0;
}

int64_t spmi_gated_scan_states(int64_t T, int64_t N, int64_t H) {
  return T > 0 && N > 0 && H > 0 ? (T - 1) / group_of(plan_for(T, N, H, kBwdSteps)) : 0;
}

int spmi_gated_scan_fwd_saved(const void* gates, int dtype, int64_t gates_t, int64_t gates_n, const float* h0,
                              int64_t h0_n, const uint8_t* active, int64_t active_t, int64_t active_n, int64_t T,
                              int64_t N, int64_t H, void* h, int64_t h_t, int64_t h_n, float* last, float* states,
                              void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_sizes("spmi_gated_scan_fwd", dtype, T, N, H)) return rc;
  if (N == 0) return SPMI_OK;
  SPMI_REQUIRE(last && (T == 0 || (gates && h)), SPMI_ERR_INVALID_ARG, "spmi_gated_scan_fwd: null pointer");
  const Plan q = plan_for(T, N, H, kFwdSteps);
  SPMI_REQUIRE(q.splits == 1 || (ws && ws_bytes >= maps_bytes(T, N, H, kFwdSteps)), SPMI_ERR_WORKSPACE,
               "spmi_gated_scan_fwd: workspace of %zu bytes is too small", ws_bytes);
  SPMI_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 15) == 0, SPMI_ERR_INVALID_ARG,
               "spmi_gated_scan_fwd: the workspace must be aligned to 16 bytes");
  ScanArgs a{};
  a.gates = gates; a.gates_t = gates_t; a.gates_n = gates_n;
  a.h0 = h0; a.h0_n = h0_n;
  a.active = active; a.active_t = active_t; a.active_n = active_n;
  a.h = h; a.h_t = h_t; a.h_n = h_n; a.last = last; a.states = states;
  a.T = T; a.N = N; a.H = static_cast<int>(H); a.Hq = static_cast<int>((H + 3) / 4);
  a.per_split = q.per_split; a.splits = q.splits; a.maps = static_cast<float*>(ws);
  const bool tiny = H < 4;
  if (dtype == SPMI_DTYPE_F32) (tiny ? launch_fwd<float, true> : launch_fwd<float, false>)(a, q, as_stream(stream));
  else (tiny ? launch_fwd<bf16, true> : launch_fwd<bf16, false>)(a, q, as_stream(stream));
  SPMI_CHECK_LAUNCH("spmi_gated_scan_fwd");
  return SPMI_OK;
}

int spmi_gated_scan_fwd(const void* gates, int dtype, int64_t gates_t, int64_t gates_n, const float* h0, int64_t h0_n,
                        const uint8_t* active, int64_t active_t, int64_t active_n, int64_t T, int64_t N, int64_t H,
                        void* h, int64_t h_t, int64_t h_n, float* last, void* ws, size_t ws_bytes, void* stream) {
  return spmi_gated_scan_fwd_saved(gates, dtype, gates_t, gates_n, h0, h0_n, active, active_t, active_n, T, N, H, h,
                                   h_t, h_n, last, nullptr, ws, ws_bytes, stream);
}

int spmi_gated_scan_bwd(const void* gates, int dtype, int64_t gates_t, int64_t gates_n, const float* h0, int64_t h0_n,
                        const uint8_t* active, int64_t active_t, int64_t active_n, int64_t T, int64_t N, int64_t H,
                        const void* h, int64_t h_t, int64_t h_n, const float* states, const void* g, int64_t g_t,
                        int64_t g_n, const float* g_last, int64_t gl_n, void* dgates, int64_t dg_t, int64_t dg_n, float* dh0,
                        void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_sizes("spmi_gated_scan_bwd", dtype, T, N, H)) return rc;
  if (N == 0 || (T == 0 && !dh0)) return SPMI_OK;
  const bool f32 = dtype == SPMI_DTYPE_F32;
  const Plan q = plan_for(T, N, H, kBwdSteps);
  const int64_t group = group_of(q);
  SPMI_REQUIRE((T == 0 || gates) && (T <= group || (f32 ? h != nullptr : states != nullptr)), SPMI_ERR_INVALID_ARG,
               "spmi_gated_scan_bwd: null pointer");
  SPMI_REQUIRE(q.splits == 1 || (ws && ws_bytes >= maps_bytes(T, N, H, kBwdSteps)), SPMI_ERR_WORKSPACE,
               "spmi_gated_scan_bwd: workspace of %zu bytes is too small", ws_bytes);
  SPMI_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 15) == 0, SPMI_ERR_INVALID_ARG,
               "spmi_gated_scan_bwd: the workspace must be aligned to 16 bytes");
  ScanArgs a{};
  a.gates = gates; a.gates_t = gates_t; a.gates_n = gates_n;
  a.h0 = h0; a.h0_n = h0_n;
  a.active = active; a.active_t = active_t; a.active_n = active_n;
  if (T > group && f32) {  // float32 states are whole where they stand in h
    a.before = static_cast<const float*>(h) + (group - 1) * h_t; a.before_g = group * h_t; a.before_n = h_n;
  } else if (T > group) {
    a.before = states; a.before_g = N * H; a.before_n = H;
  }
  a.g = g; a.g_t = g_t; a.g_n = g_n; a.g_last = g_last; a.gl_n = gl_n;
  a.dgates = dgates; a.dg_t = dg_t; a.dg_n = dg_n; a.dh0 = dh0;
  a.T = T; a.N = N; a.H = static_cast<int>(H); a.Hq = static_cast<int>((H + 3) / 4);
  a.per_split = q.walk ? T + group : q.per_split;  // walking: all steps of the last group too
  a.splits = q.splits; a.maps = static_cast<float*>(ws);
  const bool tiny = H < 4;
  if (f32) (tiny ? launch_bwd<float, true> : launch_bwd<float, false>)(a, q, as_stream(stream));
  else (tiny ? launch_bwd<bf16, true> : launch_bwd<bf16, false>)(a, q, as_stream(stream));
  SPMI_CHECK_LAUNCH("spmi_gated_scan_bwd");
  return SPMI_OK;
}

size_t spmi_gated_step_workspace_bytes(int64_t M, int64_t nodes) {
  return M > kLookRows && nodes > 0 ? static_cast<size_t>(nodes) * sizeof(int32_t) : 0;
}

int spmi_gated_step(const void* gates, int dtype, int64_t ldg, float* h_mem, int64_t nodes, const int64_t* ids,
                    int64_t M, int64_t H, float* h_out, float* h_before, int mem_write, void* ws, size_t ws_bytes,
                    void* stream) {
  if (int rc = check_sizes("spmi_gated_step", dtype, 1, M, H)) return rc;
  SPMI_REQUIRE(nodes >= 0 && M < (1ll << 31), SPMI_ERR_INVALID_ARG, "spmi_gated_step: %lld nodes, %lld rows",
               (long long)nodes, (long long)M);
  SPMI_REQUIRE(ids || M <= nodes, SPMI_ERR_INVALID_ARG, "spmi_gated_step: more rows than nodes");
  if (M == 0) return SPMI_OK;
  SPMI_REQUIRE(gates && h_out && (h_mem || nodes == 0), SPMI_ERR_INVALID_ARG, "spmi_gated_step: null pointer");
  const bool scatter = ids && mem_write;
  const bool owners = scatter && M > kLookRows;
  SPMI_REQUIRE(!owners || (ws && ws_bytes >= spmi_gated_step_workspace_bytes(M, nodes)) || nodes == 0,
               SPMI_ERR_WORKSPACE, "spmi_gated_step: workspace of %zu bytes is too small", ws_bytes);
  hipStream_t st = as_stream(stream);
  StepArgs a{gates, ldg, h_mem, ids, M, nodes, static_cast<int>(H), static_cast<int>((H + 3) / 4), h_out, h_before,
             mem_write != 0 && !ids, owners ? static_cast<int32_t*>(ws) : nullptr};
  const int64_t need = (M * a.Hq + kThreads - 1) / kThreads;
  const unsigned grid = static_cast<unsigned>(need < 8192 ? need : 8192);
  if (dtype == SPMI_DTYPE_F32) step_kernel<float><<<grid, kThreads, 0, st>>>(a);
  else step_kernel<bf16><<<grid, kThreads, 0, st>>>(a);
  SPMI_CHECK_LAUNCH("spmi_gated_step");
  if (scatter && nodes > 0) {
    if (owners) {
      step_owner_kernel<<<static_cast<unsigned>((M + 255) / 256), 256, 0, st>>>(ids, M, nodes, a.owner);
      SPMI_CHECK_LAUNCH("spmi_gated_step");
    }
    const int64_t blocks = (M + 3) / 4;
    step_write_kernel<<<static_cast<unsigned>(blocks < 8192 ? blocks : 8192), kThreads, 0, st>>>(a);
    SPMI_CHECK_LAUNCH("spmi_gated_step");
  }
  return SPMI_OK;
}

}  // extern "C"
