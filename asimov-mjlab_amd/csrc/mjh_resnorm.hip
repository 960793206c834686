// mjh_resnorm.hip — a residual block's epilogue fused with the next block's norm, and dropout (gfx950).
//
//   p = norm_post(y)            (x - mean) rstd w + b; rms: mean = 0; without post weights p = y
//   u = keep ? p / (1 - prob) : 0      counter-based bits (mjh_seq.h), nothing stored
//   s = residual + scale * act(gate) * u
//   n = norm_pre(s)
// The statistics, s inside n, and all sums are float32; s and n are rounded once, at their store.
//
// A group of `TPR` lanes holds a row, 8 elements a lane, so every tensor is read once and every statistic is
// taken from registers (the variance around the mean, in a second pass over registers). Groups up to a wave
// reduce with lane exchanges, wider ones through shared memory. The backward pass keeps s and p nowhere: it
// forms them again from y, residual and gate, the tensors that it has to read in any case, with the forward
// pass's (mean, rstd) of each row. Weight gradients: a group adds its rows in registers, groups of a workgroup
// join in shared memory, workgroups in a second launch, each in a fixed order.
#include <algorithm>
#include <cstring>

#include "mjh_seq.h"

namespace {
using namespace mjh_seq;

constexpr int kPer = 8;     // elements a lane holds
constexpr int kMaxTpr = 1024;
constexpr int kSums = 5;    // post weight, post bias, scale, pre weight, pre bias
enum { kPostW, kPostB, kScale, kPreW, kPreB };

struct Args {
  const void* y; ll ys;
  const void* r; ll rs;
  const void* gate; ll gs;
  const void* post_w; const void* post_b; const void* pre_w; const void* pre_b; const void* scale;
  int w32;        // weights are float32 (else of the rows' type)
  int scale_one;  // one scale for all channels
  void* s; ll ss;
  void* n; ll ns;
  float* stats;   // (R, 4): post mean, post rstd, pre mean, pre rstd
  const void* ds; ll dss;
  const void* dn; ll dns;
  void* dy; ll dys;
  void* dr; ll drs;
  void* dgate; ll dgs;
  float* sums;    // (workgroups, kSums, D)
  mjh_i64* ctr_out;
  Drop drop;
  float eps;
  int R, D, layer, act, post, pre;
};

template <class T, bool VEC>
struct Lanes {
  static constexpr int kVec = VEC ? 16 / (int)sizeof(T) : 1;
  static constexpr int kPieces = kPer / kVec;
};
// column of a lane's element k: pieces of kVec neighbours, a group's pieces side by side
template <class T, bool VEC, int TPR>
__device__ __forceinline__ int col(int lane, int k) {
  constexpr int V = Lanes<T, VEC>::kVec;
  return (k / V * TPR + lane) * V + k % V;
}
template <class T, bool VEC, int TPR>
__device__ __forceinline__ void read(const T* p, int lane, int D, bool on, T (&o)[kPer]) {
  constexpr int V = Lanes<T, VEC>::kVec;
#pragma unroll
  for (int k = 0; k < kPer; k += V) {
    const int c = col<T, VEC, TPR>(lane, k);
    Pack<T, V> v{};
    if (on && c < D) v = load<T, V>(p + c);
#pragma unroll
    for (int j = 0; j < V; j++) o[k + j] = v.v[j];
  }
}
template <class T, bool VEC, int TPR>
__device__ __forceinline__ void write(T* p, int lane, int D, bool on, const float (&f)[kPer]) {
  constexpr int V = Lanes<T, VEC>::kVec;
#pragma unroll
  for (int k = 0; k < kPer; k += V) {
    const int c = col<T, VEC, TPR>(lane, k);
    float o[V];
#pragma unroll
    for (int j = 0; j < V; j++) o[j] = f[k + j];
    if (on && c < D) store<T, V>(p + c, o);
  }
}
// channel weights; 1 or 0 where there are none
template <class T, bool VEC, int TPR>
__device__ __forceinline__ void weights(const void* w, int w32, int lane, int D, float none, float (&o)[kPer]) {
#pragma unroll
  for (int k = 0; k < kPer; k++) {
    const int c = col<T, VEC, TPR>(lane, k);
    o[k] = none;
    if (w && c < D) o[k] = w32 ? static_cast<const float*>(w)[c] : (float)static_cast<const T*>(w)[c];
  }
}

// Sums of NV values over a row's lanes, in every lane. Wider groups than a wave: shared memory, two barriers.
template <int TPR, int NV>
__device__ __forceinline__ void row_sum(float (&v)[NV], float* shared) {
#pragma unroll
  for (int m = (TPR < 64 ? TPR : 64) / 2; m > 0; m >>= 1)
#pragma unroll
    for (int k = 0; k < NV; k++) v[k] += __shfl_xor(v[k], m);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < NV; k++) shared[wave * NV + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; k++) {
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < W; j++) t += shared[(first + j) * NV + k];
      v[k] = t;
    }
    __syncthreads();
  }
}

constexpr int block_of(int tpr) { return tpr < 256 ? 256 : tpr; }

__device__ __forceinline__ unsigned long long drop_base(const Drop& d) { return mjh::Rng(d.seed, d.key, d.ctr).base; }

// keep bits of a lane's elements (bit k: element k); the row's first element has index row * D
template <class T, bool VEC, int TPR>
__device__ __forceinline__ unsigned keep_bits(unsigned long long base, const Drop& d, ll first, int lane) {
  constexpr int V = Lanes<T, VEC>::kVec;
  unsigned bits = 0;
#pragma unroll
  for (int k = 0; k < kPer; k += V) {
    const unsigned long long i = (unsigned long long)(first + col<T, VEC, TPR>(lane, k));
    if (V > 1 && !(i & 1)) {
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const unsigned long long w = drop_word(base, (i + j) >> 1);
        bits |= (unsigned)drop_keep(w, 0, d.thr) << (k + j);
        bits |= (unsigned)drop_keep(w, 1, d.thr) << (k + j + 1);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; j++)
        bits |= (unsigned)drop_keep(drop_word(base, (i + j) >> 1), (int)((i + j) & 1), d.thr) << (k + j);
    }
  }
  return bits;
}

// mean and 1 / deviation of a row held in registers (columns beyond D hold 0 in v)
template <class T, bool VEC, int TPR>
__device__ __forceinline__ void row_stats(const float (&v)[kPer], const Args& a, int lane, float* shared, float& mean,
                                          float& rstd) {
  mean = 0.f;
  float t[1];
  if (a.layer) {
    t[0] = 0.f;
#pragma unroll
    for (int k = 0; k < kPer; k++) t[0] += v[k];
    row_sum<TPR, 1>(t, shared);
    mean = t[0] / (float)a.D;
  }
  t[0] = 0.f;
#pragma unroll
  for (int k = 0; k < kPer; k++) {
    const float c = col<T, VEC, TPR>(lane, k) < a.D ? v[k] - mean : 0.f;
    t[0] += c * c;
  }
  row_sum<TPR, 1>(t, shared);
  rstd = 1.f / sqrtf(t[0] / (float)a.D + a.eps);
}

struct Act {
  float value, slope;
  __device__ __forceinline__ Act(float g, int act) {
    const float q = sigmoid_small(g);
    const float pos = g < 0.f ? q : 1.f - q, neg = g < 0.f ? 1.f - q : q;
    if (act == MJH_ACT_SIGMOID) {
      value = pos;
      slope = pos * neg;
    } else {
      // g sigmoid(g); at an infinite gate its limits: g, and 0 for -inf
      value = pos == 0.f ? 0.f : g * pos;
      const float t = neg == 0.f || pos == 0.f ? 0.f : g * neg;
      slope = pos * (1.f + t);
    }
    if (g != g) value = slope = g;
  }
};

template <class T, bool VEC, int TPR>
__global__ __launch_bounds__(block_of(TPR)) void resnorm_forward(const Args a) {
  constexpr int kGroups = block_of(TPR) / TPR;
  __shared__ float shared[block_of(TPR) / 64];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  if (a.ctr_out && blockIdx.x == 0 && threadIdx.x == 0) *a.ctr_out = a.drop.ctr ? *a.drop.ctr : 0;
  const bool block = a.y != nullptr;
  const unsigned long long base = a.drop.thr ? drop_base(a.drop) : 0;
  float post_w[kPer], post_b[kPer], pre_w[kPer], pre_b[kPer], scale[kPer];
  weights<T, VEC, TPR>(a.post_w, a.w32, lane, a.D, 1.f, post_w);
  weights<T, VEC, TPR>(a.post_b, a.w32, lane, a.D, 0.f, post_b);
  weights<T, VEC, TPR>(a.pre_w, a.w32, lane, a.D, 1.f, pre_w);
  weights<T, VEC, TPR>(a.pre_b, a.w32, lane, a.D, 0.f, pre_b);
  weights<T, VEC, TPR>(a.scale_one ? nullptr : a.scale, a.w32, lane, a.D, 1.f, scale);
  if (a.scale_one) {
    const float one = a.w32 ? *static_cast<const float*>(a.scale) : (float)*static_cast<const T*>(a.scale);
#pragma unroll
    for (int k = 0; k < kPer; k++) scale[k] = one;
  }
  for (ll first = (ll)blockIdx.x * kGroups; first < a.R; first += (ll)gridDim.x * kGroups) {
    const ll row = first + group;
    const bool on = row < a.R;
    T rr[kPer];
    read<T, VEC, TPR>(static_cast<const T*>(a.r) + row * a.rs, lane, a.D, on, rr);
    float s[kPer], stats[4] = {0.f, 1.f, 0.f, 1.f};
    if (block) {
      T ry[kPer], rg[kPer];
      read<T, VEC, TPR>(static_cast<const T*>(a.y) + row * a.ys, lane, a.D, on, ry);
      if (a.gate) read<T, VEC, TPR>(static_cast<const T*>(a.gate) + row * a.gs, lane, a.D, on, rg);
      float y[kPer];
#pragma unroll
      for (int k = 0; k < kPer; k++) y[k] = (float)ry[k];
      if (a.post) row_stats<T, VEC, TPR>(y, a, lane, shared, stats[0], stats[1]);
      const unsigned keep = a.drop.thr ? keep_bits<T, VEC, TPR>(base, a.drop, row * a.D, lane) : ~0u;
#pragma unroll
      for (int k = 0; k < kPer; k++) {
        float p = a.post ? (y[k] - stats[0]) * stats[1] * post_w[k] + post_b[k] : y[k];
        p = (keep >> k & 1u) ? p * a.drop.scale : 0.f;
        if (a.gate) p *= Act((float)rg[k], a.act).value;
        s[k] = (float)rr[k] + scale[k] * p;
      }
      write<T, VEC, TPR>(static_cast<T*>(a.s) + row * a.ss, lane, a.D, on, s);
    } else {
#pragma unroll
      for (int k = 0; k < kPer; k++) s[k] = (float)rr[k];
    }
    if (a.pre) {
#pragma unroll
      for (int k = 0; k < kPer; k++)
        if (col<T, VEC, TPR>(lane, k) >= a.D) s[k] = 0.f;
      row_stats<T, VEC, TPR>(s, a, lane, shared, stats[2], stats[3]);
      float n[kPer];
#pragma unroll
      for (int k = 0; k < kPer; k++) n[k] = (s[k] - stats[2]) * stats[3] * pre_w[k] + pre_b[k];
      write<T, VEC, TPR>(static_cast<T*>(a.n) + row * a.ns, lane, a.D, on, n);
    }
    if (a.stats && on && lane == 0) store<float, 4>(a.stats + row * 4, stats);
  }
}

// BLOCK: there is a y (else only the norm before). BIAS: bias gradients are wanted.
template <class T, bool VEC, int TPR, bool BLOCK, bool BIAS>
__global__ __launch_bounds__(block_of(TPR)) void resnorm_backward(const Args a) {
  constexpr int kGroups = block_of(TPR) / TPR;
  __shared__ float shared[block_of(TPR) / 64 * 2];
  __shared__ float join[kGroups > 1 ? block_of(TPR) * kPer : 1];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const unsigned long long base = BLOCK && a.drop.thr ? drop_base(a.drop) : 0;
  float post_w[kPer], post_b[kPer], pre_w[kPer], scale[kPer];
  weights<T, VEC, TPR>(a.pre_w, a.w32, lane, a.D, 1.f, pre_w);
  if (BLOCK) {
    weights<T, VEC, TPR>(a.post_w, a.w32, lane, a.D, 1.f, post_w);
    weights<T, VEC, TPR>(BIAS ? a.post_b : nullptr, a.w32, lane, a.D, 0.f, post_b);
    weights<T, VEC, TPR>(a.scale_one ? nullptr : a.scale, a.w32, lane, a.D, 1.f, scale);
    if (a.scale_one) {
      const float one = a.w32 ? *static_cast<const float*>(a.scale) : (float)*static_cast<const T*>(a.scale);
#pragma unroll
      for (int k = 0; k < kPer; k++) scale[k] = one;
    }
  }
  float sum[kSums][kPer];
#pragma unroll
  for (int q = 0; q < kSums; q++)
#pragma unroll
    for (int k = 0; k < kPer; k++) sum[q][k] = 0.f;
  const float inv = 1.f / (float)a.D;
  for (ll first = (ll)blockIdx.x * kGroups; first < a.R; first += (ll)gridDim.x * kGroups) {
    const ll row = first + group;
    const bool on = row < a.R;
    T rr[kPer], ry[kPer], rg[kPer], rds[kPer], rdn[kPer];
    if (a.pre) read<T, VEC, TPR>(static_cast<const T*>(a.r) + row * a.rs, lane, a.D, on, rr);
    if (BLOCK) {
      read<T, VEC, TPR>(static_cast<const T*>(a.y) + row * a.ys, lane, a.D, on, ry);
      if (a.gate) read<T, VEC, TPR>(static_cast<const T*>(a.gate) + row * a.gs, lane, a.D, on, rg);
    }
    if (a.ds) read<T, VEC, TPR>(static_cast<const T*>(a.ds) + row * a.dss, lane, a.D, on, rds);
    if (a.dn) read<T, VEC, TPR>(static_cast<const T*>(a.dn) + row * a.dns, lane, a.D, on, rdn);
    Pack<float, 4> st{};
    if (on) st = load<float, 4>(a.stats + row * 4);
    const unsigned keep = BLOCK && a.drop.thr ? keep_bits<T, VEC, TPR>(base, a.drop, row * a.D, lane) : ~0u;
    float ds[kPer], yhat[kPer], u[kPer], av[kPer], slope[kPer];
#pragma unroll
    for (int k = 0; k < kPer; k++) {
      ds[k] = a.ds ? (float)rds[k] : 0.f;
      if (BLOCK) {
        yhat[k] = a.post ? ((float)ry[k] - st.v[0]) * st.v[1] : (float)ry[k];
        const float p = a.post ? yhat[k] * post_w[k] + post_b[k] : yhat[k];
        u[k] = (keep >> k & 1u) ? p * a.drop.scale : 0.f;
        av[k] = 1.f;
        slope[k] = 0.f;
        if (a.gate) {
          const Act t((float)rg[k], a.act);
          av[k] = t.value;
          slope[k] = t.slope;
        }
      }
    }
    if (a.dn) {
      float hat[kPer], t[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kPer; k++) {
        const bool in = on && col<T, VEC, TPR>(lane, k) < a.D;
        const float s = BLOCK ? (float)rr[k] + scale[k] * (av[k] * u[k]) : (float)rr[k];
        hat[k] = in ? (s - st.v[2]) * st.v[3] : 0.f;
        const float dn = (float)rdn[k];
        sum[kPreW][k] += dn * hat[k];
        if (BIAS) sum[kPreB][k] += dn;
        const float dv = in ? dn * pre_w[k] : 0.f;
        t[0] += dv * hat[k];
        t[1] += dv;
      }
      row_sum<TPR, 2>(t, shared);
      const float c0 = t[0] * inv, c1 = a.layer ? t[1] * inv : 0.f;
#pragma unroll
      for (int k = 0; k < kPer; k++) ds[k] += ((float)rdn[k] * pre_w[k] - hat[k] * c0 - c1) * st.v[3];
    }
    if (a.dr) write<T, VEC, TPR>(static_cast<T*>(a.dr) + row * a.drs, lane, a.D, on, ds);
    if (BLOCK) {
      float dp[kPer], dg[kPer], t[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kPer; k++) {
        const bool in = on && col<T, VEC, TPR>(lane, k) < a.D;
        if (in) sum[kScale][k] += ds[k] * (av[k] * u[k]);
        const float dw = ds[k] * scale[k];
        dg[k] = dw * u[k] * slope[k];
        dp[k] = in && (keep >> k & 1u) ? dw * av[k] * a.drop.scale : 0.f;
        if (a.post) {
          if (in) sum[kPostW][k] += dp[k] * yhat[k];
          if (BIAS) sum[kPostB][k] += dp[k];
          dp[k] *= post_w[k];
          if (in) t[0] += dp[k] * yhat[k];
          t[1] += dp[k];
        }
      }
      if (a.gate && a.dgate) write<T, VEC, TPR>(static_cast<T*>(a.dgate) + row * a.dgs, lane, a.D, on, dg);
      if (a.post) {
        row_sum<TPR, 2>(t, shared);
        const float c0 = t[0] * inv, c1 = a.layer ? t[1] * inv : 0.f;
#pragma unroll
        for (int k = 0; k < kPer; k++) dp[k] = (dp[k] - yhat[k] * c0 - c1) * st.v[1];
      }
      if (a.dy) write<T, VEC, TPR>(static_cast<T*>(a.dy) + row * a.dys, lane, a.D, on, dp);
    }
  }
  if (!a.sums) return;
  float* out = a.sums + (ll)blockIdx.x * kSums * a.D;
#pragma unroll
  for (int q = 0; q < kSums; q++) {
    if (!BLOCK && q < kPreW) continue;
    if (!BIAS && (q == kPostB || q == kPreB)) continue;
    if constexpr (kGroups > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kPer; k++) join[k * block_of(TPR) + threadIdx.x] = sum[q][k];
      __syncthreads();
      if (group == 0)
#pragma unroll
        for (int k = 0; k < kPer; k++) {
          float t = 0.f;
          for (int g = 0; g < kGroups; g++) t += join[k * block_of(TPR) + g * TPR + lane];
          sum[q][k] = t;
        }
    }
    if (group == 0)
#pragma unroll
      for (int k = 0; k < kPer; k++) {
        const int c = col<T, VEC, TPR>(lane, k);
        if (c < a.D) out[q * a.D + c] = sum[q][k];
      }
  }
}

struct Join {
  const float* sums; int parts, D, rows32;  // rows32: outputs are float32 (else T)
  void* out[kSums];
  int scale_one;
  float* scale_cols;  // the scale's column sums where one scale serves all columns
};

// Column sums of the workgroups' partial sums: 64 columns by 4 strands of workgroups, joined in their order.
template <class T>
__global__ __launch_bounds__(256) void resnorm_join(const Join j) {
  __shared__ float strand[4][64];
  const int q = blockIdx.y, c = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  if (!j.out[q]) return;
  float t = 0.f;
  if (c < j.D)
    for (int p = w; p < j.parts; p += 4) t += j.sums[((ll)p * kSums + q) * j.D + c];
  strand[w][threadIdx.x & 63] = t;
  __syncthreads();
  if (w || c >= j.D) return;
  t = (strand[0][threadIdx.x] + strand[1][threadIdx.x]) + (strand[2][threadIdx.x] + strand[3][threadIdx.x]);
  if (q == kScale && j.scale_one)
    j.scale_cols[c] = t;
  else if (j.rows32)
    static_cast<float*>(j.out[q])[c] = t;
  else
    static_cast<T*>(j.out[q])[c] = (T)t;
}
template <class T>
__global__ __launch_bounds__(256) void resnorm_join_scale(const Join j) {
  __shared__ float part[256];
  float t = 0.f;
  for (int c = threadIdx.x; c < j.D; c += 256) t += j.scale_cols[c];
  part[threadIdx.x] = t;
  __syncthreads();
  for (int m = 128; m > 0; m >>= 1) {
    if ((int)threadIdx.x < m) part[threadIdx.x] += part[threadIdx.x + m];
    __syncthreads();
  }
  if (threadIdx.x) return;
  if (j.rows32)
    *static_cast<float*>(j.out[kScale]) = part[0];
  else
    *static_cast<T*>(j.out[kScale]) = (T)part[0];
}

// ---- dropout alone ------------------------------------------------------------------
struct DropArgs {
  const void* x; ll xs;
  void* y; ll ysd;
  ll rows; int cols;  // x rows of `cols` elements at stride xs (one row: flat)
  ll count;
  Drop drop;
  mjh_i64* ctr_out;
};

template <class T, int V>
__global__ __launch_bounds__(256) void dropout_flat(const DropArgs a) {
  const unsigned long long base = drop_base(a.drop);
  if (a.ctr_out && blockIdx.x == 0 && threadIdx.x == 0) *a.ctr_out = a.drop.ctr ? *a.drop.ctr : 0;
  for (ll i = ((ll)blockIdx.x * 256 + threadIdx.x) * V; i < a.count; i += (ll)gridDim.x * 256 * V) {
    const auto x = load<T, V>(static_cast<const T*>(a.x) + i);
    float o[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
      const unsigned long long w = drop_word(base, (unsigned long long)(i + j) >> 1);
      o[j] = drop_keep(w, V > 1 ? j & 1 : (int)((i + j) & 1), a.drop.thr) ? (float)x.v[j] * a.drop.scale : 0.f;
    }
    store<T, V>(static_cast<T*>(a.y) + i, o);
  }
}
template <class T>
__global__ __launch_bounds__(256) void dropout_rows(const DropArgs a) {
  const unsigned long long base = drop_base(a.drop);
  if (a.ctr_out && blockIdx.x == 0 && threadIdx.x == 0) *a.ctr_out = a.drop.ctr ? *a.drop.ctr : 0;
  for (ll i = (ll)blockIdx.x * 256 + threadIdx.x; i < a.count; i += (ll)gridDim.x * 256) {
    const ll row = i / a.cols, c = i - row * a.cols;
    const float x = (float)static_cast<const T*>(a.x)[row * a.xs + c];
    const bool keep = drop_keep(drop_word(base, (unsigned long long)i >> 1), (int)(i & 1), a.drop.thr);
    static_cast<T*>(a.y)[row * a.ysd + c] = (T)(keep ? x * a.drop.scale : 0.f);
  }
}

// ---- host side ------------------------------------------------------------------------
int tpr_of(int D) {
  int t = 8;
  while (t * kPer < D) t *= 2;
  return t;
}

// 16-byte pieces need every row of every tensor aligned to them
bool vectors(const mjh_resnorm_desc& d) {
  const size_t e = d.dtype == MJH_F32 ? 4 : 2;
  const ll v = 16 / (ll)e;
  if (d.D % v) return false;
  for (ll s : {d.ys, d.rs, d.gs, d.ss, d.ns, d.dss, d.dns, d.dys, d.drs, d.dgs})
    if (s % v) return false;
  for (const void* p : {d.y, d.r, d.gate, (const void*)d.s, (const void*)d.n, d.ds, d.dn, (const void*)d.dy,
                        (const void*)d.dr, (const void*)d.dgate})
    if (!aligned(p, 16)) return false;
  return true;
}

int check(const mjh_resnorm_desc* d) {
  if (!d) return refuse("residual norm: no description");
  if (d->R < 1 || d->D < 1) return refuse("residual norm: R and D must be positive");
  if (d->D > kMaxTpr * kPer) return refuse("residual norm: D is at most 8192");
  if (d->R > 0x7fffffffll) return refuse("residual norm: R must be below 2^31");
  if (d->dtype < 0 || d->dtype > 2) return refuse("residual norm: unknown type");
  if (!d->r) return refuse("residual norm: the residual is needed");
  if (!d->y && (d->gate || d->post || d->scale)) return refuse("residual norm: gate, post norm and scale need y");
  if (d->thr > (1ull << 32)) return refuse("dropout: threshold above 2^32");
  return 0;
}

Args args_of(const mjh_resnorm_desc& d) {
  Args a;
  std::memset(&a, 0, sizeof(a));
  a.y = d.y; a.ys = d.ys;
  a.r = d.r; a.rs = d.rs;
  a.gate = d.gate; a.gs = d.gs;
  a.post_w = d.post_w; a.post_b = d.post_b; a.pre_w = d.pre_w; a.pre_b = d.pre_b; a.scale = d.scale;
  a.w32 = d.w32;
  a.scale_one = d.scale && d.scale_one;
  a.s = d.s; a.ss = d.ss;
  a.n = d.n; a.ns = d.ns;
  a.stats = d.stats;
  a.ds = d.ds; a.dss = d.dss;
  a.dn = d.dn; a.dns = d.dns;
  a.dy = d.dy; a.dys = d.dys;
  a.dr = d.dr; a.drs = d.drs;
  a.dgate = d.dgate; a.dgs = d.dgs;
  a.drop = {d.seed, d.key, d.ctr, d.thr, d.thr ? d.drop_scale : 1.f};
  a.ctr_out = d.ctr_out;
  a.eps = d.eps;
  a.R = (int)d.R; a.D = d.D; a.layer = d.layer; a.act = d.act; a.post = d.post; a.pre = d.pre;
  return a;
}

unsigned grid_of(int tpr, ll rows, bool back) {
  const int groups = block_of(tpr) / tpr;
  const ll need = (rows + groups - 1) / groups;
  if (!back) return (unsigned)std::min<ll>(need, 256 * 16);
  // backward: workgroups write partial sums, so each takes several rows per group
  return (unsigned)std::max<ll>(1, std::min<ll>(need / 8, 1024));
}

bool wants_bias(const mjh_resnorm_desc& d) { return d.post_b || d.pre_b; }

template <class T, bool VEC, int TPR>
void launch_tpr(const Args& a, bool back, bool bias, hipStream_t s) {
  const dim3 grid(grid_of(TPR, a.R, back)), block(block_of(TPR));
  if (!back)
    resnorm_forward<T, VEC, TPR><<<grid, block, 0, s>>>(a);
  else if (a.y)
    bias ? resnorm_backward<T, VEC, TPR, true, true><<<grid, block, 0, s>>>(a)
         : resnorm_backward<T, VEC, TPR, true, false><<<grid, block, 0, s>>>(a);
  else
    bias ? resnorm_backward<T, VEC, TPR, false, true><<<grid, block, 0, s>>>(a)
         : resnorm_backward<T, VEC, TPR, false, false><<<grid, block, 0, s>>>(a);
}
template <class T, bool VEC>
void launch_rows(const Args& a, bool back, bool bias, hipStream_t s) {
  switch (tpr_of(a.D)) {
    case 8: return launch_tpr<T, VEC, 8>(a, back, bias, s);
    case 16: return launch_tpr<T, VEC, 16>(a, back, bias, s);
    case 32: return launch_tpr<T, VEC, 32>(a, back, bias, s);
    case 64: return launch_tpr<T, VEC, 64>(a, back, bias, s);
    case 128: return launch_tpr<T, VEC, 128>(a, back, bias, s);
    case 256: return launch_tpr<T, VEC, 256>(a, back, bias, s);
    case 512: return launch_tpr<T, VEC, 512>(a, back, bias, s);
    default: return launch_tpr<T, VEC, 1024>(a, back, bias, s);
  }
}
template <class T>
void launch_type(const mjh_resnorm_desc& d, const Args& a, bool back, hipStream_t s) {
  vectors(d) ? launch_rows<T, true>(a, back, wants_bias(d), s) : launch_rows<T, false>(a, back, wants_bias(d), s);
}
void launch(const mjh_resnorm_desc& d, const Args& a, bool back, hipStream_t s) {
  if (d.dtype == MJH_F32)
    launch_type<float>(d, a, back, s);
  else if (d.dtype == MJH_BF16)
    launch_type<bf16>(d, a, back, s);
  else
    launch_type<f16>(d, a, back, s);
}

template <class T>
void launch_join(const Join& j, hipStream_t s) {
  resnorm_join<T><<<dim3((j.D + 63) / 64, kSums), dim3(256), 0, s>>>(j);
  if (j.scale_one && j.out[kScale]) resnorm_join_scale<T><<<dim3(1), dim3(256), 0, s>>>(j);
}

template <class T>
void launch_dropout(const DropArgs& a, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const ll most = 256 * 32;
  if (a.rows == 1 && a.count % V == 0 && aligned(a.x, 16) && aligned(a.y, 16)) {
    const ll n = (a.count / V + 255) / 256;
    dropout_flat<T, V><<<dim3((unsigned)std::min(n, most)), dim3(256), 0, s>>>(a);
  } else {
    const ll n = (a.count + 255) / 256;
    if (a.rows == 1)
      dropout_flat<T, 1><<<dim3((unsigned)std::min(n, most)), dim3(256), 0, s>>>(a);
    else
      dropout_rows<T><<<dim3((unsigned)std::min(n, most)), dim3(256), 0, s>>>(a);
  }
}

}  // namespace

extern "C" {

long long mjh_resnorm_workspace(const mjh_resnorm_desc* d) {
  if (check(d)) return -1;
  return 4 * ((ll)grid_of(tpr_of(d->D), d->R, true) * kSums * d->D + d->D);
}

int mjh_resnorm_forward(const mjh_resnorm_desc* d, void* stream) {
  if (int rc = check(d)) return rc;
  if ((d->y && !d->s) || (d->pre && !d->n) || (!d->y && !d->pre)) return refuse("residual norm forward: an output is missing");
  launch(*d, args_of(*d), false, reinterpret_cast<hipStream_t>(stream));
  return launched();
}

int mjh_resnorm_backward(const mjh_resnorm_desc* d, void* stream) {
  if (int rc = check(d)) return rc;
  if (!d->stats || (!d->ds && !d->dn) || (d->dn && !d->pre)) return refuse("residual norm backward: statistics or gradients are missing");
  const bool sums = d->d_post_w || d->d_post_b || d->d_scale || d->d_pre_w || d->d_pre_b;
  if (sums && (!d->ws || d->ws_bytes < mjh_resnorm_workspace(d))) return refuse("residual norm backward: workspace too small");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Args a = args_of(*d);
  a.sums = sums ? static_cast<float*>(d->ws) : nullptr;
  launch(*d, a, true, s);
  if (int rc = launched()) return rc;
  if (!sums) return 0;
  Join j;
  std::memset(&j, 0, sizeof(j));
  j.sums = a.sums;
  j.parts = (int)grid_of(tpr_of(a.D), a.R, true);
  j.D = a.D;
  j.rows32 = a.w32;
  j.out[kPostW] = d->d_post_w; j.out[kPostB] = d->d_post_b; j.out[kScale] = d->d_scale;
  j.out[kPreW] = d->d_pre_w; j.out[kPreB] = d->d_pre_b;
  j.scale_one = a.scale_one;
  j.scale_cols = a.sums + (ll)j.parts * kSums * a.D;
  if (d->dtype == MJH_F32)
    launch_join<float>(j, s);
  else if (d->dtype == MJH_BF16)
    launch_join<bf16>(j, s);
  else
    launch_join<f16>(j, s);
  return launched();
}

int mjh_dropout(const void* x, long long xs, void* y, long long ys, long long rows, int cols, int dtype, float scale,
                unsigned long long thr, unsigned long long seed, unsigned long long key, const mjh_i64* ctr,
                mjh_i64* ctr_out, void* stream) {
  if (rows < 0 || cols < 0) return refuse("dropout: negative size");
  if (dtype < 0 || dtype > 2) return refuse("dropout: unknown type");
  if (thr > (1ull << 32)) return refuse("dropout: threshold above 2^32");
  if (rows == 0 || cols == 0) return 0;
  if (!x || !y) return refuse("dropout: x and y are needed");
  DropArgs a;
  a.x = x; a.xs = xs; a.y = y; a.ysd = ys;
  a.count = rows * cols;
  const bool flat = rows == 1 || (xs == cols && ys == cols);
  a.rows = flat ? 1 : rows;
  a.cols = cols;
  a.drop = {seed, key, ctr, thr, scale};
  a.ctr_out = ctr_out;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MJH_F32)
    launch_dropout<float>(a, s);
  else if (dtype == MJH_BF16)
    launch_dropout<bf16>(a, s);
  else
    launch_dropout<f16>(a, s);
  return launched();
}

}  // extern "C"
