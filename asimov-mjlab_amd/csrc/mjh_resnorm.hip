// mjh_resnorm.hip — a residual block's epilogue fused with the next block's norm, and dropout (gfx950).
//
//   p = norm_post(y)            (x - mean) rstd w + b; rms: mean = 0; without post weights p = y
//   u = keep ? p / (1 - prob) : 0      counter-based bits (mjh_seq.h), nothing stored
//   s = residual + scale * act(gate) * u
//   n = norm_pre(s)
// The statistics, s inside n, and all sums are float32; s and n are rounded once, at their store.
//
// Rows of up to 2,048 elements (16-bit types: 4,096; forward also float32 rows of up to 4,096 that fill their waves,
// 2,047 x 4,096: 39 us, 49 as streams): a group of lanes holds a row, 8 elements a lane, so every tensor is read once
// and every statistic is taken from registers (the variance around the mean, in a second pass over registers). One lane
// (rows shorter than 16 bytes) to 64, several rows a workgroup, or a workgroup of two to eight waves. Longer rows:
// streams over the row, which read it again, largely from the caches, where holding it would leave a CU one workgroup
// and nothing to hide its barriers (2,048 x 8,192 bfloat16, forward: 57 us, 63 held by 16 waves).
// The backward pass keeps s and p nowhere: it forms them again from y, residual and gate, the tensors that it has to
// read in any case, with the forward pass's (mean, rstd) of each row. Weight gradients: a group (a thread that owns
// columns) adds its rows in registers, groups of a workgroup join in shared memory, workgroups in a second launch,
// each in a fixed order.
#include <algorithm>
#include <cstring>

#include "mjh_seq.h"

namespace {
using namespace mjh_seq;

constexpr int kPer = 8;  // elements a lane holds
constexpr ll kColumnWaves = 256 * 4 * 4;  // waves of the long rows' column stream: 4 a SIMD
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
  float* sums;    // (parts, kSums, D)
  float* coef;    // (R, 4): the row sums of the long rows' backward pass
  mjh_i64* ctr_out;
  Drop drop;
  float eps, inv;  // inv = 1 / D
  int R, D, layer, act, post, pre;
  ll row0;    // long rows: the first row of this launch
  int tpr;    // lanes that hold a row
  int parts;  // workgroups (long rows: strands of rows) of the backward pass
};

// The sum over groups of L neighbouring lanes, in every lane: four steps inside a row of 16 lanes (neighbours, pairs,
// then mirrored halves, whose lanes hold equal sums by then), the rest by lane exchange.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int L>
__device__ __forceinline__ float lane_sum(float v) {
  if (L == 1) return v;
  v += dpp<0xB1>(v);                 // quad_perm 1 0 3 2
  v += dpp<0x4E>(v);                 // quad_perm 2 3 0 1
  v += dpp<0x141>(v);                // row_half_mirror
  if (L >= 16) v += dpp<0x140>(v);   // row_mirror
  if (L >= 32) v += __shfl_xor(v, 16);
  if (L >= 64) v += __shfl_xor(v, 32);
  return v;
}

// Where a lane's N neighbouring elements of a row lie: slot p holds elements p N and on. What is left of a row that N
// does not divide (kTail) is the end of the row's last N elements, of which the slot's own are marked: every lane reads
// whole pieces and none in a branch, whose result would be waited for there (98,304 x 99 floats, backward: 75 us, 96
// with a branch for single elements).
// kWhole: every slot is a piece of its own. kTiny: rows shorter than a piece, slot 0 reads them element by element.
enum { kWhole, kTail, kTiny };
template <class T, int N, int FIT>
struct Piece {
  static constexpr unsigned kAll = (1u << N) - 1u;
  int c;          // first column read
  unsigned mask;  // bit j: element c + j is the slot's own
  __device__ __forceinline__ Piece() {}
  __device__ __forceinline__ Piece(int p, int D) : c(p * N), mask(kAll) {
    if (FIT == kTail) {
      c = min(c, D - N);
      const int skip = p * N - c;
      mask = skip >= N ? 0u : kAll << skip & kAll;
    } else if (FIT == kTiny) {
      c = 0;
      mask = p ? 0u : (1u << D) - 1u;
    }
  }
  __device__ __forceinline__ bool has(int j) const { return FIT == kWhole || (mask >> j & 1u); }
  template <class W>
  __device__ __forceinline__ Pack<W, N> get(const W* q) const {
    if constexpr (FIT != kTiny) return load_loose<W, N>(q + c);
    Pack<W, N> v{};
#pragma unroll
    for (int j = 0; j < N; j++)
      if (has(j)) v.v[j] = q[j];
    return v;
  }
  __device__ __forceinline__ Pack<T, N> read(const void* p, ll row, ll step) const {
    return get(static_cast<const T*>(p) + row * step);
  }
  __device__ __forceinline__ void write(void* p, ll row, ll step, const float (&f)[N]) const {
    T* q = static_cast<T*>(p) + row * step + c;
    if (FIT == kWhole || mask == kAll) {
      store_loose<T, N>(q, f);
    } else {
#pragma unroll
      for (int j = 0; j < N; j++)
        if (has(j)) q[j] = (T)f[j];
    }
  }
  // channel weights; `none` where there are none
  __device__ __forceinline__ void weights(const void* w, int w32, float none, float* o) const {
#pragma unroll
    for (int j = 0; j < N; j++) o[j] = none;
    if (!w) return;
    if (w32) {
      const auto v = get(static_cast<const float*>(w));
#pragma unroll
      for (int j = 0; j < N; j++) o[j] = v.v[j];
    } else {
      const auto v = get(static_cast<const T*>(w));
#pragma unroll
      for (int j = 0; j < N; j++) o[j] = (float)v.v[j];
    }
  }
  __device__ __forceinline__ void scales(const Args& a, float* o) const {
    if (!a.scale_one) return weights(a.scale, a.w32, 1.f, o);
    const float one = a.w32 ? *static_cast<const float*>(a.scale) : (float)*static_cast<const T*>(a.scale);
#pragma unroll
    for (int j = 0; j < N; j++) o[j] = one;
  }
  // keep bits (bit j: element j). Neighbours share a word, and the words of a piece are one addition apart; a piece
  // that begins at an odd index begins with the second half of a word.
  template <bool EVEN>  // D and c are even
  __device__ __forceinline__ unsigned keep_bits(unsigned long long base, const Drop& d, ll row, int D) const {
    const unsigned long long i = (unsigned long long)(row * D + c);
    unsigned long long z = base + ((i >> 1) + 1ull) * 0x9e3779b97f4a7c15ull, w = mjh::mix64(z);
    unsigned bits = 0;
    const bool odd = !EVEN && (i & 1);
    if (odd) bits = drop_keep(w, 1, d.thr);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      if (j > 0 || odd) {
        z += 0x9e3779b97f4a7c15ull;
        w = mjh::mix64(z);
      }
      const unsigned low = drop_keep(w, 0, d.thr), high = drop_keep(w, 1, d.thr);
      bits |= (low | high << 1) << (j + (odd ? 1 : 0));
    }
    return bits;
  }
};

__device__ __forceinline__ unsigned long long drop_base(const Drop& d) { return mjh::Rng(d.seed, d.key, d.ctr).base; }

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

// act(gate) (and its slope) of a lane's elements; one branch for all
template <class T, bool SLOPE, int N>
__device__ __forceinline__ void activate(const T (&g)[N], const Args& a, float (&value)[N], float (&slope)[N]) {
  if (!a.gate) {
#pragma unroll
    for (int k = 0; k < N; k++) value[k] = 1.f, slope[k] = 0.f;
  } else if (a.act == MJH_ACT_SIGMOID) {
#pragma unroll
    for (int k = 0; k < N; k++) {
      const Act t((float)g[k], MJH_ACT_SIGMOID);
      value[k] = t.value;
      if (SLOPE) slope[k] = t.slope;
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; k++) {
      const Act t((float)g[k], MJH_ACT_SILU);
      value[k] = t.value;
      if (SLOPE) slope[k] = t.slope;
    }
  }
}

// ---- rows held in registers -------------------------------------------------------------
// TPR: 1 (rows shorter than a piece), or 8 to 64 lanes hold a row; 256, 512: a workgroup of a.tpr threads (whole
// waves) does.
constexpr int threads_of(int tpr) { return tpr > 256 ? tpr : 256; }
template <class T, bool FULL, int TPR>
struct Row {
  static constexpr int N = 16 / (int)sizeof(T), kPieces = kPer / N;
  static constexpr bool kWaves = TPR > 64;
  static constexpr int kGroups = kWaves ? 1 : 256 / TPR;  // rows a workgroup holds
  int group, lane, lanes, D, turn = 0;
  typedef Piece<T, N, (FULL ? kWhole : TPR == 1 ? kTiny : kTail)> At;
  At at[kPieces];
  __device__ __forceinline__ explicit Row(const Args& a) : D(a.D) {
    lanes = kWaves ? a.tpr : TPR;
    lane = kWaves ? threadIdx.x : threadIdx.x % TPR;
    group = kWaves ? 0 : threadIdx.x / TPR;
#pragma unroll
    for (int k = 0; k < kPieces; k++) at[k] = At(k * lanes + lane, a.D);
  }
  __device__ __forceinline__ bool has(int k) const { return at[k / N].has(k % N); }
  __device__ __forceinline__ void read(const void* p, ll row, ll step, T (&o)[kPer]) const {
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
      const auto v = at[k].read(p, row, step);
#pragma unroll
      for (int j = 0; j < N; j++) o[k * N + j] = v.v[j];
    }
  }
  __device__ __forceinline__ void write(void* p, ll row, ll step, bool on, const float (&f)[kPer]) const {
    if (!on) return;
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
      float o[N];
#pragma unroll
      for (int j = 0; j < N; j++) o[j] = f[k * N + j];
      at[k].write(p, row, step, o);
    }
  }
  __device__ __forceinline__ void weights(const void* w, int w32, float none, float (&o)[kPer]) const {
#pragma unroll
    for (int k = 0; k < kPieces; k++) at[k].weights(w, w32, none, o + k * N);
  }
  __device__ __forceinline__ void scales(const Args& a, float (&o)[kPer]) const {
#pragma unroll
    for (int k = 0; k < kPieces; k++) at[k].scales(a, o + k * N);
  }
  __device__ __forceinline__ unsigned keep_bits(unsigned long long base, const Drop& d, ll row) const {
    unsigned bits = 0;
#pragma unroll
    for (int k = 0; k < kPieces; k++) bits |= (at[k].template keep_bits<FULL>(base, d, row, D) & ((1u << N) - 1u)) << (k * N);
    return bits;
  }
  // Sums of NV values over a row's lanes, in every lane. Several waves: through shared memory (2 x 8 x 2 floats), in
  // turns of two halves, so that one barrier keeps a turn's writes from the reads of the turn before the last.
  template <int NV>
  __device__ __forceinline__ void sum(float (&v)[NV], float (*shared)[16]) {
#pragma unroll
    for (int k = 0; k < NV; k++) v[k] = lane_sum<(kWaves ? 64 : TPR)>(v[k]);
    if constexpr (kWaves) {
      float* const s = shared[turn];
      turn ^= 1;
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < NV; k++) s[(threadIdx.x >> 6) * 2 + k] = v[k];
      __syncthreads();
      const int waves = lanes >> 6;
#pragma unroll
      for (int k = 0; k < NV; k++) v[k] = s[k] + s[2 + k];
#pragma unroll
      for (int j = 2; j < TPR / 64; j++)
        if (j < waves)
#pragma unroll
          for (int k = 0; k < NV; k++) v[k] += s[j * 2 + k];
    }
  }
  // mean and 1 / deviation of a row held in registers
  __device__ __forceinline__ void stats(const float (&v)[kPer], const Args& a, float (*shared)[16], float& mean, float& rstd) {
    mean = 0.f;
    float t[1];
    if (a.layer) {
      t[0] = 0.f;
#pragma unroll
      for (int k = 0; k < kPer; k++) t[0] += has(k) ? v[k] : 0.f;
      sum<1>(t, shared);
      mean = t[0] * a.inv;
    }
    t[0] = 0.f;
#pragma unroll
    for (int k = 0; k < kPer; k++) {
      const float c = has(k) ? v[k] - mean : 0.f;
      t[0] += c * c;
    }
    sum<1>(t, shared);
    rstd = __builtin_amdgcn_rsqf(__builtin_fmaf(t[0], a.inv, a.eps));  // to 1 ulp
  }
};

// Bound by bytes (98,304 x 256 bfloat16, all parts: 60 us, 4.2 TB/s, 55 at the least; 16,384 x 2,048: 50 us, 5.3
// TB/s); for a few rows by its chain of sums (16 x 1,000 float16: 5.0 us).
template <class T, bool FULL, int TPR>
__global__ __launch_bounds__(threads_of(TPR)) void resnorm_forward(const Args a) {
  typedef Row<T, FULL, TPR> R;
  __shared__ float shared[2][16];
  R at(a);
  if (a.ctr_out && blockIdx.x == 0 && threadIdx.x == 0) *a.ctr_out = a.drop.ctr ? *a.drop.ctr : 0;
  const bool block = a.y != nullptr;
  const unsigned long long base = a.drop.thr ? drop_base(a.drop) : 0;
  float post_w[kPer], post_b[kPer], pre_w[kPer], pre_b[kPer], scale[kPer];
  at.weights(a.post_w, a.w32, 1.f, post_w);
  at.weights(a.post_b, a.w32, 0.f, post_b);
  at.weights(a.pre_w, a.w32, 1.f, pre_w);
  at.weights(a.pre_b, a.w32, 0.f, pre_b);
  at.scales(a, scale);
  T raw[kPer], raw_y[kPer], raw_g[kPer];
  auto fetch = [&](ll row) {
    row = min(row, (ll)a.R - 1);
    at.read(a.r, row, a.rs, raw);
    if (block) at.read(a.y, row, a.ys, raw_y);
    if (a.gate) at.read(a.gate, row, a.gs, raw_g);
  };
  const ll step = (ll)gridDim.x * R::kGroups;
  fetch((ll)blockIdx.x * R::kGroups + at.group);
  for (ll first = (ll)blockIdx.x * R::kGroups; first < a.R; first += step) {
    const ll row = first + at.group;
    const bool on = row < a.R;
    float s[kPer], mean = 0.f, rstd = 1.f, pre_mean = 0.f, pre_rstd = 1.f;
#pragma unroll
    for (int k = 0; k < kPer; k++) s[k] = (float)raw[k];
    if (block) {
      float p[kPer], av[kPer], slope[kPer];
#pragma unroll
      for (int k = 0; k < kPer; k++) p[k] = (float)raw_y[k];
      if (a.post) {
        at.stats(p, a, shared, mean, rstd);
#pragma unroll
        for (int k = 0; k < kPer; k++) p[k] = __builtin_fmaf((p[k] - mean) * rstd, post_w[k], post_b[k]);
      }
      if (a.drop.thr) {
        const unsigned keep = at.keep_bits(base, a.drop, row);
#pragma unroll
        for (int k = 0; k < kPer; k++) p[k] = (keep >> k & 1u) ? p[k] * a.drop.scale : 0.f;
      }
      activate<T, false>(raw_g, a, av, slope);
#pragma unroll
      for (int k = 0; k < kPer; k++) s[k] = __builtin_fmaf(scale[k], av[k] * p[k], s[k]);
      at.write(a.s, row, a.ss, on, s);
    }
    if (a.pre) {
      at.stats(s, a, shared, pre_mean, pre_rstd);
#pragma unroll
      for (int k = 0; k < kPer; k++) s[k] = __builtin_fmaf((s[k] - pre_mean) * pre_rstd, pre_w[k], pre_b[k]);
      at.write(a.n, row, a.ns, on, s);
    }
    if (a.stats && on && at.lane == 0) store<float, 4>(a.stats + row * 4, {mean, rstd, pre_mean, pre_rstd});
    fetch(row + step);
  }
}

// Bound by bytes (98,304 x 256 bfloat16, all parts: 88 us, 4.6 TB/s, 81 at the least; 16,384 x 2,048 without gate: 86
// us, 4.7 TB/s).
// BLOCK: there is a y (else only the norm before). BIAS: there are biases.
template <class T, bool FULL, int TPR, bool BLOCK, bool BIAS>
__global__ __launch_bounds__(threads_of(TPR)) void resnorm_backward(const Args a) {
  typedef Row<T, FULL, TPR> R;
  __shared__ float shared[2][16];
  __shared__ float join[R::kGroups > 1 ? 256 * kPer : 1];
  R at(a);
  const unsigned long long base = BLOCK && a.drop.thr ? drop_base(a.drop) : 0;
  float post_w[kPer], post_b[kPer], pre_w[kPer], scale[kPer];
  at.weights(a.pre_w, a.w32, 1.f, pre_w);
  if (BLOCK) {
    at.weights(a.post_w, a.w32, 1.f, post_w);
    if (BIAS) at.weights(a.post_b, a.w32, 0.f, post_b);
    at.scales(a, scale);
  }
  float sum[kSums][kPer];
#pragma unroll
  for (int q = 0; q < kSums; q++)
#pragma unroll
    for (int k = 0; k < kPer; k++) sum[q][k] = 0.f;
  // Rows behind the last read the last again (a branch would wait for its loads) and count for nothing.
  // The row ahead is loaded only where one workgroup fills a CU, which then waits for its loads and barriers alone
  // (8,192 x 4,096 bfloat16: 165 us, 194 without; 98,304 x 256: 108 us with it, 85 without).
  constexpr bool AHEAD = TPR > 256;
  auto fetch = [&](ll row, Pack<float, 4>& st, T (&r)[kPer], T (&y)[kPer], T (&g)[kPer], T (&ds)[kPer], T (&dn)[kPer]) {
    row = min(row, (ll)a.R - 1);
    st = load<float, 4>(a.stats + row * 4);
    if (BLOCK) {
      at.read(a.y, row, a.ys, y);
      if (a.gate) at.read(a.gate, row, a.gs, g);
    }
    if (a.dn) {
      at.read(a.r, row, a.rs, r);
      at.read(a.dn, row, a.dns, dn);
    }
    if (a.ds) at.read(a.ds, row, a.dss, ds);
  };
  T next_r[kPer], next_y[kPer], next_g[kPer], next_ds[kPer], next_dn[kPer];
  Pack<float, 4> next_st{};
  if constexpr (AHEAD) fetch((ll)blockIdx.x * R::kGroups + at.group, next_st, next_r, next_y, next_g, next_ds, next_dn);
  for (ll first = (ll)blockIdx.x * R::kGroups; first < a.R; first += (ll)gridDim.x * R::kGroups) {
    const ll row = first + at.group;
    const bool on = row < a.R;
    T raw_r[kPer], raw_y[kPer], raw_g[kPer], raw_ds[kPer], raw_dn[kPer];
    Pack<float, 4> st{};
    if constexpr (AHEAD) {
      st = next_st;
#pragma unroll
      for (int k = 0; k < kPer; k++) {
        raw_r[k] = next_r[k]; raw_y[k] = next_y[k]; raw_g[k] = next_g[k]; raw_ds[k] = next_ds[k]; raw_dn[k] = next_dn[k];
      }
      fetch(row + (ll)gridDim.x * R::kGroups, next_st, next_r, next_y, next_g, next_ds, next_dn);
    } else {
      fetch(row, st, raw_r, raw_y, raw_g, raw_ds, raw_dn);
    }
    const float mean = st.v[0], rstd = st.v[1], pre_mean = st.v[2], pre_rstd = st.v[3];
    bool in[kPer];
#pragma unroll
    for (int k = 0; k < kPer; k++) in[k] = on && at.has(k);
    float ds[kPer], yhat[kPer], u[kPer], av[kPer], slope[kPer];
    unsigned keep = ~0u;
#pragma unroll
    for (int k = 0; k < kPer; k++) ds[k] = 0.f;
    if (a.ds) {
#pragma unroll
      for (int k = 0; k < kPer; k++) ds[k] = (float)raw_ds[k];
    }
    if (BLOCK) {
#pragma unroll
      for (int k = 0; k < kPer; k++) u[k] = yhat[k] = (float)raw_y[k];
      if (a.post) {
#pragma unroll
        for (int k = 0; k < kPer; k++) {
          yhat[k] = (yhat[k] - mean) * rstd;
          u[k] = BIAS ? __builtin_fmaf(yhat[k], post_w[k], post_b[k]) : yhat[k] * post_w[k];
        }
      }
      if (a.drop.thr) {
        keep = at.keep_bits(base, a.drop, row);
#pragma unroll
        for (int k = 0; k < kPer; k++) u[k] = (keep >> k & 1u) ? u[k] * a.drop.scale : 0.f;
      }
      activate<T, true>(raw_g, a, av, slope);
    }
    if (a.dn) {
      float hat[kPer], t[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kPer; k++) {
        const float r = (float)raw_r[k];
        const float s = BLOCK ? __builtin_fmaf(scale[k], av[k] * u[k], r) : r;
        hat[k] = in[k] ? (s - pre_mean) * pre_rstd : 0.f;
        const float dn = (float)raw_dn[k];
        if (in[k]) sum[kPreW][k] += dn * hat[k];
        if (BIAS) sum[kPreB][k] += in[k] ? dn : 0.f;
        const float dv = in[k] ? dn * pre_w[k] : 0.f;
        t[0] += dv * hat[k];
        t[1] += dv;
      }
      at.template sum<2>(t, shared);
      const float c0 = t[0] * a.inv, c1 = a.layer ? t[1] * a.inv : 0.f;
#pragma unroll
      for (int k = 0; k < kPer; k++) ds[k] += ((float)raw_dn[k] * pre_w[k] - hat[k] * c0 - c1) * pre_rstd;
    }
    if (a.dr) at.write(a.dr, row, a.drs, on, ds);
    if (BLOCK) {
      float dg[kPer], t[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kPer; k++) {
        if (in[k]) sum[kScale][k] += ds[k] * (av[k] * u[k]);
        const float dw = ds[k] * scale[k];
        dg[k] = dw * u[k] * slope[k];
        ds[k] = in[k] ? dw * av[k] : 0.f;
      }
      if (a.drop.thr) {
#pragma unroll
        for (int k = 0; k < kPer; k++) ds[k] = (keep >> k & 1u) ? ds[k] * a.drop.scale : 0.f;
      }
      if (a.gate && a.dgate) at.write(a.dgate, row, a.dgs, on, dg);
      if (a.post) {
#pragma unroll
        for (int k = 0; k < kPer; k++) {
          if (in[k]) sum[kPostW][k] += ds[k] * yhat[k];
          if (BIAS) sum[kPostB][k] += ds[k];
          ds[k] *= post_w[k];
          if (in[k]) t[0] += ds[k] * yhat[k];
          t[1] += ds[k];
        }
        at.template sum<2>(t, shared);
        const float c0 = t[0] * a.inv, c1 = a.layer ? t[1] * a.inv : 0.f;
#pragma unroll
        for (int k = 0; k < kPer; k++) ds[k] = (ds[k] - yhat[k] * c0 - c1) * rstd;
      }
      if (a.dy) at.write(a.dy, row, a.dys, on, ds);
    }
  }
  if (!a.sums) return;
  float* out = a.sums + (ll)blockIdx.x * kSums * a.D;
#pragma unroll
  for (int q = 0; q < kSums; q++) {
    if (!BLOCK && q < kPreW) continue;
    if (!BIAS && (q == kPostB || q == kPreB)) continue;
    if constexpr (R::kGroups > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kPer; k++) join[k * 256 + threadIdx.x] = sum[q][k];
      __syncthreads();
      if (at.group == 0)
#pragma unroll
        for (int k = 0; k < kPer; k++) {
          float t = 0.f;
          for (int g = 0; g < R::kGroups; g++) t += join[k * 256 + g * TPR + at.lane];
          sum[q][k] = t;
        }
    }
    if (at.group == 0)
#pragma unroll
      for (int k = 0; k < kPer; k++)
        if (at.has(k)) out[q * a.D + at.at[k / R::N].c + k % R::N] = sum[q][k];
  }
}

// ---- longer rows: streams over the row -------------------------------------------------------
// Sum over a workgroup of 256 threads, in every thread; `shared` in turns of two halves as above.
struct Block256 {
  int turn = 0;
  __device__ __forceinline__ float sum(float v, float (*shared)[4]) {
    v = lane_sum<64>(v);
    float* const s = shared[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
  }
};

// Mean and squared distance from it of the elements a thread has met, piece by piece (the pieces' own means are
// merged, so a row far from 0 loses nothing), then over the workgroup around the row's mean. rms: plain squares.
struct Moments {
  float n = 0.f, mean = 0.f, m2 = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N], unsigned mask, int layer) {
    if (!layer) {
#pragma unroll
      for (int j = 0; j < N; j++)
        if (mask >> j & 1u) m2 += v[j] * v[j];
      return;
    }
    if (!mask) return;
    const float k = (float)__popc(mask), inv = __builtin_amdgcn_rcpf(k);
    float m = 0.f, q = 0.f;
#pragma unroll
    for (int j = 0; j < N; j++) m += mask >> j & 1u ? v[j] : 0.f;
    m *= inv;
#pragma unroll
    for (int j = 0; j < N; j++) q += mask >> j & 1u ? (v[j] - m) * (v[j] - m) : 0.f;
    const float share = k * __builtin_amdgcn_rcpf(n + k), d = m - mean;
    m2 += q + d * d * n * share;
    mean += d * share;
    n += k;
  }
  __device__ __forceinline__ void finish(const Args& a, Block256& b, float (*shared)[4], float& row_mean, float& rstd) const {
    row_mean = 0.f;
    float t = m2;
    if (a.layer) {
      row_mean = b.sum(n * mean, shared) * a.inv;
      t += n * (mean - row_mean) * (mean - row_mean);
    }
    rstd = __builtin_amdgcn_rsqf(__builtin_fmaf(b.sum(t, shared), a.inv, a.eps));
  }
};

// f(piece, slot) over a row's slots by a workgroup of 256; the row's end, where it is no whole piece, in a call of its
// own, so that the others need no masks (2,048 x 8,192 bfloat16, forward: 63 us, 78 with them). One piece at a time:
// the waves are many (backward's row sums, 2,047 x 4,097 floats: 31 us, 33 by twos, 42 by fours).
template <class T, int N, class F>
__device__ __forceinline__ void over_row(int D, F f) {
  const int whole = D / N;
#pragma unroll 1
  for (int p = threadIdx.x; p < whole; p += 256) f(Piece<T, N, kWhole>(p, D), p);
  if (D % N && (int)threadIdx.x == whole % 256) f(Piece<T, N, kTail>(whole, D), whole);
}

// One workgroup a row, three passes over it: the statistics of y; s, which is written, and its statistics; n. The
// float32 s waits in shared memory for the last pass (KEEP, up to 8,192 columns, each thread's own), or is formed once
// more: n is not taken from the rounded s. 2,047 x 4,097 floats: 55 us, 3.0 TB/s; every row waits twice for its sums.
template <class T, bool KEEP>
__global__ __launch_bounds__(256) void resnorm_stream(const Args a) {
  constexpr int N = 16 / (int)sizeof(T);
  __shared__ float shared[2][4];
  extern __shared__ float kept[];  // slot by slot: (N, slots)
  if (a.ctr_out && a.row0 + blockIdx.x == 0 && threadIdx.x == 0) *a.ctr_out = a.drop.ctr ? *a.drop.ctr : 0;
  const ll row = a.row0 + blockIdx.x;
  const bool block = a.y != nullptr;
  const unsigned long long base = a.drop.thr ? drop_base(a.drop) : 0;
  const int slots = (a.D + N - 1) / N;
  Block256 b;
  float mean = 0.f, rstd = 1.f, pre_mean = 0.f, pre_rstd = 1.f;
  if (block && a.post) {
    Moments m;
    over_row<T, N>(a.D, [&](const auto& at, int) {
      const auto y = at.read(a.y, row, a.ys);
      float v[N];
#pragma unroll
      for (int j = 0; j < N; j++) v[j] = (float)y.v[j];
      m.add(v, at.mask, a.layer);
    });
    m.finish(a, b, shared, mean, rstd);
  }
  auto form = [&](const auto& at, float (&s)[N]) {
    const auto r = at.read(a.r, row, a.rs);
#pragma unroll
    for (int j = 0; j < N; j++) s[j] = (float)r.v[j];
    if (!block) return;
    const auto y = at.read(a.y, row, a.ys);
    Pack<T, N> g{};
    if (a.gate) g = at.read(a.gate, row, a.gs);
    float p[N], av[N], slope[N], w[N], bias[N];
#pragma unroll
    for (int j = 0; j < N; j++) p[j] = (float)y.v[j];
    if (a.post) {
      at.weights(a.post_w, a.w32, 1.f, w);
      at.weights(a.post_b, a.w32, 0.f, bias);
#pragma unroll
      for (int j = 0; j < N; j++) p[j] = __builtin_fmaf((p[j] - mean) * rstd, w[j], bias[j]);
    }
    if (a.drop.thr) {
      const unsigned keep = at.template keep_bits<false>(base, a.drop, row, a.D);
#pragma unroll
      for (int j = 0; j < N; j++) p[j] = (keep >> j & 1u) ? p[j] * a.drop.scale : 0.f;
    }
    activate<T, false>(g.v, a, av, slope);
    at.scales(a, w);
#pragma unroll
    for (int j = 0; j < N; j++) s[j] = __builtin_fmaf(w[j], av[j] * p[j], s[j]);
  };
  Moments m;
  if (block || a.pre) {
    over_row<T, N>(a.D, [&](const auto& at, int p) {
      float s[N];
      form(at, s);
      if (block) at.write(a.s, row, a.ss, s);
      m.add(s, at.mask, a.layer);
      if (KEEP) {
#pragma unroll
        for (int j = 0; j < N; j++) kept[j * slots + p] = s[j];
      }
    });
  }
  if (a.pre) {
    m.finish(a, b, shared, pre_mean, pre_rstd);
    over_row<T, N>(a.D, [&](const auto& at, int p) {
      float s[N], w[N], bias[N];
      if (KEEP) {
#pragma unroll
        for (int j = 0; j < N; j++) s[j] = kept[j * slots + p];
      } else {
        form(at, s);
      }
      at.weights(a.pre_w, a.w32, 1.f, w);
      at.weights(a.pre_b, a.w32, 0.f, bias);
#pragma unroll
      for (int j = 0; j < N; j++) s[j] = __builtin_fmaf((s[j] - pre_mean) * pre_rstd, w[j], bias[j]);
      at.write(a.n, row, a.ns, s);
    });
  }
  if (a.stats && threadIdx.x == 0) store<float, 4>(a.stats + row * 4, {mean, rstd, pre_mean, pre_rstd});
}

// Backward, two streams: the first takes a row's sums, the second, whose threads own columns and walk the rows, forms
// the gradients and the columns' sums (held in registers instead, 2,047 x 4,097 floats took 170 us, these 100).
//
// The norm of y needs sums over ds, the gradient of s, which itself has the row's sums c0, c1 in it. It is linear
// in them, ds = X - rstd (hat c0 + c1) with X = ds_in + rstd dn w, so the first stream takes the sums of X q, hat q
// and q (q = the factor from ds to the gradient of the normalised y, once times yhat, once alone) in the same pass.
// 4 elements a thread, whatever the type: 8 of a 16-bit type cost the registers of half the waves (2,048 x 8,192
// bfloat16: 104 us, then 72 as 4).
constexpr int kBack = 4;
template <class T>
struct Raw {
  Pack<T, kBack> y, r, g, ds, dn;
  template <bool BLOCK, class P>
  __device__ __forceinline__ void fetch(const Args& a, const P& at, ll row) {
    if (BLOCK) {
      y = at.read(a.y, row, a.ys);
      if (a.gate) g = at.read(a.gate, row, a.gs);
    }
    if (a.dn) {
      r = at.read(a.r, row, a.rs);
      dn = at.read(a.dn, row, a.dns);
    }
    if (a.ds) ds = at.read(a.ds, row, a.dss);
  }
};

// What both streams form of a row's piece before its sums are known.
template <class T, bool BLOCK, bool BIAS>
struct Formed {
  static constexpr int N = kBack;
  float ds[N], dn[N], hat[N], yhat[N], u[N], av[N], slope[N];
  unsigned keep;
  template <class P>
  __device__ __forceinline__ Formed(const Args& a, const P& at, const Raw<T>& raw, const Pack<float, 4>& st, ll row,
                                    unsigned long long base, const float (&post_w)[N], const float (&post_b)[N],
                                    const float (&scale)[N]) {
    keep = ~0u;
#pragma unroll
    for (int j = 0; j < N; j++) {
      ds[j] = a.ds ? (float)raw.ds.v[j] : 0.f;
      dn[j] = a.dn ? (float)raw.dn.v[j] : 0.f;
      hat[j] = a.dn ? (float)raw.r.v[j] : 0.f;
    }
    if (BLOCK) {
#pragma unroll
      for (int j = 0; j < N; j++) {
        yhat[j] = (float)raw.y.v[j];
        if (a.post) yhat[j] = (yhat[j] - st.v[0]) * st.v[1];
        u[j] = a.post ? (BIAS ? __builtin_fmaf(yhat[j], post_w[j], post_b[j]) : yhat[j] * post_w[j]) : yhat[j];
      }
      if (a.drop.thr) {
        keep = at.template keep_bits<false>(base, a.drop, row, a.D);
#pragma unroll
        for (int j = 0; j < N; j++) u[j] = (keep >> j & 1u) ? u[j] * a.drop.scale : 0.f;
      }
      activate<T, true>(raw.g.v, a, av, slope);
    }
    if (a.dn) {
#pragma unroll
      for (int j = 0; j < N; j++) {
        const float s = BLOCK ? __builtin_fmaf(scale[j], av[j] * u[j], hat[j]) : hat[j];
        hat[j] = at.has(j) ? (s - st.v[2]) * st.v[3] : 0.f;
      }
    }
  }
};

// One workgroup a row: (c0, c1) of the norm before, (c0, c1) of the norm of y (2,047 x 4,097 floats: 31 us, 5.4 TB/s).
template <class T, bool BLOCK, bool BIAS>
__global__ __launch_bounds__(256) void resnorm_rows(const Args a) {
  constexpr int N = kBack;
  __shared__ float shared[4][8];
  const ll row = a.row0 + blockIdx.x;
  const unsigned long long base = BLOCK && a.drop.thr ? drop_base(a.drop) : 0;
  const auto st = load<float, 4>(a.stats + row * 4);
  float t[8] = {};  // dv hat, dv, X q0, hat q0, q0, X q1, hat q1, q1
  over_row<T, N>(a.D, [&](const auto& at, int) {
    Raw<T> raw;
    raw.template fetch<BLOCK>(a, at, row);
    float pre_w[N], post_w[N], post_b[N], scale[N];
    at.weights(a.pre_w, a.w32, 1.f, pre_w);
    if (BLOCK) {
      at.weights(a.post_w, a.w32, 1.f, post_w);
      if (BIAS) at.weights(a.post_b, a.w32, 0.f, post_b);
      at.scales(a, scale);
    }
    const Formed<T, BLOCK, BIAS> f(a, at, raw, st, row, base, post_w, post_b, scale);
#pragma unroll
    for (int j = 0; j < N; j++) {
      if (!at.has(j)) continue;
      const float dv = f.dn[j] * pre_w[j];
      t[0] += dv * f.hat[j];
      t[1] += dv;
      if (BLOCK) {
        const float x = __builtin_fmaf(dv, st.v[3], f.ds[j]);
        float q = scale[j] * f.av[j] * post_w[j];
        q = (f.keep >> j & 1u) ? (a.drop.thr ? q * a.drop.scale : q) : 0.f;
        const float q0 = q * f.yhat[j];
        t[2] += x * q0;
        t[3] += f.hat[j] * q0;
        t[4] += q0;
        t[5] += x * q;
        t[6] += f.hat[j] * q;
        t[7] += q;
      }
    }
  });
#pragma unroll
  for (int k = 0; k < 8; k++) {
    t[k] = lane_sum<64>(t[k]);
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6][k] = t[k];
  }
  __syncthreads();
  if (threadIdx.x) return;
#pragma unroll
  for (int k = 0; k < 8; k++) t[k] = ((shared[0][k] + shared[1][k]) + (shared[2][k] + shared[3][k])) * a.inv;
  const float c0 = t[0], c1 = a.layer ? t[1] : 0.f;
  const float out[4] = {c0, c1, t[2] - st.v[3] * (c0 * t[3] + c1 * t[4]),
                        a.layer ? t[5] - st.v[3] * (c0 * t[6] + c1 * t[7]) : 0.f};
  store<float, 4>(a.coef + row * 4, out);
}

// A wave owns 64 slots of columns and walks rows blockIdx.y, + gridDim.y, ... (2,047 x 4,097 floats: 56 us, 4.8 TB/s).
template <class T, bool BLOCK, bool BIAS>
__global__ __launch_bounds__(64) void resnorm_columns(const Args a) {
  constexpr int N = kBack;
  const Piece<T, N, kTail> at(blockIdx.x * 64 + threadIdx.x, a.D);
  if (!at.mask) return;
  const unsigned long long base = BLOCK && a.drop.thr ? drop_base(a.drop) : 0;
  float pre_w[N], post_w[N], post_b[N], scale[N];
  at.weights(a.pre_w, a.w32, 1.f, pre_w);
  if (BLOCK) {
    at.weights(a.post_w, a.w32, 1.f, post_w);
    if (BIAS) at.weights(a.post_b, a.w32, 0.f, post_b);
    at.scales(a, scale);
  }
  float sum[kSums][N];
#pragma unroll
  for (int q = 0; q < kSums; q++)
#pragma unroll
    for (int j = 0; j < N; j++) sum[q][j] = 0.f;
  Raw<T> cur, next;
  auto st = load<float, 4>(a.stats + (ll)blockIdx.y * 4), k = load<float, 4>(a.coef + (ll)blockIdx.y * 4);
  cur.template fetch<BLOCK>(a, at, blockIdx.y);
  wait_loads();
  for (ll row = blockIdx.y; row < a.R; row += gridDim.y) {
    const ll ahead = min(row + gridDim.y, (ll)a.R - 1);  // under way while this row is worked on
    const auto next_st = load<float, 4>(a.stats + ahead * 4), next_k = load<float, 4>(a.coef + ahead * 4);
    next.template fetch<BLOCK>(a, at, ahead);
    const Formed<T, BLOCK, BIAS> f(a, at, cur, st, row, base, post_w, post_b, scale);
    float ds[N], dg[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
      ds[j] = f.ds[j];
      if (a.dn) {
        ds[j] += (f.dn[j] * pre_w[j] - f.hat[j] * k.v[0] - k.v[1]) * st.v[3];
        sum[kPreW][j] += f.dn[j] * f.hat[j];
        if (BIAS) sum[kPreB][j] += f.dn[j];
      }
    }
    if (a.dr) at.write(a.dr, row, a.drs, ds);
    if (BLOCK) {
#pragma unroll
      for (int j = 0; j < N; j++) {
        sum[kScale][j] += ds[j] * (f.av[j] * f.u[j]);
        const float dw = ds[j] * scale[j];
        dg[j] = dw * f.u[j] * f.slope[j];
        ds[j] = (f.keep >> j & 1u) ? (a.drop.thr ? dw * f.av[j] * a.drop.scale : dw * f.av[j]) : 0.f;
        if (a.post) {
          sum[kPostW][j] += ds[j] * f.yhat[j];
          if (BIAS) sum[kPostB][j] += ds[j];
          ds[j] = (ds[j] * post_w[j] - f.yhat[j] * k.v[2] - k.v[3]) * st.v[1];
        }
      }
      if (a.gate && a.dgate) at.write(a.dgate, row, a.dgs, dg);
      if (a.dy) at.write(a.dy, row, a.dys, ds);
    }
    cur = next;
    st = next_st;
    k = next_k;
  }
  if (!a.sums) return;
  float* out = a.sums + (ll)blockIdx.y * kSums * a.D;
#pragma unroll
  for (int q = 0; q < kSums; q++) {
    if (!BLOCK && q < kPreW) continue;
    if (!BIAS && (q == kPostB || q == kPreB)) continue;
#pragma unroll
    for (int j = 0; j < N; j++)
      if (at.has(j)) out[q * a.D + at.c + j] = sum[q][j];
  }
}

struct Join {
  const float* sums;
  int parts, D, w32;  // w32: outputs are float32 (else T)
  int q[kSums];       // the sums that are wanted
  void* out[kSums];
  float* scale_cols;  // the scale's column sums where one scale serves all columns (else NULL)
};

// Column sums of the workgroups' partial sums: 32 columns by 32 strands of workgroups, loads of a strand
// independent of each other (64 columns by 4 strands took 62 us for 1,024 workgroups, this 5); strands joined in
// their order.
template <class T>
__global__ __launch_bounds__(1024) void resnorm_join(const Join j) {
  __shared__ float strand[32][33];
  const int q = j.q[blockIdx.y], x = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + x;
  float t = 0.f;
  if (c < j.D) {
    const float* p = j.sums + (ll)q * j.D + c;
#pragma unroll 8
    for (int k = w; k < j.parts; k += 32) t += p[(ll)k * kSums * j.D];
  }
  strand[w][x] = t;
  __syncthreads();
  if (w || c >= j.D) return;
  t = 0.f;
#pragma unroll
  for (int k = 0; k < 32; k++) t += strand[k][x];
  if (q == kScale && j.scale_cols)
    j.scale_cols[c] = t;
  else if (j.w32)
    static_cast<float*>(j.out[q])[c] = t;
  else
    static_cast<T*>(j.out[q])[c] = (T)t;
}
template <class T>
__global__ __launch_bounds__(256) void resnorm_join_scale(const Join j) {
  __shared__ float part[256];
  float t = 0.f;
#pragma unroll 8
  for (int c = threadIdx.x; c < j.D; c += 256) t += j.scale_cols[c];
  part[threadIdx.x] = t;
  __syncthreads();
  for (int m = 128; m > 0; m >>= 1) {
    if ((int)threadIdx.x < m) part[threadIdx.x] += part[threadIdx.x + m];
    __syncthreads();
  }
  if (threadIdx.x) return;
  if (j.w32)
    *static_cast<float*>(j.out[kScale]) = part[0];
  else
    *static_cast<T*>(j.out[kScale]) = (T)part[0];
}

// ---- dropout alone ------------------------------------------------------------------
struct DropArgs {
  const void* x; ll xs;
  void* y; ll ysd;
  ll rows, cols;  // x rows of `cols` elements at stride xs (one row: flat)
  ll count;
  Drop drop;
  mjh_i64* ctr_out;
};

// A stream of 16-byte pieces, V elements each; the words of a piece are one addition apart. A word costs two 64-bit
// products, so a word for two elements keeps the arithmetic below the memory's time (at 50 million bfloat16
// elements 42 us, 4.8 TB/s, 38.5 at the least; a copy of that size runs at 5.1, an element-wise torch kernel at 5.6).
template <class T>
__global__ __launch_bounds__(256) void dropout_flat(const DropArgs a) {
  constexpr int V = 16 / (int)sizeof(T);
  const unsigned long long base = drop_base(a.drop);
  if (a.ctr_out && blockIdx.x == 0 && threadIdx.x == 0) *a.ctr_out = a.drop.ctr ? *a.drop.ctr : 0;
  for (ll i = ((ll)blockIdx.x * 256 + threadIdx.x) * V; i < a.count; i += (ll)gridDim.x * 256 * V) {
    const T* px = static_cast<const T*>(a.x) + i;
    T* py = static_cast<T*>(a.y) + i;
    unsigned long long z = base + (((unsigned long long)i >> 1) + 1ull) * 0x9e3779b97f4a7c15ull;
    if (i + V <= a.count) {
      const auto x = load_loose<T, V>(px);
      float o[V];
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const unsigned long long w = mjh::mix64(z);
        o[j] = drop_keep(w, 0, a.drop.thr) ? (float)x.v[j] * a.drop.scale : 0.f;
        o[j + 1] = drop_keep(w, 1, a.drop.thr) ? (float)x.v[j + 1] * a.drop.scale : 0.f;
        z += 0x9e3779b97f4a7c15ull;
      }
      store_loose<T, V>(py, o);
    } else {  // the last elements
      for (int j = 0; i + j < a.count; j++) {
        const unsigned long long w = mjh::mix64(z);
        py[j] = (T)(drop_keep(w, j & 1, a.drop.thr) ? (float)px[j] * a.drop.scale : 0.f);
        if (j & 1) z += 0x9e3779b97f4a7c15ull;
      }
    }
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
// lanes that hold a row (8 elements each, as slots of 16 bytes): one, a power of two up to a wave, then whole waves
int lanes_of(int D, int dtype) {
  const int n = dtype == MJH_F32 ? 4 : 8, slots = (D + n - 1) / n, lanes = (slots * n + kPer - 1) / kPer;
  if (D < n) return 1;
  if (lanes > 64) return (lanes + 63) / 64 * 64;
  int t = 8;
  while (t < lanes) t *= 2;
  return t;
}
bool long_row(int D, int dtype) { return lanes_of(D, dtype) > (dtype == MJH_F32 ? 256 : 512); }

// the backward pass's parts write partial sums each, so a part takes several rows
unsigned parts_of(int D, ll rows, int dtype) {
  if (long_row(D, dtype)) {
    const ll tiles = ((D + kBack - 1) / kBack + 63) / 64;
    return (unsigned)std::max<ll>(1, std::min<ll>(rows / 4, kColumnWaves / tiles));
  }
  const int lanes = lanes_of(D, dtype);
  const ll groups = lanes > 64 ? 1 : 256 / lanes, waves = lanes > 64 ? lanes / 64 : 4;
  return (unsigned)std::max<ll>(1, std::min<ll>((rows + groups - 1) / groups / 4, 256 * 12 / waves));
}

int check(const mjh_resnorm_desc* d) {
  if (!d) return refuse("residual norm: no description");
  if (d->R < 1 || d->D < 1) return refuse("residual norm: R and D must be positive");
  if (d->R > 0x7fffffffll) return refuse("residual norm: R must be below 2^31");
  if (d->dtype < 0 || d->dtype > 2) return refuse("residual norm: unknown type");
  if (d->D > 1 << 24) return refuse("residual norm: D is at most 2^24");
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
  a.inv = (float)(1.0 / d.D);
  a.R = (int)d.R; a.D = d.D; a.layer = d.layer; a.act = d.act; a.post = d.post; a.pre = d.pre;
  a.tpr = lanes_of(d.D, d.dtype);
  a.parts = (int)parts_of(d.D, d.R, d.dtype);
  return a;
}

bool wants_bias(const mjh_resnorm_desc& d) { return d.post_b || d.pre_b; }

// As many workgroups as are resident, each with the same number of row groups: one more round of a few workgroups, or
// one more row for some, costs what a whole round does (forward, 8,191 x 2,999 bfloat16: 116 us, 149 with 32 waves a CU
// asked for whatever their registers).
template <class K>
int waves_per_simd(K kernel) {
  int n = 0;
  return hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 256, 0) == hipSuccess && n ? n : 2;
}
ll resident(int threads, int waves_simd) { return 256ll * std::max(1, waves_simd * 256 / threads); }
template <class T, bool FULL, int TPR>
void launch_forward(const Args& a, hipStream_t s) {
  static const int waves_simd = waves_per_simd(resnorm_forward<T, FULL, TPR>);
  const int threads = TPR > 64 ? a.tpr : 256;
  const ll per = TPR > 64 ? 1 : 256 / TPR, groups = (a.R + per - 1) / per, most = resident(threads, waves_simd);
  const ll rounds = (groups + most - 1) / most, grid = (groups + rounds - 1) / rounds;
  resnorm_forward<T, FULL, TPR><<<dim3((unsigned)grid), dim3(threads), 0, s>>>(a);
}
// As many parts as are resident, where the rows are enough (98,304 x 99 floats, 2 waves a SIMD by their registers: 94
// us as 2 workgroups a CU, 119 as 3; 98,304 x 256 bfloat16, 3 waves a SIMD: 99 and 86). Each has sums to write and
// join, so a part takes 4 rows at least (parts_of(), which the workspace holds).
template <class T, bool FULL, int TPR, bool BLOCK, bool BIAS>
void launch_backward(Args& a, hipStream_t s) {
  static const int waves_simd = waves_per_simd(resnorm_backward<T, FULL, TPR, BLOCK, BIAS>);
  const int threads = TPR > 64 ? a.tpr : 256;
  a.parts = (int)std::min<ll>(a.parts, resident(threads, waves_simd));
  resnorm_backward<T, FULL, TPR, BLOCK, BIAS><<<dim3(a.parts), dim3(threads), 0, s>>>(a);
}
template <class T, bool FULL>
void launch_forward_rows(const Args& a, hipStream_t s) {
  if constexpr (!FULL)
    if (a.tpr == 1) return launch_forward<T, FULL, 1>(a, s);
  if (a.tpr == 8) return launch_forward<T, FULL, 8>(a, s);
  if (a.tpr == 16) return launch_forward<T, FULL, 16>(a, s);
  if (a.tpr == 32) return launch_forward<T, FULL, 32>(a, s);
  if (a.tpr == 64) return launch_forward<T, FULL, 64>(a, s);
  if (a.tpr <= 256) return launch_forward<T, FULL, 256>(a, s);
  if constexpr (sizeof(T) == 2 || FULL) launch_forward<T, FULL, 512>(a, s);
}
template <class T, bool FULL, bool BLOCK, bool BIAS>
void launch_backward_rows(Args& a, hipStream_t s) {
  if constexpr (!FULL)
    if (a.tpr == 1) return launch_backward<T, FULL, 1, BLOCK, BIAS>(a, s);
  if (a.tpr == 8) return launch_backward<T, FULL, 8, BLOCK, BIAS>(a, s);
  if (a.tpr == 16) return launch_backward<T, FULL, 16, BLOCK, BIAS>(a, s);
  if (a.tpr == 32) return launch_backward<T, FULL, 32, BLOCK, BIAS>(a, s);
  if (a.tpr == 64) return launch_backward<T, FULL, 64, BLOCK, BIAS>(a, s);
  if (sizeof(T) == 4 || a.tpr <= 256) return launch_backward<T, FULL, 256, BLOCK, BIAS>(a, s);
  if constexpr (sizeof(T) == 2) launch_backward<T, FULL, 512, BLOCK, BIAS>(a, s);
}
// One workgroup a row, in launches whose threads stay below 2^32 (a loop over rows in the kernels cost a tenth).
template <class F>
void by_row(Args a, F launch_rows) {
  constexpr ll most = 1 << 23;
  for (; a.row0 < a.R; a.row0 += most) launch_rows(a, (unsigned)std::min<ll>(most, a.R - a.row0));
}
template <class T, bool BLOCK, bool BIAS>
void launch_backward_as(Args& a, bool streams, hipStream_t s) {
  if (streams) {
    by_row(a, [&](const Args& b, unsigned rows) { resnorm_rows<T, BLOCK, BIAS><<<dim3(rows), dim3(256), 0, s>>>(b); });
    resnorm_columns<T, BLOCK, BIAS><<<dim3(((a.D + kBack - 1) / kBack + 63) / 64, a.parts), dim3(64), 0, s>>>(a);
  } else if (a.tpr * kPer == a.D) {
    launch_backward_rows<T, true, BLOCK, BIAS>(a, s);
  } else {
    launch_backward_rows<T, false, BLOCK, BIAS>(a, s);
  }
}
template <class T>
void launch_type(const mjh_resnorm_desc& d, Args& a, bool back, hipStream_t s) {
  const bool streams = long_row(d.D, d.dtype), bias = wants_bias(d);
  if (back && a.y)
    bias ? launch_backward_as<T, true, true>(a, streams, s) : launch_backward_as<T, true, false>(a, streams, s);
  else if (back)
    bias ? launch_backward_as<T, false, true>(a, streams, s) : launch_backward_as<T, false, false>(a, streams, s);
  else if (streams && a.tpr <= 512 && a.tpr * kPer == a.D)
    launch_forward_rows<T, true>(a, s);
  else if (streams && a.D <= 8192)
    by_row(a, [&](const Args& b, unsigned rows) {
      resnorm_stream<T, true><<<dim3(rows), dim3(256), a.D * 4 + 64, s>>>(b);
    });
  else if (streams)
    by_row(a, [&](const Args& b, unsigned rows) { resnorm_stream<T, false><<<dim3(rows), dim3(256), 0, s>>>(b); });
  else
    a.tpr * kPer == a.D ? launch_forward_rows<T, true>(a, s) : launch_forward_rows<T, false>(a, s);
}
void launch(const mjh_resnorm_desc& d, Args& a, bool back, hipStream_t s) {
  if (d.dtype == MJH_F32)
    launch_type<float>(d, a, back, s);
  else if (d.dtype == MJH_BF16)
    launch_type<bf16>(d, a, back, s);
  else
    launch_type<f16>(d, a, back, s);
}

template <class T>
void launch_join(const Join& j, int wanted, hipStream_t s) {
  resnorm_join<T><<<dim3((j.D + 31) / 32, wanted), dim3(1024), 0, s>>>(j);
  if (j.scale_cols && j.out[kScale]) resnorm_join_scale<T><<<dim3(1), dim3(256), 0, s>>>(j);
}

template <class T>
void launch_dropout(const DropArgs& a, hipStream_t s) {
  const ll most = 256 * 32, per = a.rows == 1 ? 256 * 16 / (ll)sizeof(T) : 256;
  const dim3 grid((unsigned)std::min((a.count + per - 1) / per, most));
  if (a.rows == 1)
    dropout_flat<T><<<grid, dim3(256), 0, s>>>(a);
  else
    dropout_rows<T><<<grid, dim3(256), 0, s>>>(a);
}

}  // namespace

extern "C" {

long long mjh_resnorm_workspace(const mjh_resnorm_desc* d) {
  if (check(d)) return -1;
  // row sums of long rows (first: 16-byte aligned), partial sums, the scale's column sums
  return 4 * ((long_row(d->D, d->dtype) ? 4 * d->R : 0) + (ll)parts_of(d->D, d->R, d->dtype) * kSums * d->D + d->D);
}

int mjh_resnorm_forward(const mjh_resnorm_desc* d, void* stream) {
  if (int rc = check(d)) return rc;
  if ((d->y && !d->s) || (d->pre && !d->n) || (!d->y && !d->pre)) return refuse("residual norm forward: an output is missing");
  Args a = args_of(*d);
  launch(*d, a, false, reinterpret_cast<hipStream_t>(stream));
  return launched();
}

int mjh_resnorm_backward(const mjh_resnorm_desc* d, void* stream) {
  if (int rc = check(d)) return rc;
  if (!d->stats || (!d->ds && !d->dn) || (d->dn && !d->pre)) return refuse("residual norm backward: statistics or gradients are missing");
  const bool sums = d->d_post_w || d->d_post_b || d->d_scale || d->d_pre_w || d->d_pre_b;
  if ((sums || long_row(d->D, d->dtype)) && (!d->ws || d->ws_bytes < mjh_resnorm_workspace(d)))
    return refuse("residual norm backward: workspace too small");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Args a = args_of(*d);
  a.coef = static_cast<float*>(d->ws);
  a.sums = sums ? static_cast<float*>(d->ws) + (long_row(d->D, d->dtype) ? 4 * (ll)a.R : 0) : nullptr;
  launch(*d, a, true, s);
  if (int rc = launched()) return rc;
  if (!sums) return 0;
  Join j;
  std::memset(&j, 0, sizeof(j));
  j.sums = a.sums;
  j.parts = a.parts;
  j.D = a.D;
  j.w32 = a.w32;
  j.out[kPostW] = d->d_post_w; j.out[kPostB] = d->d_post_b; j.out[kScale] = d->d_scale;
  j.out[kPreW] = d->d_pre_w; j.out[kPreB] = d->d_pre_b;
  int wanted = 0;
  for (int q = 0; q < kSums; q++)
    if (j.out[q]) j.q[wanted++] = q;
  if (a.scale_one) j.scale_cols = a.sums + (ll)j.parts * kSums * a.D;
  if (d->dtype == MJH_F32)
    launch_join<float>(j, wanted, s);
  else if (d->dtype == MJH_BF16)
    launch_join<bf16>(j, wanted, s);
  else
    launch_join<f16>(j, wanted, s);
  return launched();
}

int mjh_dropout(const void* x, long long xs, void* y, long long ys, long long rows, long long cols, int dtype, float scale,
                unsigned long long thr, unsigned long long seed, unsigned long long key, const mjh_i64* ctr,
                mjh_i64* ctr_out, void* stream) {
  if (rows < 0 || cols < 0) return refuse("dropout: negative size");
  if (dtype < 0 || dtype > 2) return refuse("dropout: unknown type");
  if (thr > (1ull << 32)) return refuse("dropout: threshold above 2^32");
  if (rows == 0 || cols == 0) return 0;
  if (!x || !y) return refuse("dropout: x and y are needed");
  if (rows > (1ll << 62) / cols) return refuse("dropout: more than 2^62 elements");
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
