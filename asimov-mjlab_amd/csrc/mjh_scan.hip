// mjh_scan.hip — gated linear recurrence over a rollout (gfx950): forward, backward, single step.
//
// Row n, channel d, gate g = d / (D / G):
//   decay: a = gate,           h_t = a h' + x_t
//   blend: a = sigmoid(gate),  h_t = a h' + (1 - a) x_t       h' = reset[t, n] ? 0 : h_{t-1}
// Steps t >= lengths[n] leave the state, output 0 and have no gradient. Backward, from the last step on:
//   delta_t = dh_t + E_t,  E_{t-1} = reset ? 0 : a_t delta_t,  E_last = dstate,  dstate0 = E before step 0
//   dx = delta (decay), (1 - a) delta (blend);  dgate = sum over the gate's channels of
//   delta h' (decay), delta (h' - x) a (1 - a) (blend)
//
// A thread owns V neighbouring channels of one row and walks the steps; the state stays in float32 registers.
// Loads of kSteps steps are issued together. The work is a stream: its floor is the bytes of x, gate and h
// (forward) and of x, gate, dh, dx and dgate (backward). The backward pass does not read h: the forward pass
// keeps the float32 state every kSteps steps (4 / kSteps bytes an element) and the backward pass runs the
// recurrence again from it inside a block of steps, so that no gradient sees a state rounded to 16 bits and
// x, which the blend needs anyway, is not joined by a second stream.
//
// With few channels the steps are cut into chunks: one launch forms each chunk's (product of a, result from 0),
// a second joins them into the state that comes into each chunk, and the main launch starts from that.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "mjh_seq.h"

namespace mjh_seq {
thread_local const char* g_why = "";
}

namespace {
using namespace mjh_seq;

constexpr int kBlock = 256;
constexpr int kSteps = 8;  // steps per block of loads, and between kept states

struct Args {
  const void* x; ll xt, xn;
  const void* gate; ll gt, gn;
  const float* state;
  const unsigned char* reset; ll rt, rn;
  const int* lengths;
  void* h; ll ht, hn;
  float* last;
  float* kept;
  const void* dh; ll dht, dhn;
  const float* dlast;
  void* dx; ll dxt, dxn;
  void* dgate; ll dgt, dgn;
  float* dstate;
  double* agg_a; float* agg_b; unsigned char* agg_cut;  // per chunk: (N, D), (N, D), (N,)
  float* part;                                         // per-wave sums of a head wider than a wave: (T, N, G, W)
  int T, N, D, G, K;  // K = D / G channels per gate
  int dv;             // vectors per row
  int chunk, nchunk;  // steps per chunk (a multiple of kSteps), chunks
  int lanes, waves;   // heads: lanes per head inside a wave (power of two), waves per head
};

struct Where {
  int n, d, g;
  bool on;   // there are channels here
  bool row;  // heads: the head exists (a lane beside its channels may still end up with a step's sum)
};

// Channels flat over (row, vector): consecutive lanes read consecutive addresses across row ends too.
template <int V>
__device__ __forceinline__ Where flat_where(const Args& a) {
  unsigned i = blockIdx.x * kBlock + threadIdx.x;
  Where w;
  w.on = w.row = i < (unsigned)a.N * (unsigned)a.dv;
  if (!w.on) i = (unsigned)a.N * (unsigned)a.dv - 1;
  w.n = (int)(i / (unsigned)a.dv);
  w.d = (int)(i - (unsigned)w.n * (unsigned)a.dv) * V;
  w.g = a.K == 1 ? w.d : w.d / a.K;
  return w;
}

// A head's channels in neighbouring lanes of one wave (or of a.waves waves), for the sum over them.
template <int V>
__device__ __forceinline__ Where head_where(const Args& a, int& lane_in_head, int& part) {
  const unsigned lane = threadIdx.x & 63u;
  const unsigned wave = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6);
  unsigned slot;
  if (a.waves == 1) {
    slot = wave * (64u / (unsigned)a.lanes) + lane / (unsigned)a.lanes;
    lane_in_head = (int)(lane % (unsigned)a.lanes);
    part = 0;
  } else {
    slot = wave / (unsigned)a.waves;
    part = (int)(wave % (unsigned)a.waves);
    lane_in_head = (int)lane;
  }
  Where w;
  const int c = (part * 64 + lane_in_head) * V;
  w.row = slot < (unsigned)a.N * (unsigned)a.G;
  w.on = w.row && c < a.K;
  if (!w.row) slot = (unsigned)a.N * (unsigned)a.G - 1;
  w.n = (int)(slot / (unsigned)a.G);
  w.g = (int)(slot % (unsigned)a.G);
  w.d = w.g * a.K + c;
  return w;
}

template <bool BLEND>
struct Gate {
  float a, b;  // the factors of the previous state and of x
  __device__ __forceinline__ explicit Gate(float g) {
    if constexpr (BLEND) {
      const float q = sigmoid_small(g);
      a = g < 0.f ? q : 1.f - q;
      b = g < 0.f ? 1.f - q : q;
    } else {
      a = g;
      b = 1.f;
    }
  }
};

// The chunks' results become the state that comes into each chunk (forward: from the chunks before it; BACK: the
// gradient from the chunks after it), written over the chunk's own result in agg_b. A workgroup holds 32 channels
// by up to 32 groups; a group takes kJoin neighbouring chunks, all loads in flight at once (2,048 channels by 512
// chunks: 8.3 us; 16 channels by 64 groups 1 more, 8 by 64 6 more; one thread a channel and a loop over 256 chunks
// 70). A chunk with a reset inside passes nothing on, whatever comes in (not 0 times it: the state before a reset may
// be infinite or NaN), and a state of 0 adds nothing, however far the product of the gates overflows. No load stands
// in a branch, where it would be waited for (1,000 x 8 x 99 with resets: 5.0 us, twice that with its flags' loads in one).
//
// Products of gates are float64, here and in the launches that form them: a small state may grow, and a large one
// shrink, by any factor of up to 2^277 inside float32's range, over a chunk or a group of them. A product beyond
// float64's range takes every other state beyond float32's in either case: the recurrence itself overflows there
// (a product of infinity and a later 0 is its NaN too) or has nothing left. 1.6 us of the 8.3.
constexpr int kJoin = 16, kMaxChunks = 32 * kJoin;
__device__ __forceinline__ float carry(double p, float s, float q, bool cut) {
  return cut || s == 0.f ? q : (float)__builtin_fma(p, (double)s, (double)q);
}
template <bool BACK>
__global__ __launch_bounds__(1024) void scan_join(const Args a) {
  __shared__ double sa[32][32];
  __shared__ float sb[32][32];
  __shared__ unsigned char sc[32][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const ll nd = (ll)a.N * a.D, own = (ll)blockIdx.x * 32 + lane, at = min(own, nd - 1);
  const bool on = own < nd;
  const int n = (int)((unsigned)at / (unsigned)a.D);
  const float* edge = BACK ? a.dlast : a.state;
  const float first = on && edge ? edge[at] : 0.f;
  double p[kJoin];
  float q[kJoin];
  unsigned flag[kJoin], cut = 0;  // cut, bit k: a reset inside chunk k
#pragma unroll
  for (int k = 0; k < kJoin; k++) {  // chunks behind the last read the last again
    const int i = min(w * kJoin + k, a.nchunk - 1);  // in the order of the recurrence
    const ll c = BACK ? a.nchunk - 1 - i : i;
    p[k] = a.agg_a[c * nd + at];
    q[k] = a.agg_b[c * nd + at];
    flag[k] = 0;
  }
  if (a.reset) {
#pragma unroll
    for (int k = 0; k < kJoin; k++) {
      const int i = min(w * kJoin + k, a.nchunk - 1);
      flag[k] = a.agg_cut[(ll)(BACK ? a.nchunk - 1 - i : i) * a.N + n];
    }
  }
#pragma unroll
  for (int k = 0; k < kJoin; k++) {
    const bool in = w * kJoin + k < a.nchunk;
    p[k] = in ? p[k] : 1.;
    q[k] = in ? q[k] : 0.f;
    cut |= (unsigned)(in && flag[k]) << k;
  }
  double ta = 1.;
  float tb = 0.f;
#pragma unroll
  for (int k = 0; k < kJoin; k++) {
    tb = carry(p[k], tb, q[k], cut >> k & 1u);
    ta *= p[k];
  }
  sa[w][lane] = ta;
  sb[w][lane] = tb;
  sc[w][lane] = cut != 0;
  __syncthreads();
  float s = first;
#pragma unroll 8
  for (int k = 0; k < w; k++) s = carry(sa[k][lane], s, sb[k][lane], sc[k][lane]);
#pragma unroll
  for (int k = 0; k < kJoin; k++) {
    const int i = w * kJoin + k;
    if (!on || i >= a.nchunk) break;
    a.agg_b[(BACK ? a.nchunk - 1 - i : i) * nd + at] = s;
    s = carry(p[k], s, q[k], cut >> k & 1u);
  }
}

// The state (BACK: gradient) that comes into chunk c.
template <int V, bool BACK>
__device__ __forceinline__ void incoming(const Args& a, ll at, int c, float (&s)[V]) {
  const float* from = a.nchunk > 1 ? a.agg_b + c * ((ll)a.N * a.D) : BACK ? a.dlast : a.state;
#pragma unroll
  for (int v = 0; v < V; v++) s[v] = 0.f;
  if (!from) return;
  const auto p = load<float, V>(from + at);
#pragma unroll
  for (int v = 0; v < V; v++) s[v] = p.v[v];
}

// A wave's place in the (T, N) reset flags. Where its rows are at most 8 neighbours (D of 16 and more), one load
// brings the flags of kSteps steps for all of them: lane l reads step l % 8 of row l / 8, and a ballot hands every
// lane its row's bits (a load per step and lane took 8 us of the 96 us of a 24 x 4,096 x 256 training pass).
struct Flags {
  int n0;
  bool wide;
  __device__ __forceinline__ explicit Flags(const Where& w) {
    n0 = __builtin_amdgcn_readfirstlane(w.n);
    wide = __builtin_amdgcn_readlane(w.n, 63) - n0 < 8;
  }
  // called by all lanes of the wave
  __device__ __forceinline__ unsigned raw(const Args& a, const Where& w, int tb, int end) const {
    static_assert(kSteps == 8, "8 steps by 8 rows fill a wave");
    if (!a.reset) return 0;
    if (wide) {
      const int lane = threadIdx.x & 63;
      return a.reset[(ll)min(tb + (lane & 7), end - 1) * a.rt + (ll)min(n0 + (lane >> 3), a.N - 1) * a.rn];
    }
    unsigned bits = 0;
    for (int j = 0; j < kSteps; j++) bits |= (unsigned)(a.reset[(ll)min(tb + j, end - 1) * a.rt + (ll)w.n * a.rn] != 0) << j;
    return bits;
  }
  __device__ __forceinline__ unsigned bits(const Args& a, const Where& w, unsigned raw) const {
    if (!a.reset) return 0;
    return wide ? (unsigned)(__ballot(raw != 0) >> (8 * (w.n - n0))) & 255u : raw;
  }
};

// What a thread reads for kSteps steps from tb on; steps from `end` on read step end - 1 again and are not used.
// Lanes with nothing to read (`on` false) take part for the flags.
template <class T, class GT, int V, int GV, bool X, bool DH>
struct Block {
  Pack<T, V> x[kSteps], dh[kSteps];
  Pack<GT, GV> g[kSteps];
  unsigned flags;

  __device__ __forceinline__ void read(const Args& a, const Where& w, const Flags& f, bool on, int tb, int end) {
    flags = f.raw(a, w, tb, end);
    if (!on) return;
    const T* px = static_cast<const T*>(a.x) + (ll)w.n * a.xn + w.d;
    const GT* pg = static_cast<const GT*>(a.gate) + (ll)w.n * a.gn + w.g;
    const T* pd = static_cast<const T*>(a.dh) + (ll)w.n * a.dhn + w.d;
    px += tb * a.xt;
    pg += tb * a.gt;
#pragma unroll
    for (int j = 0; j < kSteps; j++) {
      if constexpr (X) x[j] = load<T, V>(px);
      g[j] = load<GT, GV>(pg);
      if (j + 1 == kSteps) break;
      if constexpr (X) px += tb + j + 1 < end ? a.xt : 0;
      pg += tb + j + 1 < end ? a.gt : 0;
    }
    if constexpr (DH) {
      if (a.dh) {
        pd += tb * a.dht;
#pragma unroll
        for (int j = 0; j < kSteps; j++) {
          dh[j] = load<T, V>(pd);
          if (j + 1 < kSteps) pd += tb + j + 1 < end ? a.dht : 0;
        }
      } else {
#pragma unroll
        for (int j = 0; j < kSteps; j++) dh[j] = Pack<T, V>{};
      }
    }
  }
};

// the largest value of the wave's lanes, the same in all
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v = max(v, __shfl_xor(v, m));
  return __builtin_amdgcn_readfirstlane(v);
}

template <int V>
__device__ __forceinline__ void store_products(double* p, const double (&f)[V]) {
  Pack<double, V> o;
#pragma unroll
  for (int v = 0; v < V; v++) o.v[v] = f[v];
  *reinterpret_cast<Pack<double, V>*>(p) = o;
}

// What a chunk's steps do to the state that comes in, h -> A h + B: A = product of a, B = the result from 0. One
// reading of x and gate (16,384 x 2,048 bfloat16: 16 us, 4.3 TB/s; 23 within a training pass, after a launch whose
// outputs are still being written out; more loads under way, or wider ones, are the same). 64 registers, so that all
// 524,288 threads are resident; 72 for two gates a thread, which spill in 64 (200 x 240 x 256 blend, backward: 15.0 us,
// 16.2 so).
template <class T, class GT, int V, int GV, bool BLEND>
__global__ __launch_bounds__(kBlock, GV == 2 ? 7 : 8) void scan_forward_agg(const Args a) {
  const Where w = flat_where<V>(a);
  const Flags flags(w);
  const int c = blockIdx.y, t0 = c * a.chunk, t1 = min(a.T, t0 + a.chunk);
  const int live = !w.on ? 0 : a.lengths ? min(a.lengths[w.n], t1) : t1;
  const int stop = a.lengths ? wave_max(live) : t1;  // the same in all lanes, as every read and ballot needs
  const ll nd = (ll)a.N * a.D, at = (ll)w.n * a.D + w.d;
  float s[V];
  double prod[V];
#pragma unroll
  for (int v = 0; v < V; v++) s[v] = 0.f, prod[v] = 1.;
  bool cut = false;
  for (int tb = t0; tb < stop; tb += kSteps) {
    Block<T, GT, V, GV, true, false> b;
    b.read(a, w, flags, tb < live, tb, t1);
    const unsigned bits = flags.bits(a, w, b.flags);
    if (__all(bits == 0 && tb + kSteps <= live)) {
#pragma unroll
      for (int j = 0; j < kSteps; j++)
#pragma unroll
        for (int v = 0; v < V; v++) {
          const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
          const float x = (float)b.x[j].v[v];
          s[v] = __builtin_fmaf(f.a, s[v], BLEND ? f.b * x : x);
          prod[v] *= (double)f.a;
        }
    } else {
#pragma unroll
      for (int j = 0; j < kSteps; j++) {
        if (tb + j >= live) continue;
        const bool reset = bits >> j & 1u;
        cut |= reset;
#pragma unroll
        for (int v = 0; v < V; v++) {
          const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
          const float x = (float)b.x[j].v[v];
          s[v] = __builtin_fmaf(f.a, reset ? 0.f : s[v], BLEND ? f.b * x : x);
          prod[v] = reset ? 0. : prod[v] * (double)f.a;
        }
      }
    }
  }
  if (!w.on) return;
  store_products(a.agg_a + c * nd + at, prod);
  store<float, V>(a.agg_b + c * nd + at, s);
  if (a.reset && w.d == 0) a.agg_cut[(ll)c * a.N + w.n] = cut;
}

// The outputs. Bound by bytes (24 x 4,096 x 256 bfloat16 with kept states: 38 us, 4.5 TB/s). AHEAD: loads of the next
// block under way while this one is worked on, for chunked launches; with a thread for every channel of many rows the
// waves that its registers cost are worth more (24 x 4,096 x 256 bfloat16 without kept states: 33 us against 40).
template <class T, class GT, int V, int GV, bool BLEND, bool AHEAD>
__global__ __launch_bounds__(kBlock) void scan_forward(const Args a) {
  const Where w = flat_where<V>(a);
  const Flags flags(w);
  const int c = blockIdx.y, t0 = c * a.chunk, t1 = min(a.T, t0 + a.chunk);
  const int live = !w.on ? 0 : a.lengths ? min(a.lengths[w.n], t1) : t1;
  const int stop = a.lengths ? wave_max(live) : t1;
  const ll nd = (ll)a.N * a.D, at = (ll)w.n * a.D + w.d;
  float s[V];
  incoming<V, false>(a, at, c, s);
  T* ph = static_cast<T*>(a.h) + (ll)w.n * a.hn + w.d;
  Block<T, GT, V, GV, true, false> b, next;
  if (AHEAD && t0 < stop) b.read(a, w, flags, t0 < live, t0, t1);
  if (AHEAD) wait_loads();
  int tb = t0;
  for (; tb < stop; tb += kSteps) {
    if (a.kept && w.on) store<float, V>(a.kept + (ll)(tb / kSteps) * nd + at, s);
    if (!AHEAD) b.read(a, w, flags, tb < live, tb, t1);
    if (AHEAD && tb + kSteps < stop) next.read(a, w, flags, tb + kSteps < live, tb + kSteps, t1);
    const unsigned bits = flags.bits(a, w, b.flags);
    if (__all(bits == 0 && tb + kSteps <= live)) {
#pragma unroll
      for (int j = 0; j < kSteps; j++) {
#pragma unroll
        for (int v = 0; v < V; v++) {
          const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
          const float x = (float)b.x[j].v[v];
          s[v] = __builtin_fmaf(f.a, s[v], BLEND ? f.b * x : x);
        }
        store<T, V>(ph + (ll)(tb + j) * a.ht, s);
      }
    } else {  // a reset, a row's end or the last step inside
#pragma unroll
      for (int j = 0; j < kSteps; j++) {
        float out[V];
#pragma unroll
        for (int v = 0; v < V; v++) {
          out[v] = 0.f;
          if (tb + j < live) {
            const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
            const float x = (float)b.x[j].v[v];
            out[v] = s[v] = __builtin_fmaf(f.a, bits >> j & 1u ? 0.f : s[v], BLEND ? f.b * x : x);
          }
        }
        if (w.on && tb + j < t1) store<T, V>(ph + (ll)(tb + j) * a.ht, out);
      }
    }
    if (AHEAD) b = next;
  }
  if (!w.on) return;
  for (; tb < t1; tb += kSteps) {  // beyond the rows' lengths: nothing to read
    if (a.kept) store<float, V>(a.kept + (ll)(tb / kSteps) * nd + at, s);
    const float none[V] = {};
#pragma unroll
    for (int j = 0; j < kSteps; j++)
      if (tb + j < t1) store<T, V>(ph + (ll)(tb + j) * a.ht, none);
  }
  if (c == a.nchunk - 1) store<float, V>(a.last + at, s);
}

// The chunk's effect on the gradient that comes in from the steps after it.
template <class T, class GT, int V, int GV, bool BLEND>
__global__ __launch_bounds__(kBlock, GV == 2 ? 7 : 8) void scan_backward_agg(const Args a) {
  const Where w = flat_where<V>(a);
  const Flags flags(w);
  const int c = blockIdx.y, t0 = c * a.chunk, t1 = min(a.T, t0 + a.chunk);
  const int live = !w.on ? 0 : a.lengths ? min(a.lengths[w.n], t1) : t1;
  const int stop = a.lengths ? wave_max(live) : t1;
  const ll nd = (ll)a.N * a.D, at = (ll)w.n * a.D + w.d;
  float e[V];
  double prod[V];
#pragma unroll
  for (int v = 0; v < V; v++) e[v] = 0.f, prod[v] = 1.;
  bool cut = false;
  for (int tb = t0 + (max(stop - t0, 0) + kSteps - 1) / kSteps * kSteps - kSteps; tb >= t0; tb -= kSteps) {
    Block<T, GT, V, GV, false, true> b;
    b.read(a, w, flags, tb < live, tb, t1);
    const unsigned bits = flags.bits(a, w, b.flags);
    if (__all(bits == 0 && tb + kSteps <= live)) {
#pragma unroll
      for (int j = kSteps - 1; j >= 0; j--)
#pragma unroll
        for (int v = 0; v < V; v++) {
          const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
          e[v] = f.a * ((float)b.dh[j].v[v] + e[v]);
          prod[v] *= (double)f.a;
        }
    } else {
#pragma unroll
      for (int j = kSteps - 1; j >= 0; j--) {
        if (tb + j >= live) continue;
        const bool reset = bits >> j & 1u;
        cut |= reset;
#pragma unroll
        for (int v = 0; v < V; v++) {
          const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
          e[v] = reset ? 0.f : f.a * ((float)b.dh[j].v[v] + e[v]);
          prod[v] = reset ? 0. : prod[v] * (double)f.a;
        }
      }
    }
  }
  if (!w.on) return;
  store_products(a.agg_a + c * nd + at, prod);
  store<float, V>(a.agg_b + c * nd + at, e);
  if (a.reset && w.d == 0) a.agg_cut[(ll)c * a.N + w.n] = cut;
}

// kSteps values summed over groups of `lanes` lanes (a power of two). While a lane holds several steps it hands
// half of them to its partner and takes the other half's terms (4 + 2 + 1 exchanges for 8 steps where summing each
// step by itself takes 8 at every level). Returns the first step this lane ends with; `count` steps are left in
// v[0..], the same in the lanes that differ in the bits of `same` only. A fixed order: no run differs from another.
__device__ __forceinline__ int sum_over_lanes(float (&v)[kSteps], int lane, int lanes, int& count, int& same) {
  int m = lanes >> 1, base = 0;
  count = kSteps;
#pragma unroll
  for (int n = kSteps; n > 1; n /= 2) {
    if (m > 0) {
      const bool up = lane & m;
#pragma unroll
      for (int i = 0; i < n / 2; i++) {
        const float send = up ? v[i] : v[i + n / 2], mine = up ? v[i + n / 2] : v[i];
        v[i] = mine + __shfl_xor(send, m);
      }
      base += up ? n / 2 : 0;
      count = n / 2;
      m >>= 1;
    }
  }
  same = m ? 2 * m - 1 : 0;
  for (; m > 0; m >>= 1) v[0] += __shfl_xor(v[0], m);
  return base;
}

// The gradients, steps in blocks from the last on: the states of a block forward from the kept one, then its steps
// backward. Bound by bytes at the 3 waves a SIMD that its registers leave (24 x 4,096 x 256 bfloat16: 59 us, 4.6 TB/s).
// HEADS: dgate is summed over a head's lanes; lanes beside its channels take part with 0.
template <class T, class GT, int V, int GV, bool BLEND, bool HEADS>
__global__ __launch_bounds__(kBlock) void scan_backward(const Args a) {
  int lane = 0, part = 0;
  const Where w = HEADS ? head_where<V>(a, lane, part) : flat_where<V>(a);
  const Flags flags(w);
  const bool on = w.on;
  const int c = blockIdx.y, t0 = c * a.chunk, t1 = min(a.T, t0 + a.chunk);
  const ll nd = (ll)a.N * a.D, at = (ll)w.n * a.D + w.d;
  const int live = !on ? 0 : a.lengths ? min(a.lengths[w.n], t1) : t1;
  const int stop = a.lengths ? wave_max(live) : t1;
  float e[V];
#pragma unroll
  for (int v = 0; v < V; v++) e[v] = 0.f;
  if (on) incoming<V, true>(a, at, c, e);
  T* px = static_cast<T*>(a.dx) + (ll)w.n * a.dxn + w.d;
  GT* pg = static_cast<GT*>(a.dgate) + (ll)w.n * a.dgn + w.g;
  const int last = t0 + (t1 - 1 - t0) / kSteps * kSteps;
  Block<T, GT, V, GV, true, true> b, next;
  Pack<float, V> k, nextk;
  auto fetch = [&](Block<T, GT, V, GV, true, true>& to, Pack<float, V>& tok, int tb) {
    if (tb < t0 || tb >= stop) return;  // beyond the rows' lengths: nothing to read
    to.read(a, w, flags, tb < live, tb, t1);
    if (tb < live) tok = load<float, V>(a.kept + (ll)(tb / kSteps) * nd + at);
  };
  fetch(b, k, last);
  wait_loads();
  for (int tb = last; tb >= t0; tb -= kSteps) {
    fetch(next, nextk, tb - kSteps);  // under way while this block is worked on
    float sum[kSteps];
    const unsigned bits = tb < stop ? flags.bits(a, w, b.flags) : 0u;
    if (__all(bits == 0 && tb + kSteps <= live)) {
      // the states before each step, forward from the kept one; then the steps backward
      float fa[kSteps][GV], fb[kSteps][GV], before[kSteps][V], s[V];
#pragma unroll
      for (int v = 0; v < V; v++) s[v] = k.v[v];
#pragma unroll
      for (int j = 0; j < kSteps; j++) {
#pragma unroll
        for (int v = 0; v < GV; v++) {
          const Gate<BLEND> f((float)b.g[j].v[v]);
          fa[j][v] = f.a;
          fb[j][v] = f.b;
        }
#pragma unroll
        for (int v = 0; v < V; v++) {
          const float x = (float)b.x[j].v[v];
          before[j][v] = s[v];
          s[v] = __builtin_fmaf(fa[j][GV == 1 ? 0 : v], s[v], BLEND ? fb[j][GV == 1 ? 0 : v] * x : x);
        }
      }
#pragma unroll
      for (int j = kSteps - 1; j >= 0; j--) {
        float dx[V], dg[V];
        sum[j] = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++) {
          const float ga = fa[j][GV == 1 ? 0 : v], gb = fb[j][GV == 1 ? 0 : v];
          const float delta = (float)b.dh[j].v[v] + e[v];
          dx[v] = BLEND ? gb * delta : delta;
          dg[v] = BLEND ? dx[v] * ga * (before[j][v] - (float)b.x[j].v[v]) : delta * before[j][v];
          e[v] = ga * delta;
          sum[j] += dg[v];
        }
        if (a.dx) store<T, V>(px + (ll)(tb + j) * a.dxt, dx);
        if constexpr (!HEADS)
          if (a.dgate) store<GT, V>(pg + (ll)(tb + j) * a.dgt, dg);
      }
    } else {  // a reset, a row's end, the last step, or lanes beside a head's channels
      float s[V], before[kSteps][V];
#pragma unroll
      for (int v = 0; v < V; v++) s[v] = k.v[v];
#pragma unroll
      for (int j = 0; j < kSteps; j++) {
        if (tb + j >= live) continue;
#pragma unroll
        for (int v = 0; v < V; v++) {
          const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
          const float x = (float)b.x[j].v[v];
          before[j][v] = bits >> j & 1u ? 0.f : s[v];
          s[v] = __builtin_fmaf(f.a, before[j][v], BLEND ? f.b * x : x);
        }
      }
#pragma unroll
      for (int j = kSteps - 1; j >= 0; j--) {
        float dx[V], dg[V];
        sum[j] = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++) {
          dx[v] = dg[v] = 0.f;
          if (tb + j < live) {
            const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
            const float delta = (float)b.dh[j].v[v] + e[v];
            dx[v] = BLEND ? f.b * delta : delta;
            dg[v] = BLEND ? dx[v] * f.a * (before[j][v] - (float)b.x[j].v[v]) : delta * before[j][v];
            e[v] = bits >> j & 1u ? 0.f : f.a * delta;
          }
          sum[j] += dg[v];
        }
        if (on && tb + j < t1) {
          if (a.dx) store<T, V>(px + (ll)(tb + j) * a.dxt, dx);
          if constexpr (!HEADS)
            if (a.dgate) store<GT, V>(pg + (ll)(tb + j) * a.dgt, dg);
        }
      }
    }
    b = next;
    k = nextk;
    if constexpr (HEADS) {
      if (a.dgate) {
        int count, same;
        const int first = sum_over_lanes(sum, lane, a.lanes, count, same);
        if (w.row && !(lane & same)) {
#pragma unroll
          for (int i = 0; i < kSteps; i++) {
            const int t = tb + first + i;
            if (i < count && t < t1) {
              if (a.waves == 1)
                pg[(ll)t * a.dgt] = (GT)sum[i];
              else
                a.part[(((ll)t * a.N + w.n) * a.G + w.g) * a.waves + part] = sum[i];
            }
          }
        }
      }
    }
  }
  if (c == 0 && a.dstate && on) store<float, V>(a.dstate + at, e);
}

// dgate of heads wider than a wave: the waves' sums, in their order.
template <class GT>
__global__ __launch_bounds__(kBlock) void scan_join_heads(const Args a) {
  const ll i = (ll)blockIdx.x * kBlock + threadIdx.x;
  if (i >= (ll)a.T * a.N * a.G) return;
  float sum = 0.f;
  for (int k = 0; k < a.waves; k++) sum += a.part[i * a.waves + k];
  const int g = (int)(i % a.G);
  const ll tn = i / a.G;
  static_cast<GT*>(a.dgate)[(tn / a.N) * a.dgt + (tn % a.N) * a.dgn + g] = (GT)sum;
}

// One step: out = a h' + ..., the state read from a.state and written to a.last (the same rows, or others). 4,096 x 256
// bfloat16: 4.6 us, 3.2 TB/s; 1 x 128: 1.8 us.
template <class T, class GT, int V, int GV, bool BLEND>
__global__ __launch_bounds__(kBlock) void scan_step(const Args a) {
  const Where w = flat_where<V>(a);
  if (!w.on) return;
  const ll at = (ll)w.n * a.D + w.d;
  const auto x = load<T, V>(static_cast<const T*>(a.x) + (ll)w.n * a.xn + w.d);
  const auto g = load<GT, GV>(static_cast<const GT*>(a.gate) + (ll)w.n * a.gn + w.g);
  const auto s = load<float, V>(a.state + at);
  const bool r = a.reset && a.reset[(ll)w.n * a.rn];
  float out[V];
#pragma unroll
  for (int v = 0; v < V; v++) {
    const Gate<BLEND> f((float)g.v[GV == 1 ? 0 : v]);
    const float add = BLEND ? f.b * (float)x.v[v] : (float)x.v[v];
    out[v] = r ? add : __builtin_fmaf(f.a, s.v[v], add);
  }
  store<float, V>(a.last + at, out);
  store<T, V>(static_cast<T*>(a.h) + (ll)w.n * a.hn + w.d, out);
}

// ---- host side ------------------------------------------------------------------
enum Kernel { kForward, kForwardAgg, kBackward, kBackwardAgg, kStep };

struct Plan {
  Args a;
  bool heads;            // gates shared by channels
  int v;                 // channels per thread of the launch at hand
  unsigned blocks;       // flat mapping
  unsigned head_blocks;  // head mapping
};

// Channels per thread: the launch's geometry.
void set_width(Plan& p, int v) {
  Args& a = p.a;
  p.v = v;
  a.dv = a.D / v;
  p.blocks = (unsigned)(((ll)a.N * a.dv + kBlock - 1) / kBlock);
  const int per = (a.K + v - 1) / v;  // lanes a head needs
  a.lanes = 1;
  while (a.lanes < per && a.lanes < 64) a.lanes *= 2;
  a.waves = (per + 63) / 64;
  const ll slots = (ll)a.N * a.G;
  const ll waves = a.waves == 1 ? (slots + 64 / a.lanes - 1) / (64 / a.lanes) : slots * a.waves;
  p.head_blocks = (unsigned)((waves + 3) / 4);
}

size_t type_size(int t) { return t == MJH_F32 ? 4 : 2; }

// V channels per thread need every row, step and pointer aligned to them.
bool fits(const mjh_scan_desc& s, int v) {
  const int k = s.D / s.G;
  if (s.D % v || (k > 1 && k % v)) return false;
  const size_t eb = type_size(s.dtype) * v, gb = type_size(s.gtype) * v;
  const ll st[] = {s.xt, s.xn, s.ht, s.hn, s.dht, s.dhn, s.dxt, s.dxn};
  for (ll q : st)
    if (q % v) return false;
  for (const void* p : {s.x, (const void*)s.h, s.dh, (const void*)s.dx})
    if (!aligned(p, eb)) return false;
  if (k == 1) {
    for (ll q : {s.gt, s.gn, s.dgt, s.dgn})
      if (q % v) return false;
    if (!aligned(s.gate, gb) || !aligned(s.dgate, gb)) return false;
  }
  for (const void* p : {(const void*)s.state, (const void*)s.last, (const void*)s.kept, (const void*)s.dlast, (const void*)s.dstate})
    if (!aligned(p, 4 * (size_t)v)) return false;
  return true;
}

// Two neighbouring channels a thread where strides allow (16,384 x 2,048 bfloat16, shared gates: 133 us of kernels
// against 153 with one; 24 x 8,192 x 512: 367, 388), but for gates of their own in 65,536 to 131,072 channels, which one
// channel a thread makes enough threads for a launch without chunks (200 x 480 x 256: 134 us, 148 in chunks).
//
// Chunks: from kFull threads on none (24 x 4,096 x 256: 99 us). Below, enough for kThreads threads, of kLeast blocks of
// steps each (16,384 x 2,048: 133 us, 138 for half as many threads, 132 for twice; 4,001 x 12 x 512: 47, 50, 47), or of
// one block while that makes no more than kFew threads (1,000 x 8 x 99: 30 us, 38 without; for all, 200 x 240 x 256: 99
// against 93).
constexpr int kWide = 2;
constexpr ll kThreads = 524288, kFull = 65536, kLeast = 2, kFew = 262144;

int make_plan(const mjh_scan_desc* s, Plan& p) {
  if (!s) return refuse("scan: no description");
  if (s->T < 1 || s->N < 1 || s->D < 1 || s->G < 1) return refuse("scan: T, N, D and G must be positive");
  if (s->D % s->G) return refuse("scan: G must divide D");
  if ((ll)s->N * s->D > 0x7fffffffll || s->T > 1 << 30) return refuse("scan: N * D must be below 2^31, T at most 2^30");
  if (s->dtype < 0 || s->dtype > 2 || (s->gtype != s->dtype && s->gtype != MJH_F32))
    return refuse("scan: the gate must have x's type or float32");
  if (s->mode != MJH_SCAN_DECAY && s->mode != MJH_SCAN_BLEND) return refuse("scan: unknown mode");
  Args& a = p.a;
  std::memset(&a, 0, sizeof(a));
  a.x = s->x; a.xt = s->xt; a.xn = s->xn;
  a.gate = s->gate; a.gt = s->gt; a.gn = s->gn;
  a.state = s->state;
  a.reset = s->reset; a.rt = s->rt; a.rn = s->rn;
  a.lengths = s->lengths;
  a.h = s->h; a.ht = s->ht; a.hn = s->hn;
  a.last = s->last; a.kept = s->kept;
  a.dh = s->dh; a.dht = s->dht; a.dhn = s->dhn;
  a.dlast = s->dlast;
  a.dx = s->dx; a.dxt = s->dxt; a.dxn = s->dxn;
  a.dgate = s->dgate; a.dgt = s->dgt; a.dgn = s->dgn;
  a.dstate = s->dstate;
  a.T = s->T; a.N = s->N; a.D = s->D; a.G = s->G; a.K = s->D / s->G;
  p.heads = a.K > 1;
  const ll channels = (ll)a.N * a.D;
  set_width(p, fits(*s, kWide) && (p.heads || channels < kFull || channels >= kWide * kFull) ? kWide : 1);
  const ll threads = (ll)a.N * a.dv;
  const ll blocks = (a.T + kSteps - 1) / kSteps;
  ll n = 1;
  if (threads < kFull) {
    n = std::max(std::min((kThreads + threads - 1) / threads, blocks / kLeast), std::min(kFew / threads, blocks));
    n = std::max<ll>(1, std::min<ll>(n, kMaxChunks));
  }
  const ll per_chunk = (blocks + n - 1) / n;
  a.chunk = (int)(per_chunk * kSteps);
  a.nchunk = (int)((a.T + a.chunk - 1) / a.chunk);
  return 0;
}

ll agg_floats(const Plan& p) {
  const Args& a = p.a;
  if (a.nchunk == 1) return 0;
  const ll nd = (ll)a.N * a.D;
  return 3 * a.nchunk * nd + ((ll)a.nchunk * a.N + 3) / 4;
}
ll part_floats(const Plan& p) {
  const Args& a = p.a;
  return p.heads && a.waves > 1 ? (ll)a.T * a.N * a.G * a.waves : 0;
}
void place(Plan& p, float* ws) {
  Args& a = p.a;
  const ll nd = (ll)a.N * a.D;
  a.agg_a = reinterpret_cast<double*>(ws);
  a.agg_b = ws + 2 * a.nchunk * nd;
  a.agg_cut = reinterpret_cast<unsigned char*>(ws + 3 * a.nchunk * nd);
  a.part = ws + agg_floats(p);
}

template <class T, class GT, int V, int GV, bool BLEND>
void launch_as(Kernel k, const Plan& p, hipStream_t s) {
  const Args& a = p.a;
  const dim3 grid(p.blocks, a.nchunk), block(kBlock);
  switch (k) {
    case kForward:
      if (a.nchunk > 1)
        scan_forward<T, GT, V, GV, BLEND, true><<<grid, block, 0, s>>>(a);
      else
        scan_forward<T, GT, V, GV, BLEND, false><<<grid, block, 0, s>>>(a);
      break;
    case kForwardAgg:
      scan_forward_agg<T, GT, V, GV, BLEND><<<grid, block, 0, s>>>(a);
      scan_join<false><<<dim3((unsigned)(((ll)a.N * a.D + 31) / 32)), dim3(32 * ((a.nchunk + kJoin - 1) / kJoin)), 0, s>>>(a);
      break;
    case kBackwardAgg:
      scan_backward_agg<T, GT, V, GV, BLEND><<<grid, block, 0, s>>>(a);
      scan_join<true><<<dim3((unsigned)(((ll)a.N * a.D + 31) / 32)), dim3(32 * ((a.nchunk + kJoin - 1) / kJoin)), 0, s>>>(a);
      break;
    case kBackward:
      if (!p.heads) {
        scan_backward<T, GT, V, V, BLEND, false><<<grid, block, 0, s>>>(a);
        break;
      }
      scan_backward<T, GT, V, 1, BLEND, true><<<dim3(p.head_blocks, a.nchunk), block, 0, s>>>(a);
      if (a.waves > 1 && a.dgate) {
        const ll n = (ll)a.T * a.N * a.G;
        scan_join_heads<GT><<<dim3((unsigned)((n + kBlock - 1) / kBlock)), block, 0, s>>>(a);
      }
      break;
    case kStep:
      scan_step<T, GT, V, GV, BLEND><<<dim3(p.blocks), block, 0, s>>>(a);
      break;
  }
}
template <class T, class GT>
void launch_typed(Kernel k, const Plan& p, int mode, hipStream_t s) {
  auto go = [&](auto blend) {
    constexpr bool B = decltype(blend)::value;
    if (p.v == 1)
      launch_as<T, GT, 1, 1, B>(k, p, s);
    else if (p.heads)
      launch_as<T, GT, kWide, 1, B>(k, p, s);
    else
      launch_as<T, GT, kWide, kWide, B>(k, p, s);
  };
  if (mode == MJH_SCAN_BLEND)
    go(std::true_type{});
  else
    go(std::false_type{});
}
int launch(Kernel k, const Plan& p, const mjh_scan_desc& d, void* stream) {
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool g32 = d.gtype == MJH_F32;
  if (d.dtype == MJH_F32)
    launch_typed<float, float>(k, p, d.mode, s);
  else if (d.dtype == MJH_BF16)
    g32 ? launch_typed<bf16, float>(k, p, d.mode, s) : launch_typed<bf16, bf16>(k, p, d.mode, s);
  else
    g32 ? launch_typed<f16, float>(k, p, d.mode, s) : launch_typed<f16, f16>(k, p, d.mode, s);
  return launched();
}

}  // namespace

extern "C" {

const char* mjh_seq_last_error(void) { return g_why; }

size_t mjh_sizeof_scan_desc(void) { return sizeof(mjh_scan_desc); }
size_t mjh_sizeof_resnorm_desc(void) { return sizeof(mjh_resnorm_desc); }

int mjh_scan_steps(void) { return kSteps; }

long long mjh_scan_workspace(const mjh_scan_desc* d, int back) {
  Plan p;
  if (make_plan(d, p)) return -1;
  return 4 * (agg_floats(p) + (back ? part_floats(p) : 0));
}

int mjh_scan_forward(const mjh_scan_desc* d, void* stream) {
  Plan p;
  if (int rc = make_plan(d, p)) return rc;
  if (!d->x || !d->gate || !d->h || !d->last) return refuse("scan forward: x, gate, h and last are needed");
  if (d->ws_bytes < 4 * agg_floats(p) || (agg_floats(p) && !d->ws)) return refuse("scan forward: workspace too small");
  if (agg_floats(p) && !aligned(d->ws, 16)) return refuse("scan forward: the workspace must be aligned to 16 bytes");
  place(p, static_cast<float*>(d->ws));
  if (p.a.nchunk > 1)
    if (int rc = launch(kForwardAgg, p, *d, stream)) return rc;
  return launch(kForward, p, *d, stream);
}

int mjh_scan_backward(const mjh_scan_desc* d, void* stream) {
  Plan p;
  if (int rc = make_plan(d, p)) return rc;
  if (!d->x || !d->gate || !d->kept) return refuse("scan backward: x, gate and the kept states are needed");
  const ll need = agg_floats(p) + part_floats(p);
  if (d->ws_bytes < 4 * need || (need && !d->ws)) return refuse("scan backward: workspace too small");
  if (need && !aligned(d->ws, 16)) return refuse("scan backward: the workspace must be aligned to 16 bytes");
  place(p, static_cast<float*>(d->ws));
  if (p.a.nchunk > 1)
    if (int rc = launch(kBackwardAgg, p, *d, stream)) return rc;
  return launch(kBackward, p, *d, stream);
}

int mjh_scan_step(const mjh_scan_desc* d, void* stream) {
  Plan p;
  if (int rc = make_plan(d, p)) return rc;
  if (d->T != 1) return refuse("scan step: T must be 1");
  if (!d->x || !d->gate || !d->h || !d->last || !d->state) return refuse("scan step: x, gate, state, h and last are needed");
  return launch(kStep, p, *d, stream);
}

}  // extern "C"
