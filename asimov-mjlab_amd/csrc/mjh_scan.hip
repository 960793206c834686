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
// and the main launch joins those of the chunks before its own.
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
  float* agg_a; float* agg_b; unsigned char* agg_cut;  // per chunk: (N, D), (N, D), (N,)
  float* part;                                         // per-wave sums of a head wider than a wave: (T, N, G, W)
  int T, N, D, G, K;  // K = D / G channels per gate
  int dv;             // vectors per row
  int chunk, nchunk;  // steps per chunk (a multiple of kSteps), chunks
  int lanes, waves;   // heads: lanes per head inside a wave (power of two), waves per head
};

struct Where {
  int n, d, g;
  bool on;
};

// Channels flat over (row, vector): consecutive lanes read consecutive addresses across row ends too.
template <int V>
__device__ __forceinline__ Where flat_where(const Args& a) {
  const unsigned i = blockIdx.x * kBlock + threadIdx.x;
  Where w;
  w.on = i < (unsigned)a.N * (unsigned)a.dv;
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
  w.on = slot < (unsigned)a.N * (unsigned)a.G && c < a.K;
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

// The float32 state before chunk c (forward: from the first chunk on; backward: gradient after chunk c, from
// the last on). A chunk with a reset inside passes nothing on, whatever comes in (not 0 times it: the state
// before a reset may be infinite or NaN).
template <int V, bool BACK>
__device__ __forceinline__ void join_chunks(const Args& a, const Where& w, int c, float (&s)[V]) {
  const ll nd = (ll)a.N * a.D, at = (ll)w.n * a.D + w.d;
  for (int k = BACK ? a.nchunk - 1 : 0; BACK ? k > c : k < c; BACK ? k-- : k++) {
    const auto p = load<float, V>(a.agg_a + k * nd + at);
    const auto q = load<float, V>(a.agg_b + k * nd + at);
    const bool cut = a.reset && a.agg_cut[(ll)k * a.N + w.n];
#pragma unroll
    for (int v = 0; v < V; v++) s[v] = cut ? q.v[v] : __builtin_fmaf(p.v[v], s[v], q.v[v]);
  }
}

template <class T, class GT, int V, int GV>
struct Block {
  Pack<T, V> x[kSteps];
  Pack<GT, GV> g[kSteps];
  unsigned char r[kSteps];

  // steps tb .. tb + kSteps; those from `end` on read step end - 1 again and are not used
  template <bool WITH_X>
  __device__ __forceinline__ void read(const Args& a, const Where& w, int tb, int end) {
    const T* px = static_cast<const T*>(a.x) + (ll)w.n * a.xn + w.d;
    const GT* pg = static_cast<const GT*>(a.gate) + (ll)w.n * a.gn + w.g;
#pragma unroll
    for (int j = 0; j < kSteps; j++) {
      const ll t = min(tb + j, end - 1);
      if constexpr (WITH_X) x[j] = load<T, V>(px + t * a.xt);
      g[j] = load<GT, GV>(pg + t * a.gt);
      r[j] = 0;
    }
    if (a.reset) {
      const unsigned char* pr = a.reset + (ll)w.n * a.rn;
#pragma unroll
      for (int j = 0; j < kSteps; j++) r[j] = pr[(ll)min(tb + j, end - 1) * a.rt];
    }
  }
};

// AGG: the chunk's (product of a, result from state 0); else the outputs.
template <class T, class GT, int V, int GV, bool BLEND, bool AGG>
__global__ __launch_bounds__(kBlock) void scan_forward(const Args a) {
  const Where w = flat_where<V>(a);
  if (!w.on) return;
  const int c = blockIdx.y, t0 = c * a.chunk, t1 = min(a.T, t0 + a.chunk);
  const int live = a.lengths ? min(a.lengths[w.n], t1) : t1;
  const ll nd = (ll)a.N * a.D, at = (ll)w.n * a.D + w.d;
  float s[V], prod[V];
#pragma unroll
  for (int v = 0; v < V; v++) s[v] = 0.f, prod[v] = 1.f;
  bool cut = false;
  if (!AGG) {
    if (a.state) {
      const auto p = load<float, V>(a.state + at);
#pragma unroll
      for (int v = 0; v < V; v++) s[v] = p.v[v];
    }
    join_chunks<V, false>(a, w, c, s);
  }
  T* ph = static_cast<T*>(a.h) + (ll)w.n * a.hn + w.d;
  for (int tb = t0; tb < t1; tb += kSteps) {
    Block<T, GT, V, GV> b;
    b.template read<true>(a, w, tb, t1);
    if (!AGG && a.kept) store<float, V>(a.kept + (ll)(tb / kSteps) * nd + at, s);
#pragma unroll
    for (int j = 0; j < kSteps; j++) {
      const int t = tb + j;
      if (t >= t1) break;
      const bool in = t < live;
      float out[V];
#pragma unroll
      for (int v = 0; v < V; v++) {
        const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
        const float x = (float)b.x[j].v[v];
        const float add = BLEND ? f.b * x : x;
        const float next = b.r[j] ? add : __builtin_fmaf(f.a, s[v], add);
        if (AGG) prod[v] = in ? (b.r[j] ? 0.f : prod[v] * f.a) : prod[v];
        s[v] = in ? next : s[v];
        out[v] = in ? next : 0.f;
      }
      if (AGG) cut |= in && b.r[j];
      if (!AGG) store<T, V>(ph + (ll)t * a.ht, out);
    }
  }
  if (AGG) {
    store<float, V>(a.agg_a + c * nd + at, prod);
    store<float, V>(a.agg_b + c * nd + at, s);
    if (a.reset && w.d == 0) a.agg_cut[(ll)c * a.N + w.n] = cut;
  } else if (c == a.nchunk - 1) {
    store<float, V>(a.last + at, s);
  }
}

// The chunk's effect on the gradient that comes in from the steps after it.
template <class T, class GT, int V, int GV, bool BLEND>
__global__ __launch_bounds__(kBlock) void scan_backward_agg(const Args a) {
  const Where w = flat_where<V>(a);
  if (!w.on) return;
  const int c = blockIdx.y, t0 = c * a.chunk, t1 = min(a.T, t0 + a.chunk);
  const int live = a.lengths ? min(a.lengths[w.n], t1) : t1;
  const ll nd = (ll)a.N * a.D, at = (ll)w.n * a.D + w.d;
  const T* pd = static_cast<const T*>(a.dh) + (ll)w.n * a.dhn + w.d;
  float e[V], prod[V];
#pragma unroll
  for (int v = 0; v < V; v++) e[v] = 0.f, prod[v] = 1.f;
  bool cut = false;
  for (int tb = t0 + (t1 - 1 - t0) / kSteps * kSteps; tb >= t0; tb -= kSteps) {
    Block<T, GT, V, GV> b;
    b.template read<false>(a, w, tb, t1);
    Pack<T, V> dh[kSteps];
#pragma unroll
    for (int j = 0; j < kSteps; j++) {
      if (a.dh)
        dh[j] = load<T, V>(pd + (ll)min(tb + j, t1 - 1) * a.dht);
      else
        dh[j] = Pack<T, V>{};
    }
#pragma unroll
    for (int j = kSteps - 1; j >= 0; j--) {
      const int t = tb + j;
      if (t >= live) continue;
#pragma unroll
      for (int v = 0; v < V; v++) {
        const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
        e[v] = b.r[j] ? 0.f : f.a * ((float)dh[j].v[v] + e[v]);
        prod[v] = b.r[j] ? 0.f : prod[v] * f.a;
      }
      cut |= b.r[j] != 0;
    }
  }
  store<float, V>(a.agg_a + c * nd + at, prod);
  store<float, V>(a.agg_b + c * nd + at, e);
  if (a.reset && w.d == 0) a.agg_cut[(ll)c * a.N + w.n] = cut;
}

// HEADS: dgate is summed over a head's lanes (a butterfly: a fixed order).
template <class T, class GT, int V, int GV, bool BLEND, bool HEADS>
__global__ __launch_bounds__(kBlock) void scan_backward(const Args a) {
  int lane = 0, part = 0;
  const Where w = HEADS ? head_where<V>(a, lane, part) : flat_where<V>(a);
  if (!HEADS && !w.on) return;
  const bool on = w.on;  // lanes beside a head's channels take part in its sums with 0
  const int c = blockIdx.y, t0 = c * a.chunk, t1 = min(a.T, t0 + a.chunk);
  const ll nd = (ll)a.N * a.D, at = (ll)w.n * a.D + w.d;
  const int live = !on ? 0 : a.lengths ? min(a.lengths[w.n], t1) : t1;
  float e[V];
#pragma unroll
  for (int v = 0; v < V; v++) e[v] = 0.f;
  if (on) {
    if (a.dlast) {
      const auto p = load<float, V>(a.dlast + at);
#pragma unroll
      for (int v = 0; v < V; v++) e[v] = p.v[v];
    }
    join_chunks<V, true>(a, w, c, e);
  }
  const T* pd = static_cast<const T*>(a.dh) + (ll)w.n * a.dhn + w.d;
  T* px = static_cast<T*>(a.dx) + (ll)w.n * a.dxn + w.d;
  GT* pg = static_cast<GT*>(a.dgate) + (ll)w.n * a.dgn + w.g;
  for (int tb = t0 + (t1 - 1 - t0) / kSteps * kSteps; tb >= t0; tb -= kSteps) {
    Block<T, GT, V, GV> b;
    Pack<T, V> dh[kSteps];
    float before[kSteps][V];
    if (on) {
      b.template read<true>(a, w, tb, t1);
      const auto k = load<float, V>(a.kept + (ll)(tb / kSteps) * nd + at);
#pragma unroll
      for (int j = 0; j < kSteps; j++) {
        if (a.dh)
          dh[j] = load<T, V>(pd + (ll)min(tb + j, t1 - 1) * a.dht);
        else
          dh[j] = Pack<T, V>{};
      }
      float s[V];
#pragma unroll
      for (int v = 0; v < V; v++) s[v] = k.v[v];
#pragma unroll
      for (int j = 0; j < kSteps; j++) {
#pragma unroll
        for (int v = 0; v < V; v++) {
          const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
          const float x = (float)b.x[j].v[v];
          before[j][v] = b.r[j] ? 0.f : s[v];
          s[v] = b.r[j] ? f.b * x : __builtin_fmaf(f.a, s[v], f.b * x);
        }
      }
    }
#pragma unroll
    for (int j = kSteps - 1; j >= 0; j--) {
      const int t = tb + j;
      if (t >= t1) continue;
      const bool in = t < live;
      float dx[V], dg[V], sum = 0.f;
#pragma unroll
      for (int v = 0; v < V; v++) {
        dx[v] = dg[v] = 0.f;
        if (in) {
          const Gate<BLEND> f((float)b.g[j].v[GV == 1 ? 0 : v]);
          const float delta = (float)dh[j].v[v] + e[v];
          if (BLEND) {
            dx[v] = f.b * delta;
            dg[v] = dx[v] * f.a * (before[j][v] - (float)b.x[j].v[v]);
          } else {
            dx[v] = delta;
            dg[v] = delta * before[j][v];
          }
          e[v] = b.r[j] ? 0.f : f.a * delta;
        }
        sum += dg[v];
      }
      if (a.dx && on) store<T, V>(px + (ll)t * a.dxt, dx);
      if (a.dgate) {
        if constexpr (HEADS) {
          for (int m = a.lanes >> 1; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
          if (on && lane == 0) {
            if (a.waves == 1)
              pg[(ll)t * a.dgt] = (GT)sum;
            else
              a.part[(((ll)t * a.N + w.n) * a.G + w.g) * a.waves + part] = sum;
          }
        } else {
          store<GT, V>(pg + (ll)t * a.dgt, dg);
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

// One step: out = a h' + ..., the state read from a.state and written to a.last (the same rows, or others).
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
  int v;         // channels per thread
  bool heads;    // gates shared by channels
  unsigned blocks;       // flat mapping
  unsigned head_blocks;  // head mapping
};

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

int make_plan(const mjh_scan_desc* s, bool back, Plan& p) {
  if (!s) return refuse("scan: no description");
  if (s->T < 1 || s->N < 1 || s->D < 1 || s->G < 1) return refuse("scan: T, N, D and G must be positive");
  if (s->D % s->G) return refuse("scan: G must divide D");
  if ((ll)s->N * s->D > 0x7fffffffll) return refuse("scan: N * D must be below 2^31");
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
  const int wide = s->dtype == MJH_F32 ? 2 : 4;
  p.v = fits(*s, wide) ? wide : 1;
  a.dv = a.D / p.v;
  const ll threads = (ll)a.N * a.dv;
  p.blocks = (unsigned)((threads + kBlock - 1) / kBlock);
  const int per = (a.K + p.v - 1) / p.v;  // lanes a head needs
  a.lanes = 1;
  while (a.lanes < per && a.lanes < 64) a.lanes *= 2;
  a.waves = (per + 63) / 64;
  const ll slots = (ll)a.N * a.G;
  const ll waves = a.waves == 1 ? (slots + 64 / a.lanes - 1) / (64 / a.lanes) : slots * a.waves;
  p.head_blocks = (unsigned)((waves + 3) / 4);
  // chunks: enough threads to keep the card's loads in flight, each chunk some blocks of steps long
  const ll want = 131072;
  ll n = threads >= want ? 1 : (want + threads - 1) / threads;
  const ll blocks = (a.T + kSteps - 1) / kSteps;
  n = std::max<ll>(1, std::min<ll>(n, blocks / 4));
  n = std::min<ll>(n, 256);
  const ll per_chunk = (blocks + n - 1) / n;
  a.chunk = (int)(per_chunk * kSteps);
  a.nchunk = (int)((a.T + a.chunk - 1) / a.chunk);
  (void)back;
  return 0;
}

ll agg_floats(const Plan& p) {
  const Args& a = p.a;
  if (a.nchunk == 1) return 0;
  const ll nd = (ll)a.N * a.D;
  return 2 * a.nchunk * nd + ((ll)a.nchunk * a.N + 3) / 4;
}
ll part_floats(const Plan& p) {
  const Args& a = p.a;
  return p.heads && a.waves > 1 ? (ll)a.T * a.N * a.G * a.waves : 0;
}
void place(Plan& p, float* ws) {
  Args& a = p.a;
  const ll nd = (ll)a.N * a.D;
  a.agg_a = ws;
  a.agg_b = ws + a.nchunk * nd;
  a.agg_cut = reinterpret_cast<unsigned char*>(ws + 2 * a.nchunk * nd);
  a.part = ws + agg_floats(p);
}

template <class T, class GT, int V, int GV, bool BLEND>
void launch_as(Kernel k, const Plan& p, hipStream_t s) {
  const Args& a = p.a;
  const dim3 grid(p.blocks, a.nchunk), block(kBlock);
  switch (k) {
    case kForward:
      scan_forward<T, GT, V, GV, BLEND, false><<<grid, block, 0, s>>>(a);
      break;
    case kForwardAgg:
      scan_forward<T, GT, V, GV, BLEND, true><<<grid, block, 0, s>>>(a);
      break;
    case kBackwardAgg:
      scan_backward_agg<T, GT, V, GV, BLEND><<<grid, block, 0, s>>>(a);
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
template <class T, class GT, int WIDE>
void launch_typed(Kernel k, const Plan& p, int mode, hipStream_t s) {
  auto go = [&](auto blend) {
    constexpr bool B = decltype(blend)::value;
    if (p.v == 1)
      launch_as<T, GT, 1, 1, B>(k, p, s);
    else if (p.heads)
      launch_as<T, GT, WIDE, 1, B>(k, p, s);
    else
      launch_as<T, GT, WIDE, WIDE, B>(k, p, s);
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
    launch_typed<float, float, 2>(k, p, d.mode, s);
  else if (d.dtype == MJH_BF16)
    g32 ? launch_typed<bf16, float, 4>(k, p, d.mode, s) : launch_typed<bf16, bf16, 4>(k, p, d.mode, s);
  else
    g32 ? launch_typed<f16, float, 4>(k, p, d.mode, s) : launch_typed<f16, f16, 4>(k, p, d.mode, s);
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
  if (make_plan(d, back != 0, p)) return -1;
  return 4 * (agg_floats(p) + (back ? part_floats(p) : 0));
}

int mjh_scan_forward(const mjh_scan_desc* d, void* stream) {
  Plan p;
  if (int rc = make_plan(d, false, p)) return rc;
  if (!d->x || !d->gate || !d->h || !d->last) return refuse("scan forward: x, gate, h and last are needed");
  if (d->ws_bytes < 4 * agg_floats(p) || (agg_floats(p) && !d->ws)) return refuse("scan forward: workspace too small");
  place(p, static_cast<float*>(d->ws));
  if (p.a.nchunk > 1)
    if (int rc = launch(kForwardAgg, p, *d, stream)) return rc;
  return launch(kForward, p, *d, stream);
}

int mjh_scan_backward(const mjh_scan_desc* d, void* stream) {
  Plan p;
  if (int rc = make_plan(d, true, p)) return rc;
  if (!d->x || !d->gate || !d->kept) return refuse("scan backward: x, gate and the kept states are needed");
  const ll need = agg_floats(p) + part_floats(p);
  if (d->ws_bytes < 4 * need || (need && !d->ws)) return refuse("scan backward: workspace too small");
  place(p, static_cast<float*>(d->ws));
  if (p.a.nchunk > 1)
    if (int rc = launch(kBackwardAgg, p, *d, stream)) return rc;
  return launch(kBackward, p, *d, stream);
}

int mjh_scan_step(const mjh_scan_desc* d, void* stream) {
  Plan p;
  if (int rc = make_plan(d, false, p)) return rc;
  if (d->T != 1) return refuse("scan step: T must be 1");
  if (!d->x || !d->gate || !d->h || !d->last || !d->state) return refuse("scan step: x, gate, state, h and last are needed");
  return launch(kStep, p, *d, stream);
}

}  // extern "C"
