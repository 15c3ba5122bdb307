// The gated linear recurrence along the time axis of a recording,
//
//   h_t = keep_t h_{t-1} + b_t,      constant gate: keep = c, b = x;   value: keep = g_t, b = x_t;
//                                    logit: f = sigmoid(g_t), keep = f, b = (1 - f) x_t;     a reset at t: keep = 0
//
// and its backward pass, which is the same recurrence walked the other way over d_t = dh_t + keep_{t+1} d_{t+1}:
//   value: dx = d, dg = d h_{t-1};   logit: dx = (1 - f) d, dg = d f (1 - f) (h_{t-1} - x_t).
//
// Steps compose: (A, B) after (A', B') is (A A', A B' + B), so the time axis can be cut into chunks whose composites are joined by a scan.
// A keep of exactly zero DROPS the state it would multiply - whatever that holds, infinities and NaN too - in every path, so the result does
// not depend on where the axis was cut.  Carries, composites and sums are float32 for every element type; one rounding, at the store.
//
// What bounds it: memory.  Forward reads x and g and writes h (12 B per float32 element); backward reads x, g, dh and writes dx, dg (20 B):
// the states it needs are RECOMPUTED in registers from x and g, piece by piece - a chunk of a column, a tile of a row - from the state in front of the
// piece.  That is the stored one where states are float32; of 16-bit states the forward pass leaves the ones that the backward pass starts from in
// float32 as well (`edges`: a float every 4 to 16 steps of a column, every 512 of a row), so that their rounding stays out of dg = d f (1 - f) (h - x),
// which is a small difference wherever a state follows its input (inputs 1 + 0.05 noise, bfloat16, 200 steps: dg off by 0.0017, one rounding; started
// from rounded states by 0.0096).
//
// Two layouts, each with one element of time per register so that no shared-memory transpose is needed:
//   columns  a batch axis is contiguous (time-major recordings, (B, T, C) activations): lanes lie across the batch, one float32 or two 16-bit
//            columns each.  A thread walks K steps at a time, all their loads in flight; it is alone with its columns, or the time axis is cut into
//            chunks over the threads of a workgroup (LDS joins them) and, where even that leaves the chip empty, into segments over workgroups
//            (a first launch writes their composites).  Very many columns are walked forwards four or eight (16 bytes) to a thread.
//   rows     time is contiguous: lanes lie along time, eight steps each, and a group of 2^n lanes scans by wave shuffles; segments as above
//
// Measured, against 5.15 TB/s of a copy of 839 MB and 8.6 of one that stays in the last cache (128 MB):
//   columns, 200 steps x 65536                  float32   logit     forward 30.3 us (5.2 TB/s)   backward 56.1 us (4.7 TB/s)
//                                                         value     forward 29.3 us (5.4 TB/s)   backward 53.0 us (4.9 TB/s)
//                                                         constant  forward 21.4 us (4.9 TB/s)   backward 21.8 us (4.8 TB/s)
//                                               bfloat16  logit     forward 33.3 us (2.4 TB/s; 29.5 without edges)   backward 47.0 us (2.8 TB/s)
//                                                         value     forward 26.5 us (3.0 TB/s; 23.9 without edges)   backward 42.1 us (3.1 TB/s)
//                                                         constant  forward 22.9 us (2.3 TB/s)   backward 23.1 us (2.3 TB/s)
//                                               16 bits are bound by vector instructions and by what they do not hide: logit form forward 12.6 M of a wave,
//                                               20.5 us at four cycles each, and the loads of a tile that are asked for behind the join of the tile before
//   columns, 200 x 2^20, constant gate          float32   336 us (5.0 TB/s): a copy's rate
//   columns, 65536 x 64, logit form             float32   forward 10.9 + 14.7 us, backward 13.2 + 24.7 us, two launches each: 2.0 and 2.2 TB/s, bound by
//                                               latency - the segments' composites are a second walk over x and g that has to end first
//   rows, 65536 x 200 steps                     float32   logit     forward 35.8 us (4.4 TB/s)   backward 81.0 us (3.2 TB/s)
//                                                         value     forward 30.9 us (5.1 TB/s)   backward 64.8 us (4.0 TB/s)
//                                                         constant  forward 28.3 us (3.7 TB/s)   backward 30.7 us (3.4 TB/s)
//                                               bfloat16  logit     forward 34.2 us (2.3 TB/s)   backward 71.5 us (1.8 TB/s)
//                                                         value     forward 28.8 us (2.7 TB/s)   backward 54.2 us (2.4 TB/s)
//                                               bound by the instructions of the scans (logit form: 30 of 36 us forward, 50 of 81 backward) and the registers of
//                                               the backward pass.  (The scan by DPP moves instead of shuffles: slower, it spills.)
//   rows, 1665 x 1001, value gates              float32   forward 9.0 us, backward 14.2 us (2.2 and 2.3 TB/s)
#pragma once
#include "learning_common.hpp"

namespace mbt_learning {

constexpr int kGateConstant = MBT_GATE_CONSTANT, kGateValue = MBT_GATE_VALUE, kGateLogit = MBT_GATE_LOGIT;

constexpr int kMostSteps = 16;  // steps of a chunk that one thread holds in registers

struct Axis {  // one operand: address at the first step in walking order, element strides (time signed: reversed walks go down)
  void* p;
  int64_t so, st, si;
};

struct RecurrenceParams {
  Axis x, g, reset, h, dh, dx, dg;
  const float* initial;   // (outer, inner) or null
  float* final_state;     // (outer, inner) or null
  const float* dfinal;    // (outer, inner) or null
  float* dinitial;        // (outer, inner) or null
  float2* composites;     // [segment][column] (columns) / [row][segment] (rows)
  float* edges;           // [steps to the end >> edge_log2, less one](outer, inner) states in float32, or null
  int64_t steps, outer, inner;
  int64_t vectors_per_outer, vectors;  // column vectors (V columns each)
  int64_t segment;                     // steps per segment
  int32_t segments;
  int32_t lanes_log2;     // columns: column vectors per workgroup; rows: lanes per row
  int32_t whole_blocks;   // columns: no workgroup has lanes behind the last column
  int32_t edge_log2;
  int32_t batch_swapped;  // initial / final are (outer, inner) of the CALLER: 1 when the kernel's axes are exchanged
  int64_t column_blocks;
  // the constant gate as a float32 pair (0.99 is not a float32 number, and its error would be made at every step), and the powers of the
  // double that a chunk of n steps composes to; neither is zero unless the double is
  float constant, constant_rest;
  float power[kMostSteps + 1];
};

struct Composite {
  float a, b;
};
__device__ __forceinline__ float apply_step(float keep, float h, float b) { return keep == 0.0f ? b : __builtin_fmaf(keep, h, b); }
// The product of gates that are not zero must not underflow to the zero that means "dropped": it stays the smallest number, of its own sign (an
// infinity that it meets changes sign with it).
__device__ __forceinline__ float not_dropped(float a) { return a == 0.0f ? __builtin_copysignf(1.4e-45f, a) : a; }
// first, then second.  A state is the composite (0, h).
__device__ __forceinline__ Composite then(Composite first, Composite second) {
  float a = first.a * second.a;
  if (first.a != 0.0f && second.a != 0.0f) a = not_dropped(a);
  return {a, apply_step(second.a, first.b, second.b)};
}
// one step of the walk.  ENTERING: the backward pass's first, where d = grad_final comes in with a factor of one, not with the constant and its rest
template <int FORM>
__device__ __forceinline__ float advance(const RecurrenceParams& P, float keep, float h, float b, bool entering = false) {
  if (FORM != kGateConstant) return apply_step(keep, h, b);
  // (an infinite state is one times the constant; times its rest, which may be zero or of the other sign, it would turn into a NaN)
  const float finite = __builtin_amdgcn_fmed3f(h, -3.40282347e38f, 3.40282347e38f);
  return keep == 0.0f ? b : __builtin_fmaf(keep, h, __builtin_fmaf(entering ? 0.0f : P.constant_rest, finite, b));
}

// f = sigmoid(k) and 1 - f, each to about an ulp: e = exp(-|k|) with the rounding of the exponent's product carried along, r = 1 / (1 + e) by one
// Newton step on the hardware reciprocal.  A NaN stays a NaN.
__device__ __forceinline__ void sigmoid_pair(float k, float& f, float& i) {
  const float m = __builtin_fabsf(k);
  const float c = m > 110.0f ? 110.0f : m;  // exp(-110) is below the smallest float32
  const float t = -c * 1.44269502f;
  const float lo = __builtin_fmaf(-c, 1.44269502f, -t) - c * 1.92596303e-8f;
  const float e = __builtin_amdgcn_exp2f(t) * __builtin_fmaf(lo, 0.693147182f, 1.0f);
  const float d = 1.0f + e;
  float r = __builtin_amdgcn_rcpf(d);
  r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
  const float q = e * r;
  f = k >= 0.0f ? r : q;
  i = k >= 0.0f ? q : r;
}

// what multiplies the state (unless a reset drops it) and what multiplies the input; g is turned in place into the former
template <int FORM>
__device__ __forceinline__ void gate(const RecurrenceParams& P, float& g, float& inject) {
  inject = 1.0f;
  if (FORM == kGateConstant) g = P.constant;
  if (FORM == kGateLogit) {
    float f;
    sigmoid_pair(g, f, inject);
    g = f;
  }
}

// Steps of a chunk, held in registers: 16 elements of each array, so that a thread stays within the 128 registers of four waves per SIMD - the
// backward pass, where it holds four arrays at once, takes half of that.  (Rewards-to-go of 2^20 x 200 with 16, 32 and 64 elements: 332, 346, 380 us.)
constexpr int chunk_steps(int form, bool backward, int v, bool alone) {
  return (backward && (form == kGateLogit || (alone && form == kGateValue)) ? 8 : 16) / v;
}

// ---- columns -----------------------------------------------------------------------------------------------------------------------
// MODE: whole time axis in one thread (kAlone), cut over the threads of the workgroup (kJoined; after kComposites when there are segments).
enum : int { kAlone = 0, kJoined = 1, kComposites = 2 };
constexpr int kStreamed = 1;  // + kColumnsWide: past the caches

template <typename E, int V, bool STREAM>
struct Column {
  int64_t o, i;  // (the V columns of a thread are all there: the host takes V = 1 where V does not divide the axis)

  // address at step s; the next step's is t.st further (walked, not recomputed: an address per step and array would not fit the registers)
  __device__ __forceinline__ E* at(const Axis& t, int64_t s) const { return static_cast<E*>(t.p) + o * t.so + s * t.st + i * t.si; }
  __device__ __forceinline__ static void load(const E* p, float (&out)[V]) {
    Pack<E, V> v;
    if constexpr (STREAM) v = stream_load_pack<E, V>(p);
    else v = load_pack<E, V>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = static_cast<float>(v.e[j]);
  }
  __device__ __forceinline__ static void store(E* p, const float (&in)[V]) {
    Pack<E, V> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.e[j] = static_cast<E>(in[j]);
    if constexpr (STREAM) stream_store_pack<E, V>(p, v);
    else store_pack<E, V>(p, v);
  }
  __device__ __forceinline__ bool flag(const Axis& t, int64_t s, int j) const {
    return static_cast<const uint8_t*>(t.p)[o * t.so + s * t.st + (i + j) * t.si] != 0;
  }
  // (outer, inner) float32 of the caller
  __device__ __forceinline__ int64_t batch(const RecurrenceParams& P, int j) const {
    return P.batch_swapped ? (i + j) * P.outer + o : o * P.inner + i + j;
  }
  __device__ __forceinline__ void load_batch(const RecurrenceParams& P, const float* p, float (&out)[V]) const {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = p != nullptr ? p[batch(P, j)] : 0.0f;
  }
  // the edge with `left` steps behind it, a multiple of how far they lie apart
  __device__ __forceinline__ float* edge(const RecurrenceParams& P, int64_t left) const {
    return P.edges + ((left >> P.edge_log2) - 1) * (P.outer * P.inner) + batch(P, 0);
  }
  __device__ __forceinline__ void load_edge(const RecurrenceParams& P, int64_t left, float (&out)[V]) const {
    const float* p = edge(P, left);
    const int64_t next = P.batch_swapped ? P.outer : 1;
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = p[j * next];
  }
  __device__ __forceinline__ void store_edge(const RecurrenceParams& P, int64_t left, const float (&in)[V]) const {
    float* p = edge(P, left);
    const int64_t next = P.batch_swapped ? P.outer : 1;
#pragma unroll
    for (int j = 0; j < V; ++j) p[j * next] = in[j];
  }
};

// Joins the composites of a workgroup's chunks, thread order = walking order for each column: on return `mine` is everything BEFORE this thread's
// chunk, the carry included, and the carry has moved behind the last chunk if `more` is to come.  Within a wave by shuffles over its chunks
// (lane = chunk * C + column with C = 2^lanes_log2 columns), across waves through LDS: a wave folds only the waves in front of it, the last one
// folds the carry on.
template <int V>
__device__ __forceinline__ void join_chunks(Composite (&mine)[V], Composite (&carry)[V], bool more, int lanes_log2, float2* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int columns = 1 << lanes_log2, column = lane & (columns - 1);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    for (int d = columns; d < 64; d <<= 1) {
      const Composite before = {__shfl_up(mine[j].a, d), __shfl_up(mine[j].b, d)};
      if (lane >= d) mine[j] = then(before, mine[j]);
    }
    if (lane >= 64 - columns) lds[((wave + 1) * V + j) * columns + column] = make_float2(mine[j].a, mine[j].b);
    const Composite before = {__shfl_up(mine[j].a, columns & 63), __shfl_up(mine[j].b, columns & 63)};
    mine[j] = lane >= columns ? before : Composite{1.0f, 0.0f};
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) {
    Composite front = carry[j];
    for (int w = 0; w < wave; w += 4) {  // (four reads at a time: one after the other, each would wait for the one before it)
      float2 c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = lds[((w + i < wave ? w + i + 1 : 1) * V + j) * columns + column];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (w + i < wave) front = then(front, {c[i].x, c[i].y});
    }
    mine[j] = then(front, mine[j]);
    if (more && wave == waves - 1 && lane >= 64 - columns) {
      const float2 c = lds[(waves * V + j) * columns + column];
      const Composite all = then(front, {c.x, c.y});
      lds[j * columns + column] = make_float2(all.a, all.b);
    }
  }
  if (more) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 c = lds[j * columns + column];
      carry[j] = {c.x, c.y};
    }
  }
}

// The K steps of one chunk in registers: loaded, joined with the other chunks of the workgroup, walked, stored.  FULL: all K steps are there - no
// instruction of the chunk looks at n.
template <typename E, int FORM, int V, int K, bool BACKWARD, int MODE, bool FULL, bool STREAM>
__device__ __forceinline__ void walk_chunk(const RecurrenceParams& P, const Column<E, V, STREAM>& col, int64_t s0, int n, bool more, Composite (&carry)[V], float2* lds) {
  constexpr bool kStates = !BACKWARD || (MODE != kComposites && FORM != kGateConstant);  // x and the states are looked at
  constexpr bool kEdges = sizeof(E) == 2 && FORM != kGateConstant && MODE != kComposites;
  float x[K][V], f[K][V], inject[K][V], up[BACKWARD ? K : 1][V], front[V], edge[V];
  uint32_t cut[V];  // bit k: a reset at step k of the chunk
  auto there = [&](int k) { return FULL || k < n; };
  // every load of the chunk first, then the arithmetic: K independent rows in flight
  {
    const E *px = col.at(P.x, s0), *pg = col.at(P.g, s0), *pd = col.at(P.dh, s0);
#pragma unroll
    for (int k = 0; k < K; ++k, px += P.x.st, pg += P.g.st, pd += P.dh.st) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = f[k][j] = 0.0f;
      if (there(k)) {
        if (kStates) col.load(px, x[k]);
        if (FORM != kGateConstant) col.load(pg, f[k]);
        if (BACKWARD) col.load(pd, up[k]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) front[j] = 1.0f, edge[j] = 0.0f, cut[j] = 0;
  if (BACKWARD && (FULL || n > 0)) {
    // the gate that carries d into the chunk belongs to the step before it, the state in front of its last step to the step behind it
    // (the backward pass walks from the end)
    if (s0 > 0 && FORM != kGateConstant) col.load(col.at(P.g, s0 - 1), front);
    if (kStates) {
      if (s0 + n >= P.steps) col.load_batch(P, P.initial, edge);
      else if (kEdges && P.edges != nullptr) col.load_edge(P, s0 + n, edge);
      else if (P.h.p != nullptr) col.load(col.at(P.h, s0 + n), edge);
    }
  }
  if (P.reset.p != nullptr) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (there(k) && col.flag(P.reset, s0 + k, j)) cut[j] |= 1u << k;
  }
  if (BACKWARD && (FULL || n > 0) && s0 > 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float unused;
      gate<FORM>(P, front[j], unused);
      if (P.reset.p != nullptr && col.flag(P.reset, s0 - 1, j)) front[j] = 0.0f;
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) gate<FORM>(P, f[k][j], inject[k][j]);
  auto keep = [&](int k, int j) { return cut[j] >> k & 1 ? 0.0f : f[k][j]; };
  auto factor = [&](int k, int j) { return !BACKWARD ? keep(k, j) : k == 0 ? front[j] : keep(k - 1, j); };  // what multiplies the carried value at step k
  if (!BACKWARD && FORM == kGateLogit) {  // (from here on only the product is wanted)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] *= inject[k][j];
  }
  auto term = [&](int k, int j) { return BACKWARD ? up[k][j] : x[k][j]; };
  float start[V];
#pragma unroll
  for (int j = 0; j < V; ++j) start[j] = carry[j].b;
  if (MODE != kAlone) {
    Composite mine[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float a = 1.0f, b = 0.0f;
      bool dropped = false;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (there(k)) {
          const float m = factor(k, j);
          if (FORM != kGateConstant) a *= m;
          b = advance<FORM>(P, m, b, term(k, j));
          dropped = dropped || m == 0.0f;
        }
      }
      if (FORM == kGateConstant) a = P.power[BACKWARD && s0 == 0 && n > 0 ? n - 1 : n];
      mine[j] = {dropped ? 0.0f : not_dropped(a), b};
    }
    join_chunks<V>(mine, carry, more, P.lanes_log2, lds);
#pragma unroll
    for (int j = 0; j < V; ++j) start[j] = mine[j].b;
  }
  if (MODE == kComposites) return;
  if (!BACKWARD) {
    E* ph = col.at(P.h, s0);
#pragma unroll
    for (int k = 0; k < K; ++k, ph += P.h.st) {
      if (there(k)) {
#pragma unroll
        for (int j = 0; j < V; ++j) start[j] = advance<FORM>(P, keep(k, j), start[j], x[k][j]);
        col.store(ph, start);
        if (kEdges && P.edges != nullptr) {
          const int64_t left = P.steps - 1 - s0 - k;
          if (left > 0 && (left & ((int64_t{1} << P.edge_log2) - 1)) == 0) col.store_edge(P, left, start);
        }
      }
    }
    if (P.final_state != nullptr && n > 0 && s0 + n == P.steps) {
#pragma unroll
      for (int j = 0; j < V; ++j) P.final_state[col.batch(P, j)] = start[j];
    }
  } else {
    if (kStates) {  // the states once more, in the order of the forward pass: x turns into what dg multiplies
#pragma unroll
      for (int k = K - 1; k >= 0; --k) {
        if (there(k)) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float before = cut[j] >> k & 1 ? 0.0f : edge[j], value = x[k][j];
            edge[j] = apply_step(keep(k, j), edge[j], inject[k][j] * value);
            x[k][j] = FORM == kGateLogit ? f[k][j] * inject[k][j] * (before - value) : before;
          }
        }
      }
    }
    E *pdx = col.at(P.dx, s0), *pdg = col.at(P.dg, s0);
#pragma unroll
    for (int k = 0; k < K; ++k, pdx += P.dx.st, pdg += P.dg.st) {
      if (there(k)) {
        float out[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          start[j] = advance<FORM>(P, factor(k, j), start[j], up[k][j], k == 0 && s0 == 0);
          out[j] = inject[k][j] * start[j];
        }
        if (P.dx.p != nullptr) col.store(pdx, out);
        if (kStates && P.dg.p != nullptr) {
#pragma unroll
          for (int j = 0; j < V; ++j) out[j] = x[k][j] * start[j];
          col.store(pdg, out);
        }
      }
    }
    if (P.dinitial != nullptr && n > 0 && s0 + n == P.steps) {  // (what multiplies d behind the last step is that step's own gate)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float last = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (k == n - 1) last = keep(k, j);
        P.dinitial[col.batch(P, j)] = advance<FORM>(P, last, start[j], 0.0f);
      }
    }
  }
  if (MODE == kAlone) {
#pragma unroll
    for (int j = 0; j < V; ++j) carry[j].b = start[j];
  }
}

template <typename E, int FORM, int V, int K, bool BACKWARD, int MODE, bool STREAM = false>
__global__ __launch_bounds__(MODE == kAlone ? 256 : 1024, 4) void recurrence_columns(const RecurrenceParams P) {
  static_assert(K <= kMostSteps, "the powers of a constant gate");
  extern __shared__ float2 lds[];
  const int columns = MODE == kAlone ? blockDim.x : 1 << P.lanes_log2;
  const int chunk = MODE == kAlone ? 0 : threadIdx.x >> P.lanes_log2;
  const int chunks = MODE == kAlone ? 1 : blockDim.x >> P.lanes_log2;
  const int64_t block = blockIdx.x;
  const int64_t segment = MODE == kAlone ? 0 : block / P.column_blocks;
  const int64_t vector = (MODE == kAlone ? block : block % P.column_blocks) * columns + (threadIdx.x & (columns - 1));
  const bool active = vector < P.vectors;
  if (MODE == kAlone && !active) return;
  Column<E, V, STREAM> col;  // (a lane behind the last column has no steps to walk; it joins in with nothing)
  col.o = active ? vector / P.vectors_per_outer : 0;
  col.i = active ? (vector % P.vectors_per_outer) * V : 0;
  const int64_t begin = segment * P.segment, end = begin + P.segment < P.steps ? begin + P.segment : P.steps;

  Composite carry[V];  // a state (0, h), or - composites only - what the walk so far composes to
  {
    float h[V];
    col.load_batch(P, BACKWARD ? P.dfinal : P.initial, h);
#pragma unroll
    for (int j = 0; j < V; ++j) carry[j] = MODE == kComposites ? Composite{1.0f, 0.0f} : Composite{0.0f, h[j]};
  }
  if (MODE == kJoined && segment > 0) {  // the segments in front of this one: their composites, a contiguous run of them per chunk
    Composite mine[V];
    const int64_t run = (segment + chunks - 1) / chunks, from = chunk * run, to = from + run < segment ? from + run : segment;
#pragma unroll
    for (int j = 0; j < V; ++j) mine[j] = {1.0f, 0.0f};
    if (active) {
      for (int64_t q = from; q < to; q += 8) {  // (eight loads at a time)
        float2 c[8][V];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) c[i][j] = P.composites[((q + i < to ? q + i : q) * P.vectors + vector) * V + j];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (q + i < to) mine[j] = then(mine[j], {c[i][j].x, c[i][j].y});
      }
    }
    join_chunks<V>(mine, carry, true, P.lanes_log2, lds);
  }

  const int64_t tile = static_cast<int64_t>(chunks) * K;
  for (int64_t base = begin; base < end; base += tile) {
    const int64_t s0 = base + static_cast<int64_t>(chunk) * K;
    const bool more = MODE == kComposites || base + tile < end;
    // (decided for the whole workgroup, which meets at the join's barriers)
    if (base + tile <= end && P.whole_blocks) {
      walk_chunk<E, FORM, V, K, BACKWARD, MODE, true, STREAM>(P, col, s0, K, more, carry, lds);
    } else {
      const int n = !active || s0 >= end ? 0 : static_cast<int>(end - s0 < K ? end - s0 : K);
      walk_chunk<E, FORM, V, K, BACKWARD, MODE, false, STREAM>(P, col, s0, n, more, carry, lds);
    }
  }
  if (MODE == kComposites && chunk == 0 && active) {
#pragma unroll
    for (int j = 0; j < V; ++j) P.composites[(segment * P.vectors + vector) * V + j] = make_float2(carry[j].a, carry[j].b);
  }
}

// ---- rows --------------------------------------------------------------------------------------------------------------------------
// Steps of a lane: more of them mean fewer levels and lanes of the scans that bound this layout (65536 x 200 float32, value gates, 4 / 8 / 16: forward
// 40 / 32 / 48 us, backward 81 / 65 / -).
constexpr int kRowSteps = 8;

// V steps in walking order from s; memory runs the other way when the walk is reversed.  Steps at or behind `end` come back as zero.  A row's last
// lane may have some of its 16-byte pieces.
template <typename E, int V>
__device__ __forceinline__ void load_steps(const E* row, int64_t st, int64_t s, int64_t end, float (&out)[V]) {
  constexpr int W = 16 / sizeof(E);
  if (s + V <= end) {
    if (st > 0) {
      const Pack<E, V> v = load_pack<E, V>(row + s);
#pragma unroll
      for (int j = 0; j < V; ++j) out[j] = static_cast<float>(v.e[j]);
    } else {
      const Pack<E, V> v = load_pack<E, V>(row - s - (V - 1));
#pragma unroll
      for (int j = 0; j < V; ++j) out[j] = static_cast<float>(v.e[V - 1 - j]);
    }
  } else if constexpr (V > W) {
    float part[V / W][W];
#pragma unroll
    for (int k = 0; k < V / W; ++k) {
      load_steps<E, W>(row, st, s + k * W, end, part[k]);
#pragma unroll
      for (int j = 0; j < W; ++j) out[k * W + j] = part[k][j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = s + j < end ? static_cast<float>(row[(s + j) * st]) : 0.0f;
  }
}
template <typename E, int V>
__device__ __forceinline__ void store_steps(E* row, int64_t st, int64_t s, int64_t end, const float (&in)[V]) {
  constexpr int W = 16 / sizeof(E);
  if (s + V <= end) {
    Pack<E, V> v;
    if (st > 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) v.e[j] = static_cast<E>(in[j]);
      store_pack<E, V>(row + s, v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v.e[V - 1 - j] = static_cast<E>(in[j]);
      store_pack<E, V>(row - s - (V - 1), v);
    }
  } else if constexpr (V > W) {
#pragma unroll
    for (int k = 0; k < V / W; ++k) {
      float part[W];
#pragma unroll
      for (int j = 0; j < W; ++j) part[j] = in[k * W + j];
      store_steps<E, W>(row, st, s + k * W, end, part);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (s + j < end) row[(s + j) * st] = static_cast<E>(in[j]);
  }
}

// what V steps of one lane compose to, in walking order (DOWN: from the last)
template <int V, bool DOWN>
__device__ __forceinline__ Composite compose(const float (&keep)[V], const float (&term)[V]) {
  float a = 1.0f, b = 0.0f;
  bool dropped = false;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int j = DOWN ? V - 1 - i : i;
    a *= keep[j];
    b = apply_step(keep[j], b, term[j]);
    dropped = dropped || keep[j] == 0.0f;
  }
  return {dropped ? 0.0f : not_dropped(a), b};
}

// what the first n steps of one lane compose to under a constant gate: the constant with its rest, its power from the table (a drop leaves none).
// ENTERING: the first factor is one, not the constant.
template <int V>
__device__ __forceinline__ Composite constant_run(const RecurrenceParams& P, int n, bool entering, const float (&factor)[V], const float (&term)[V]) {
  float b = 0.0f;
  bool dropped = false;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (j < n) {
      b = advance<kGateConstant>(P, factor[j], b, term[j], j == 0 && entering);
      dropped = dropped || factor[j] == 0.0f;
    }
  }
  return {dropped ? 0.0f : P.power[entering && n > 0 ? n - 1 : n], b};
}

// inclusive prefix of the composites over a group of 2^log2 lanes (UP: towards higher lanes), then the exclusive one; `total`, where it is wanted: the
// whole group's
template <bool UP>
__device__ __forceinline__ void group_scan(Composite mine, int log2, Composite& exclusive, Composite& total, bool want_total) {
  const int width = 1 << log2, at = (threadIdx.x & 63) & (width - 1);
  for (int d = 1; d < width; d <<= 1) {
    const Composite other = UP ? Composite{__shfl_up(mine.a, d, width), __shfl_up(mine.b, d, width)}
                               : Composite{__shfl_down(mine.a, d, width), __shfl_down(mine.b, d, width)};
    if (UP ? at >= d : at + d < width) mine = then(other, mine);
  }
  if (want_total) total = {__shfl(mine.a, UP ? width - 1 : 0, width), __shfl(mine.b, UP ? width - 1 : 0, width)};
  if (width > 1) {
    const Composite other = UP ? Composite{__shfl_up(mine.a, 1, width), __shfl_up(mine.b, 1, width)}
                               : Composite{__shfl_down(mine.a, 1, width), __shfl_down(mine.b, 1, width)};
    exclusive = (UP ? at > 0 : at + 1 < width) ? other : Composite{1.0f, 0.0f};
  } else {
    exclusive = {1.0f, 0.0f};
  }
}

template <typename E, int FORM, int V, bool BACKWARD, bool COMPOSITES>
__global__ __launch_bounds__(256) void recurrence_rows(const RecurrenceParams P) {
  const int log2 = P.lanes_log2, width = 1 << log2, lane = (threadIdx.x & 63) & (width - 1);
  const int64_t group = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> log2;
  int64_t row = group / P.segments;
  const int64_t segment = group % P.segments, rows = P.outer * P.inner;
  // (a group past the last row walks the last one's empty range: every lane of the wave stays in step for the shuffles)
  const bool active = row < rows;
  if (!active) row = rows - 1;
  const int64_t o = row / P.inner, i = row % P.inner;
  const int64_t begin = segment * P.segment;
  const int64_t end = !active ? begin : begin + P.segment < P.steps ? begin + P.segment : P.steps;
  const int64_t last = begin + P.segment < P.steps ? begin + P.segment : P.steps;  // (loop bound: the same for every group of a wave when segments == 1)
  auto at = [&](const Axis& t) { return static_cast<E*>(t.p) + o * t.so + i * t.si; };
  const uint8_t* reset = P.reset.p == nullptr ? nullptr : static_cast<const uint8_t*>(P.reset.p) + o * P.reset.so + i * P.reset.si;
  const int64_t batch = P.batch_swapped ? i * P.outer + o : o * P.inner + i;
  const E *px = at(P.x), *pg = at(P.g), *ph = at(P.h), *pd = at(P.dh);

  const float* entering = BACKWARD ? P.dfinal : P.initial;
  constexpr bool kStates = !BACKWARD || (!COMPOSITES && FORM != kGateConstant);
  constexpr bool kEdges = sizeof(E) == 2 && FORM != kGateConstant && !COMPOSITES;
  Composite carry = COMPOSITES ? Composite{1.0f, 0.0f} : Composite{0.0f, entering != nullptr && active ? entering[batch] : 0.0f};
  if (!COMPOSITES && segment > 0) {  // (segments > 1: a group is a whole wave, so every lane takes the same way)
    Composite before = {1.0f, 0.0f};
    for (int64_t q = 0; q < segment; q += 64) {
      Composite mine = {1.0f, 0.0f}, exclusive, total;
      if (q + lane < segment) {
        const float2 c = P.composites[row * P.segments + q + lane];
        mine = {c.x, c.y};
      }
      group_scan<true>(mine, log2, exclusive, total, true);
      before = then(before, total);
    }
    carry = then(carry, before);
  }
  float keep_before = 1.0f;  // backward: the gate that carries d into this tile
  if (BACKWARD && begin > 0 && active) {
    float unused;
    if (FORM != kGateConstant) keep_before = static_cast<float>(pg[(begin - 1) * P.g.st]);
    gate<FORM>(P, keep_before, unused);
    if (reset != nullptr && reset[(begin - 1) * P.reset.st] != 0) keep_before = 0.0f;
  }

  // what one tile reads; the next tile's is requested before this one is worked on
  struct Tile {
    float x[V], g[V], up[V], edge;
    uint32_t cut;
  };
  const int64_t tile = static_cast<int64_t>(width) * V;
  auto fetch = [&](int64_t base, Tile& t) {
    const int64_t s = base + static_cast<int64_t>(lane) * V;
    t.cut = 0;
    t.edge = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) t.x[j] = t.g[j] = t.up[j] = 0.0f;
    if (kStates) load_steps<E, V>(px, P.x.st, s, end, t.x);
    if (FORM != kGateConstant) load_steps<E, V>(pg, P.g.st, s, end, t.g);
    if (BACKWARD) load_steps<E, V>(pd, P.dh.st, s, end, t.up);
    if (BACKWARD && kStates && base < end) {  // the state behind the tile (in front of it, for the forward order)
      const int64_t behind = base + tile < end ? base + tile : end;
      if (behind >= P.steps) t.edge = P.initial != nullptr ? P.initial[batch] : 0.0f;
      else if (kEdges && P.edges != nullptr) t.edge = P.edges[((behind >> P.edge_log2) - 1) * rows + batch];
      else if (P.h.p != nullptr) t.edge = static_cast<float>(ph[behind * P.h.st]);
    }
    if (reset != nullptr) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (s + j < end && reset[(s + j) * P.reset.st] != 0) t.cut |= 1u << j;
    }
  };
  Tile t, next;
  fetch(begin, t);
  for (int64_t base = begin; base < last; base += tile, t = next) {
    const bool more = COMPOSITES || base + tile < last;
    if (base + tile < last) fetch(base + tile, next);
    const int64_t s = base + static_cast<int64_t>(lane) * V;
    const int n = s >= end ? 0 : end - s < V ? static_cast<int>(end - s) : V;
    float keep[V], inject[V], term[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      gate<FORM>(P, t.g[j], inject[j]);
      keep[j] = t.cut >> j & 1 ? 0.0f : t.g[j];
      if (s + j >= end) keep[j] = 1.0f, inject[j] = 0.0f;  // steps behind the end change nothing
      term[j] = FORM == kGateLogit ? inject[j] * t.x[j] : s + j < end ? t.x[j] : 0.0f;
    }
    if (!BACKWARD) {
      const Composite mine = FORM == kGateConstant ? constant_run(P, n, false, keep, term) : compose<V, false>(keep, term);
      Composite exclusive, total;
      group_scan<true>(mine, log2, exclusive, total, more);
      if (!COMPOSITES) {
        float h = then(carry, exclusive).b, out[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (s + j < end) {
            h = advance<FORM>(P, keep[j], h, term[j]);
            if (kEdges && P.edges != nullptr) {
              const int64_t left = P.steps - 1 - s - j;
              if (left > 0 && (left & ((int64_t{1} << P.edge_log2) - 1)) == 0) P.edges[((left >> P.edge_log2) - 1) * rows + batch] = h;
            }
          }
          out[j] = h;
        }
        store_steps<E, V>(at(P.h), P.h.st, s, end, out);
        if (P.final_state != nullptr && s < P.steps && s + V >= P.steps && end == P.steps) P.final_state[batch] = h;
      }
      if (more) carry = then(carry, total);
    } else {
      // d: the gate in front of each step is its left neighbour's
      const float left = __shfl_up(keep[V - 1], 1, width);
      const float front = lane == 0 ? keep_before : left;
      float factor[V];
#pragma unroll
      for (int j = 0; j < V; ++j) factor[j] = s + j >= end ? 1.0f : j == 0 ? front : keep[j - 1];
      // (nothing comes in behind the end: up is zero there)
      const Composite mine = FORM == kGateConstant ? constant_run(P, n, s == 0, factor, t.up) : compose<V, false>(factor, t.up);
      Composite exclusive, total;
      group_scan<true>(mine, log2, exclusive, total, more);
      keep_before = __shfl(keep[V - 1], width - 1, width);  // (read only when another tile follows, and then this one was full)
      if (!COMPOSITES) {
        float scale[V];
#pragma unroll
        for (int j = 0; j < V; ++j) scale[j] = 0.0f;
        if (FORM != kGateConstant) {  // the states once more: forward order runs towards lower lanes
          Composite behind, unused;
          group_scan<false>(compose<V, true>(keep, term), log2, behind, unused, false);
          float h = apply_step(behind.a, t.edge, behind.b);
#pragma unroll
          for (int j = V - 1; j >= 0; --j) {
            if (s + j < end) {
              const float before = t.cut >> j & 1 ? 0.0f : h;
              scale[j] = FORM == kGateLogit ? t.g[j] * inject[j] * (before - t.x[j]) : before;
              h = apply_step(keep[j], h, term[j]);
            }
          }
        }
        float d = then(carry, exclusive).b, out[V], gate_out[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (s + j < end) {
            d = advance<FORM>(P, j == 0 ? front : keep[j - 1], d, t.up[j], j == 0 && s == 0);
            if (s + j + 1 == P.steps && P.dinitial != nullptr) P.dinitial[batch] = advance<FORM>(P, keep[j], d, 0.0f);
          }
          out[j] = inject[j] * d;
          gate_out[j] = scale[j] * d;
        }
        if (P.dx.p != nullptr) store_steps<E, V>(at(P.dx), P.dx.st, s, end, out);
        if (FORM != kGateConstant && P.dg.p != nullptr) store_steps<E, V>(at(P.dg), P.dg.st, s, end, gate_out);
      }
      if (more) carry = then(carry, total);
    }
  }
  if (COMPOSITES && lane == 0 && active) P.composites[row * P.segments + segment] = make_float2(carry.a, carry.b);
}

// ---- one step ----------------------------------------------------------------------------------------------------------------------
// new = keep state + inject x: what a recurrent actor does between two environment steps.  n elements, V per thread; the reset mask has
// strides of its own (a mask per lane, expanded over the lane's channels, costs one byte per lane).  2.6 us at 64000 elements, a launch's own time;
// 58 us at 2^24 float32 (5.8 TB/s), 60 with a mask per lane.
template <typename E, int FORM, int V>
__global__ __launch_bounds__(256) void recurrence_step(const float* state, const E* x, const E* g, const uint8_t* reset, int64_t reset_columns, int64_t rs,
                                                       int64_t rc, E* out, float* new_state, int64_t n) {
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * V;
  if (at >= n) return;
  const int nv = n - at < V ? static_cast<int>(n - at) : V;
  float h[V], xs[V], gs[V];
  if (nv == V) {
    const Pack<float, V> hv = load_pack<float, V>(state + at);
    const Pack<E, V> xv = load_pack<E, V>(x + at), gv = load_pack<E, V>(g + at);
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = hv.e[j], xs[j] = static_cast<float>(xv.e[j]), gs[j] = static_cast<float>(gv.e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool in = j < nv;
      h[j] = in ? state[at + j] : 0.0f;
      xs[j] = in ? static_cast<float>(x[at + j]) : 0.0f;
      gs[j] = in ? static_cast<float>(g[at + j]) : 0.0f;
    }
  }
  Pack<E, V> ov;
  Pack<float, V> sv;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    bool dropped = false;
    if (reset != nullptr && j < nv) dropped = reset[(at + j) / reset_columns * rs + (at + j) % reset_columns * rc] != 0;
    float f = gs[j], inject = 1.0f;
    if (FORM == kGateLogit) sigmoid_pair(gs[j], f, inject);
    const float next = apply_step(dropped ? 0.0f : f, h[j], inject * xs[j]);
    sv.e[j] = next;
    ov.e[j] = static_cast<E>(next);
  }
  if (nv == V) {
    store_pack<float, V>(new_state + at, sv);
    store_pack<E, V>(out + at, ov);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < nv) new_state[at + j] = sv.e[j], out[at + j] = ov.e[j];
  }
}

// one translation unit per element type (kernels_recurrence_*.hip): picks the instantiation and launches it
template <typename E>
int launch_recurrence(const RecurrenceParams& P, int form, bool backward, int which, unsigned blocks, unsigned threads, size_t lds, hipStream_t stream);
enum : int { kColumnsScalar = 0, kColumnsPair = 4, kColumnsWide = 8, kRows = 12 };  // + kAlone / kJoined / kComposites

}  // namespace mbt_learning
