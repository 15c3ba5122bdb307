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
// the states it needs are RECOMPUTED in registers from x and g, from the stored state at the edge of a chunk, instead of read back - which
// also keeps the rounding of a 16-bit state out of dg.
//
// Two layouts, each with one element of time per register so that no shared-memory transpose is needed:
//   columns  a batch axis is contiguous (time-major recordings, (B, T, C) activations): lanes lie across the batch, V neighbouring columns
//            per 16-byte access; the time axis is cut into chunks of K steps over the threads of a workgroup (LDS joins them) and, where even
//            that leaves the chip empty, into segments over workgroups (a first launch writes their composites)
//   rows     time is contiguous: lanes lie along time, V steps each, and a group of 2^n lanes scans by wave shuffles; segments as above
#pragma once
#include "learning_common.hpp"

namespace mbt_learning {

constexpr int kGateConstant = MBT_GATE_CONSTANT, kGateValue = MBT_GATE_VALUE, kGateLogit = MBT_GATE_LOGIT;

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
  int64_t steps, outer, inner;
  int64_t vectors_per_outer, vectors;  // column vectors (V columns each)
  int64_t segment;                     // steps per segment
  int32_t segments;
  int32_t lanes_log2;  // columns: column vectors per workgroup; rows: lanes per row
  int32_t batch_initial_swapped;  // initial / final are (outer, inner) of the CALLER; 1 when the kernel's axes are exchanged
  int64_t column_blocks;
  float constant;
};

__device__ __forceinline__ float apply_step(float keep, float h, float b) { return keep == 0.0f ? b : __builtin_fmaf(keep, h, b); }

struct Composite {
  float a, b;
};
// first, then second.  The product of two non-zero gates must not underflow to the zero that means "dropped".
__device__ __forceinline__ Composite then(Composite first, Composite second) {
  float a = first.a * second.a;
  if (a == 0.0f && first.a != 0.0f && second.a != 0.0f) a = 1.4e-45f;
  return {a, apply_step(second.a, first.b, second.b)};
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
  if (k != k) f = i = k;
}

template <int FORM>
__device__ __forceinline__ void gates(float g, bool reset, float constant, float& keep, float& f, float& i) {
  if (FORM == kGateConstant) f = constant, i = 1.0f;
  if (FORM == kGateValue) f = g, i = 1.0f;
  if (FORM == kGateLogit) sigmoid_pair(g, f, i);
  keep = reset ? 0.0f : f;
}

// ---- columns -----------------------------------------------------------------------------------------------------------------------
// MODE: whole time axis in one thread (kAlone), cut over the threads of the workgroup (kJoined; after kComposites when there are segments).
enum : int { kAlone = 0, kJoined = 1, kComposites = 2 };

template <typename E, int V>
struct Column {
  int64_t o, i;
  int nv;  // valid columns of the V (0: a lane without work)

  __device__ __forceinline__ void load(const Axis& t, int64_t s, float (&out)[V]) const {
    const E* p = static_cast<const E*>(t.p) + o * t.so + s * t.st + i * t.si;
    if (nv == V) {
      const Pack<E, V> v = load_pack<E, V>(p);
#pragma unroll
      for (int j = 0; j < V; ++j) out[j] = static_cast<float>(v.e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) out[j] = j < nv ? static_cast<float>(p[j]) : 0.0f;
    }
  }
  __device__ __forceinline__ void store(const Axis& t, int64_t s, const float (&in)[V]) const {
    E* p = static_cast<E*>(t.p) + o * t.so + s * t.st + i * t.si;
    if (nv == V) {
      Pack<E, V> v;
#pragma unroll
      for (int j = 0; j < V; ++j) v.e[j] = static_cast<E>(in[j]);
      store_pack<E, V>(p, v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < nv) p[j] = static_cast<E>(in[j]);
    }
  }
  __device__ __forceinline__ bool flag(const Axis& t, int64_t s, int j) const {
    return j < nv && static_cast<const uint8_t*>(t.p)[o * t.so + s * t.st + (i + j) * t.si] != 0;
  }
  // (outer, inner) float32 of the caller
  __device__ __forceinline__ int64_t batch(const RecurrenceParams& P, int j) const {
    return P.batch_initial_swapped ? (i + j) * P.outer + o : o * P.inner + i + j;
  }
  __device__ __forceinline__ void load_batch(const RecurrenceParams& P, const float* p, float (&out)[V]) const {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = p != nullptr && j < nv ? p[batch(P, j)] : 0.0f;
  }
};

// Joins the composites of a workgroup's chunks, thread order = walking order for each column: on return `mine` is the composite of
// everything BEFORE this thread's chunk, `total` of the whole workgroup.  Within a wave by shuffles over the chunks (lane = chunk * C + column
// with C = 2^lanes_log2 columns), across waves through LDS.
template <int V>
__device__ __forceinline__ void join_chunks(Composite (&mine)[V], Composite (&total)[V], int lanes_log2, float2* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int columns = 1 << lanes_log2, column = lane & (columns - 1);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    for (int d = columns; d < 64; d <<= 1) {
      const Composite before = {__shfl_up(mine[j].a, d), __shfl_up(mine[j].b, d)};
      if (lane >= d) mine[j] = then(before, mine[j]);
    }
    if (lane >= 64 - columns) lds[(wave * V + j) * columns + column] = make_float2(mine[j].a, mine[j].b);
    const Composite before = {__shfl_up(mine[j].a, columns & 63), __shfl_up(mine[j].b, columns & 63)};
    mine[j] = lane >= columns ? before : Composite{1.0f, 0.0f};
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) {
    Composite all = {1.0f, 0.0f}, front = {1.0f, 0.0f};
    for (int w = 0; w < waves; ++w) {
      if (w == wave) front = all;
      const float2 c = lds[(w * V + j) * columns + column];
      all = then(all, {c.x, c.y});
    }
    total[j] = all;
    mine[j] = then(front, mine[j]);
  }
  __syncthreads();
}

template <typename E, int FORM, int V, int K, bool BACKWARD, int MODE>
__global__ __launch_bounds__(MODE == kAlone ? 256 : 1024) void recurrence_columns(const RecurrenceParams P) {
  extern __shared__ float2 lds[];
  const int columns = MODE == kAlone ? blockDim.x : 1 << P.lanes_log2;
  const int chunk = MODE == kAlone ? 0 : threadIdx.x >> P.lanes_log2;
  const int chunks = MODE == kAlone ? 1 : blockDim.x >> P.lanes_log2;
  const int64_t block = blockIdx.x;
  const int64_t segment = MODE == kAlone ? 0 : block / P.column_blocks;
  const int64_t vector = (MODE == kAlone ? block : block % P.column_blocks) * columns + (threadIdx.x & (columns - 1));
  Column<E, V> col;
  col.o = vector / P.vectors_per_outer;
  col.i = (vector % P.vectors_per_outer) * V;
  col.nv = vector >= P.vectors ? 0 : static_cast<int>(P.inner - col.i < V ? P.inner - col.i : V);
  if (MODE == kAlone && col.nv == 0) return;
  const int64_t begin = segment * P.segment, end = begin + P.segment < P.steps ? begin + P.segment : P.steps;

  float carry[V];
  col.load_batch(P, BACKWARD ? P.dfinal : P.initial, carry);
  if (MODE == kJoined && segment > 0) {  // the segments in front of this one: their composites, a contiguous run of them per chunk
    Composite mine[V], total[V];
    const int64_t run = (segment + chunks - 1) / chunks, from = chunk * run, to = from + run < segment ? from + run : segment;
#pragma unroll
    for (int j = 0; j < V; ++j) mine[j] = {1.0f, 0.0f};
    for (int64_t q = from; q < to; ++q) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (j < col.nv) {
          const float2 c = P.composites[(q * P.vectors + vector) * V + j];
          mine[j] = then(mine[j], {c.x, c.y});
        }
      }
    }
    join_chunks<V>(mine, total, P.lanes_log2, lds);
#pragma unroll
    for (int j = 0; j < V; ++j) carry[j] = apply_step(total[j].a, carry[j], total[j].b);
  }
  Composite whole[V];  // (kComposites)
#pragma unroll
  for (int j = 0; j < V; ++j) whole[j] = {1.0f, 0.0f};

  for (int64_t base = begin; base < end; base += static_cast<int64_t>(chunks) * K) {
    const int64_t s0 = base + static_cast<int64_t>(chunk) * K;
    const int n = col.nv == 0 || s0 >= end ? 0 : static_cast<int>(end - s0 < K ? end - s0 : K);
    float x[K][V], f[K][V], inject[K][V], keep[K][V], up[BACKWARD ? K : 1][V], front[V];
    // every load of the chunk first, then the arithmetic: K independent rows in flight
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = f[k][j] = 0.0f;
      if (k < n) {
        if (!(BACKWARD && (MODE == kComposites || FORM == kGateConstant))) col.load(P.x, s0 + k, x[k]);
        if (FORM != kGateConstant) col.load(P.g, s0 + k, f[k]);
        if (BACKWARD) col.load(P.dh, s0 + k, up[k]);
      }
    }
    float edge[V];  // the state in front of the chunk's last step (walking order of the backward pass: the one behind it)
#pragma unroll
    for (int j = 0; j < V; ++j) front[j] = 1.0f, edge[j] = 0.0f;
    if (BACKWARD && n > 0) {
      if (s0 > 0) {  // the gate that carries d into the chunk belongs to the step before
        float g0[V] = {};
        if (FORM != kGateConstant) col.load(P.g, s0 - 1, g0);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float unused_f, unused_i;
          gates<FORM>(g0[j], P.reset.p != nullptr && col.flag(P.reset, s0 - 1, j), P.constant, front[j], unused_f, unused_i);
        }
      }
      if (MODE != kComposites && FORM != kGateConstant) {
        if (s0 + n < P.steps) col.load(P.h, s0 + n, edge);
        else col.load_batch(P, P.initial, edge);
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool reset = P.reset.p != nullptr && k < n && col.flag(P.reset, s0 + k, j);
        gates<FORM>(f[k][j], reset, P.constant, keep[k][j], f[k][j], inject[k][j]);
      }
    }
    float start[V];
#pragma unroll
    for (int j = 0; j < V; ++j) start[j] = carry[j];
    if (MODE != kAlone) {
      Composite mine[V], total[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        mine[j] = {1.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float m = BACKWARD ? (k == 0 ? front[j] : keep[k - 1][j]) : keep[k][j];
          const float b = BACKWARD ? up[k][j] : inject[k][j] * x[k][j];
          if (k < n) mine[j] = then(mine[j], {m, b});
        }
      }
      join_chunks<V>(mine, total, P.lanes_log2, lds);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (MODE == kComposites) {
          whole[j] = then(whole[j], total[j]);
        } else {
          start[j] = apply_step(mine[j].a, carry[j], mine[j].b);
          carry[j] = apply_step(total[j].a, carry[j], total[j].b);
        }
      }
    }
    if (MODE == kComposites) continue;
    if (!BACKWARD) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (k < n) {
#pragma unroll
          for (int j = 0; j < V; ++j) start[j] = apply_step(keep[k][j], start[j], inject[k][j] * x[k][j]);
          col.store(P.h, s0 + k, start);
        }
      }
      if (MODE == kAlone) {
#pragma unroll
        for (int j = 0; j < V; ++j) carry[j] = start[j];
      }
      if (P.final_state != nullptr && n > 0 && s0 + n == P.steps) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < col.nv) P.final_state[col.batch(P, j)] = start[j];
      }
    } else {
      if (FORM != kGateConstant) {  // the states once more, in the order of the forward pass; `up` of step k keeps dh, x becomes what dg multiplies
#pragma unroll
        for (int k = K - 1; k >= 0; --k) {
          if (k < n) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const bool dropped = P.reset.p != nullptr && col.flag(P.reset, s0 + k, j);
              const float before = dropped ? 0.0f : edge[j];
              const float value = x[k][j];
              edge[j] = apply_step(keep[k][j], edge[j], inject[k][j] * value);
              x[k][j] = FORM == kGateLogit ? f[k][j] * inject[k][j] * (before - value) : before;
            }
          }
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (k < n) {
          float out[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            start[j] = apply_step(k == 0 ? front[j] : keep[k - 1][j], start[j], up[k][j]);
            out[j] = inject[k][j] * start[j];
          }
          if (P.dx.p != nullptr) col.store(P.dx, s0 + k, out);
          if (FORM != kGateConstant && P.dg.p != nullptr) {
#pragma unroll
            for (int j = 0; j < V; ++j) out[j] = x[k][j] * start[j];
            col.store(P.dg, s0 + k, out);
          }
          if (s0 + k + 1 == P.steps && P.dinitial != nullptr) {
#pragma unroll
            for (int j = 0; j < V; ++j)
              if (j < col.nv) P.dinitial[col.batch(P, j)] = keep[k][j] == 0.0f ? 0.0f : keep[k][j] * start[j];
          }
        }
      }
      if (MODE == kAlone) {
#pragma unroll
        for (int j = 0; j < V; ++j) carry[j] = start[j];
      }
    }
  }
  if (MODE == kComposites && chunk == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < col.nv) P.composites[(segment * P.vectors + vector) * V + j] = make_float2(whole[j].a, whole[j].b);
  }
}

// ---- rows --------------------------------------------------------------------------------------------------------------------------
// V steps in walking order from s; memory runs the other way when the walk is reversed.  Steps at or behind `end` come back as zero.
template <typename E, int V>
__device__ __forceinline__ void load_steps(const E* row, int64_t st, int64_t s, int64_t end, float (&out)[V]) {
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
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = s + j < end ? static_cast<float>(row[(s + j) * st]) : 0.0f;
  }
}
template <typename E, int V>
__device__ __forceinline__ void store_steps(E* row, int64_t st, int64_t s, int64_t end, const float (&in)[V]) {
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
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (s + j < end) row[(s + j) * st] = static_cast<E>(in[j]);
  }
}

// inclusive prefix of the composites over a group of 2^log2 lanes (UP: towards higher lanes), then the exclusive one; `total`: the whole group's
template <bool UP>
__device__ __forceinline__ void group_scan(Composite mine, int log2, Composite& exclusive, Composite& total) {
  const int width = 1 << log2, at = (threadIdx.x & 63) & (width - 1);
  for (int d = 1; d < width; d <<= 1) {
    const Composite other = UP ? Composite{__shfl_up(mine.a, d, width), __shfl_up(mine.b, d, width)}
                               : Composite{__shfl_down(mine.a, d, width), __shfl_down(mine.b, d, width)};
    if (UP ? at >= d : at + d < width) mine = then(other, mine);
  }
  total = {__shfl(mine.a, UP ? width - 1 : 0, width), __shfl(mine.b, UP ? width - 1 : 0, width)};
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
  const int64_t batch = P.batch_initial_swapped ? i * P.outer + o : o * P.inner + i;
  const E *px = at(P.x), *pg = at(P.g), *ph = at(P.h), *pd = at(P.dh);

  const float* entering = BACKWARD ? P.dfinal : P.initial;
  float carry = entering != nullptr && active ? entering[batch] : 0.0f;
  if (!COMPOSITES && segment > 0) {  // (segments > 1: a group is a whole wave, so every lane takes the same way)
    Composite before = {1.0f, 0.0f};
    for (int64_t q = 0; q < segment; q += 64) {
      Composite mine = {1.0f, 0.0f}, exclusive, total;
      if (q + lane < segment) {
        const float2 c = P.composites[row * P.segments + q + lane];
        mine = {c.x, c.y};
      }
      group_scan<true>(mine, log2, exclusive, total);
      before = then(before, total);
    }
    carry = apply_step(before.a, carry, before.b);
  }
  float keep_before = 1.0f;  // backward: the gate that carries d into this tile
  if (BACKWARD && begin > 0 && active) {
    float f, in;
    gates<FORM>(FORM == kGateConstant ? 0.0f : static_cast<float>(pg[(begin - 1) * P.g.st]), reset != nullptr && reset[(begin - 1) * P.reset.st] != 0, P.constant,
                keep_before, f, in);
  }
  Composite whole = {1.0f, 0.0f};

  for (int64_t base = begin; base < last; base += static_cast<int64_t>(width) * V) {
    const int64_t s = base + static_cast<int64_t>(lane) * V;
    float x[V], g[V] = {}, up[V] = {}, keep[V], inject[V];
    if (!(BACKWARD && (COMPOSITES || FORM == kGateConstant))) load_steps<E, V>(px, P.x.st, s, end, x);
    if (FORM != kGateConstant) load_steps<E, V>(pg, P.g.st, s, end, g);
    if (BACKWARD) load_steps<E, V>(pd, P.dh.st, s, end, up);
    bool dropped[V];
    float edge = 0.0f;
    const int64_t tile_end = base + static_cast<int64_t>(width) * V < end ? base + static_cast<int64_t>(width) * V : end;
    if (BACKWARD && !COMPOSITES && FORM != kGateConstant && active && base < end) {
      if (tile_end < P.steps) edge = static_cast<float>(ph[tile_end * P.h.st]);
      else if (P.initial != nullptr) edge = P.initial[batch];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      dropped[j] = reset != nullptr && s + j < end && reset[(s + j) * P.reset.st] != 0;
      float f;
      gates<FORM>(g[j], dropped[j], P.constant, keep[j], f, inject[j]);
      g[j] = f;
      if (s + j >= end) keep[j] = 1.0f, inject[j] = 0.0f;  // steps behind the end change nothing
    }
    if (!BACKWARD) {
      Composite mine = {1.0f, 0.0f}, exclusive, total;
#pragma unroll
      for (int j = 0; j < V; ++j) mine = then(mine, {keep[j], s + j < end ? inject[j] * x[j] : 0.0f});
      group_scan<true>(mine, log2, exclusive, total);
      if (COMPOSITES) {
        whole = then(whole, total);
        continue;
      }
      float h = apply_step(exclusive.a, carry, exclusive.b), out[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (s + j < end) h = apply_step(keep[j], h, inject[j] * x[j]);
        out[j] = h;
      }
      store_steps<E, V>(at(P.h), P.h.st, s, end, out);
      if (P.final_state != nullptr && s < P.steps && s + V >= P.steps && end == P.steps) P.final_state[batch] = h;
      carry = apply_step(total.a, carry, total.b);
    } else {
      // d: the gate in front of each step is its left neighbour's
      const float left = __shfl_up(keep[V - 1], 1, width);
      const float front = lane == 0 ? keep_before : left;
      Composite mine = {1.0f, 0.0f}, exclusive, total;
#pragma unroll
      for (int j = 0; j < V; ++j) mine = then(mine, s + j < end ? Composite{j == 0 ? front : keep[j - 1], up[j]} : Composite{1.0f, 0.0f});
      group_scan<true>(mine, log2, exclusive, total);
      keep_before = __shfl(keep[V - 1], width - 1, width);  // (read only when another tile follows, and then this one was full)
      if (COMPOSITES) {
        whole = then(whole, total);
        continue;
      }
      float scale[V];
#pragma unroll
      for (int j = 0; j < V; ++j) scale[j] = 0.0f;
      if (FORM != kGateConstant) {  // the states once more: forward order runs towards lower lanes
        Composite states = {1.0f, 0.0f}, behind, unused;
#pragma unroll
        for (int j = V - 1; j >= 0; --j) states = then(states, {keep[j], s + j < end ? inject[j] * x[j] : 0.0f});
        group_scan<false>(states, log2, behind, unused);
        float h = apply_step(behind.a, edge, behind.b);
#pragma unroll
        for (int j = V - 1; j >= 0; --j) {
          if (s + j < end) {
            const float before = dropped[j] ? 0.0f : h;
            scale[j] = FORM == kGateLogit ? g[j] * inject[j] * (before - x[j]) : before;
            h = apply_step(keep[j], h, inject[j] * x[j]);
          }
        }
      }
      float d = apply_step(exclusive.a, carry, exclusive.b), out[V], gate_out[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (s + j < end) {
          d = apply_step(j == 0 ? front : keep[j - 1], d, up[j]);
          if (s + j + 1 == P.steps && P.dinitial != nullptr) P.dinitial[batch] = keep[j] == 0.0f ? 0.0f : keep[j] * d;
        }
        out[j] = inject[j] * d;
        gate_out[j] = scale[j] * d;
      }
      if (P.dx.p != nullptr) store_steps<E, V>(at(P.dx), P.dx.st, s, end, out);
      if (FORM != kGateConstant && P.dg.p != nullptr) store_steps<E, V>(at(P.dg), P.dg.st, s, end, gate_out);
      carry = apply_step(total.a, carry, total.b);
    }
  }
  if (COMPOSITES && lane == 0 && active) P.composites[row * P.segments + segment] = make_float2(whole.a, whole.b);
}

// ---- one step ----------------------------------------------------------------------------------------------------------------------
// new = keep state + inject x: what a recurrent actor does between two environment steps.  n elements, V per thread; the reset mask has
// strides of its own (a mask per lane, expanded over the lane's channels, costs one byte per lane).
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
    float keep, f, inject;
    gates<FORM>(gs[j], dropped, 0.0f, keep, f, inject);
    const float next = apply_step(keep, h[j], inject * xs[j]);
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
enum : int { kColumnsScalar = 0, kColumnsVector = 4, kRows = 8 };  // + kAlone / kJoined / kComposites (rows: 1 = with, 2 = composites only)

}  // namespace mbt_learning
