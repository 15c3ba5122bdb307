// The C entry points of the gated linear recurrence: argument checks, the choice of layout and split, launches (kernels: recurrence.hpp).
#include <cmath>

#include "recurrence.hpp"

namespace mbt_learning {
template <typename E>
int launch_recurrence_step(const float* state, const void* x, const void* g, const uint8_t* reset, int64_t reset_columns, int64_t rs, int64_t rc, void* out,
                           float* new_state, int64_t n, int form, hipStream_t stream);

namespace {

struct Plan {
  RecurrenceParams params;
  int which;            // kColumnsScalar / kColumnsVector / kRows + mode
  unsigned threads;
  int64_t blocks;
  size_t lds;
  uint64_t workspace;
  int64_t piece;        // steps that the backward pass recomputes from one state
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int log2_ceil(int64_t n) {
  int l = 0;
  while ((int64_t{1} << l) < n) ++l;
  return l;
}

Axis walk(const mbt_array3& a, int64_t steps, bool down, size_t size, bool swap) {
  Axis t = {a.data, a.stride[0], a.stride[1], a.stride[2]};
  if (swap) {
    t.so = a.stride[2];
    t.si = a.stride[0];
  }
  if (a.data != nullptr && down) t.p = static_cast<char*>(a.data) + (steps - 1) * t.st * static_cast<int64_t>(size);
  if (down) t.st = -t.st;
  return t;
}

// The layout and split of one call; touches no device.
int make_plan(const mbt_recurrence* r, bool backward, Plan& plan) {
  if (r == nullptr) return mbt_set_error(MBT_ERR_INVALID, "null argument");
  if (!dtype_known(r->dtype)) return mbt_set_error(MBT_ERR_INVALID, "dtype %d: float32, bfloat16 and float16 are known", r->dtype);
  if (r->form < kGateConstant || r->form > kGateLogit) return mbt_set_error(MBT_ERR_INVALID, "form %d is none of MBT_GATE_*", r->form);
  const uint64_t limit = uint64_t{1} << 40;
  if (r->outer < 1 || r->steps < 1 || r->inner < 1) return mbt_set_error(MBT_ERR_INVALID, "outer, steps and inner have to be at least 1");
  if (r->outer > limit || r->steps > limit || r->inner > limit || r->outer > limit / r->inner)
    return mbt_set_error(MBT_ERR_INVALID, "sizes beyond 2^40");
  const bool gated = r->form != kGateConstant;
  if (gated && r->gate.data == nullptr) return mbt_set_error(MBT_ERR_INVALID, "this form needs a gate array");
  if ((!backward || gated) && (r->inputs.data == nullptr || (!backward && r->states.data == nullptr)))
    return mbt_set_error(MBT_ERR_INVALID, "inputs and states are needed");
  if (backward && r->grad_states.data == nullptr) return mbt_set_error(MBT_ERR_INVALID, "the backward pass needs grad_states");
  if (!gated && r->grad_gate.data != nullptr) return mbt_set_error(MBT_ERR_INVALID, "a constant gate has no gradient array");
  if (!gated && !std::isfinite(r->constant)) return mbt_set_error(MBT_ERR_INVALID, "the constant gate is not finite");
  if (!gated && !std::isfinite(static_cast<float>(r->constant))) return mbt_set_error(MBT_ERR_INVALID, "the constant gate %g is not finite in float32", r->constant);

  const int64_t steps = static_cast<int64_t>(r->steps);
  const size_t size = dtype_size(r->dtype);
  const int vector = 16 / static_cast<int>(size);
  const mbt_array3* main[6] = {};
  int count = 0;
  auto add = [&](const mbt_array3& a, bool used) {
    if (used && a.data != nullptr) main[count++] = &a;
  };
  add(r->inputs, !backward || gated);
  add(r->gate, gated);
  add(r->states, !backward || gated);
  add(r->grad_states, backward);
  add(r->grad_inputs, backward);
  add(r->grad_gate, backward && gated);
  bool time_contiguous = true, inner_contiguous = true, outer_contiguous = true;
  for (int k = 0; k < count; ++k) {
    time_contiguous = time_contiguous && (main[k]->stride[1] == 1);
    inner_contiguous = inner_contiguous && (r->inner == 1 || main[k]->stride[2] == 1);
    outer_contiguous = outer_contiguous && (r->outer == 1 || main[k]->stride[0] == 1);
  }
  // lanes lie along the batch axis that is contiguous; (N, 1, T) views of a time-major recording have it in front
  const bool swap = (r->inner == 1 && r->outer > 1) || (!inner_contiguous && outer_contiguous);
  if (swap) inner_contiguous = outer_contiguous;
  const bool down = (r->reverse != 0) != backward;

  RecurrenceParams& P = plan.params;
  P = RecurrenceParams{};
  P.x = walk(r->inputs, steps, down, size, swap);
  P.g = walk(r->gate, steps, down, size, swap);
  P.reset = walk(r->reset, steps, down, 1, swap);
  P.h = walk(r->states, steps, down, size, swap);
  P.dh = walk(r->grad_states, steps, down, size, swap);
  P.dx = walk(r->grad_inputs, steps, down, size, swap);
  P.dg = walk(r->grad_gate, steps, down, size, swap);
  P.initial = r->initial;
  P.final_state = backward ? nullptr : r->final_state;
  P.dfinal = r->grad_final;
  P.dinitial = r->grad_initial;
  if (r->edge_steps != 0) {
    const int64_t apart = r->edge_steps;
    if (apart < 0 || (apart & (apart - 1)) != 0) return mbt_set_error(MBT_ERR_INVALID, "edge_steps %d is no power of two", r->edge_steps);
    if (!gated || size != 2) return mbt_set_error(MBT_ERR_INVALID, "edges belong to 16-bit states with gates");
    const uint64_t needed = (static_cast<uint64_t>(ceil_div(steps, apart)) - 1) * r->outer * r->inner * sizeof(float);
    if (needed > 0 && (r->edges == nullptr || r->edges_bytes < needed))
      return mbt_set_error(MBT_ERR_INVALID, "edges has %llu bytes; %llu are needed", (unsigned long long)(r->edges == nullptr ? 0 : r->edges_bytes),
                           (unsigned long long)needed);
    if (reinterpret_cast<uintptr_t>(r->edges) % sizeof(float) != 0) return mbt_set_error(MBT_ERR_INVALID, "edges is not aligned to 4 bytes");
    P.edges = r->edges;
    P.edge_log2 = log2_ceil(apart);
  }
  P.steps = steps;
  P.outer = static_cast<int64_t>(swap ? r->inner : r->outer);
  P.inner = static_cast<int64_t>(swap ? r->outer : r->inner);
  P.batch_swapped = swap ? 1 : 0;
  auto not_dropped = [&](double v) {  // (only a constant of zero drops what it meets: one that float32 cannot hold is its smallest number)
    const float f = static_cast<float>(v);
    return f == 0.0f && r->constant != 0.0 ? std::copysign(1.4e-45f, f) : f;
  };
  P.constant = not_dropped(r->constant);
  P.constant_rest = static_cast<float>(r->constant - static_cast<double>(P.constant));
  double power = 1.0;
  for (int k = 0; k <= kMostSteps; ++k) {
    P.power[k] = not_dropped(power);
    power *= r->constant;
  }
  P.segments = 1;
  P.segment = steps;
  plan.lds = 0;
  plan.workspace = 0;
  const int64_t batch = P.outer * P.inner;
  const int64_t chip = 256 * 1024;  // threads that fill it at 16 waves per compute unit

  if (time_contiguous && steps > 1) {
    // rows: as many lanes as the steps of a row need; a row longer than 64 lanes' is cut into segments of a tile or more, one wave each, while the chip has
    // room for them (64 rows x 4096 steps, float32 logit form: forward 10.0 us, backward 11.0; in one piece 17.4 and 30.4).  From four segments on -
    // backwards three: the launch that their composites take costs 3 us more than it gains with fewer (64 x 1100: forward 10.9 us, 9.4 in one piece;
    // backward 12.1 and 14.1; 1024 x 4096 in two segments: forward 22.7, 19.9 in one piece)
    const int lanes = log2_ceil(ceil_div(steps, kRowSteps));
    P.lanes_log2 = lanes < 6 ? lanes : 6;
    const int64_t tile = (int64_t{1} << P.lanes_log2) * kRowSteps;
    int64_t want = chip / 64 / 2 / batch;  // (8 waves per compute unit)
    const int64_t most = ceil_div(steps, tile);
    want = want < most ? want : most;
    if (want >= (backward ? 3 : 4)) {  // (more than one tile: a group is a wave)
      P.segment = ceil_div(ceil_div(steps, want), tile) * tile;
      P.segments = static_cast<int32_t>(ceil_div(steps, P.segment));
    }
    plan.which = kRows + kJoined;
    plan.piece = tile;
    plan.threads = 256;
    plan.blocks = ceil_div(batch * P.segments, 256 >> P.lanes_log2);
    if (P.segments > 1) plan.workspace = static_cast<uint64_t>(batch) * P.segments * sizeof(float2);
    return MBT_OK;
  }

  // Columns per thread: one float32 or two 16-bit elements, so that a wave's row is 256 bytes and the time axis can be cut finely; a recording with
  // columns enough for every wave of the chip to have 64 x 16 bytes of its own is walked forwards in such vectors, alone (value gates, 50 steps x 2^20
  // float32 120 us, 135 by single columns; x 2^21 bfloat16 115 us, 133 by pairs; rewards-to-go 84 and 91, 80 and 91).  Not gated float32 rows of
  // 8 MB and more: 100 x 2^21 535 us, 501 by single columns; 50 x 2^22 600 and 501.
  const int pair = inner_contiguous && size == 2 && P.inner % 2 == 0 ? 2 : 1;
  const bool wide = !backward && !(gated && size == 4 && P.inner >= (1 << 21)) && inner_contiguous && P.inner % vector == 0 && P.outer * (P.inner / vector) >= chip;
  const int v = wide ? vector : pair;
  const int base = wide ? kColumnsWide : pair == 2 ? kColumnsPair : kColumnsScalar;
  P.vectors_per_outer = ceil_div(P.inner, v);
  P.vectors = P.outer * P.vectors_per_outer;
  const int chunk = chunk_steps(r->form, backward, v, false);
  plan.piece = chunk;
  int64_t parallel = ceil_div(chip, P.vectors);
  if (parallel > ceil_div(steps, chunk)) parallel = ceil_div(steps, chunk);
  // With two thirds of the chip's threads or more a thread walks its columns alone, without joins (200 x 3 * 2^16 bfloat16: 40 us forward and 98
  // backward, 51 and 116 joined; 50 x 3 * 2^16 15 and 18, 21 and 35); with a half it would not (200 x 2^16 float32: 29.4 and 56, joined 28.3 and 51).
  if (wide || parallel <= 3) {
    plan.which = base + kAlone;
    plan.piece = chunk_steps(r->form, backward, v, true);
    if (wide && batch * steps * static_cast<int64_t>(size) * count > (int64_t{256} << 20)) plan.which = base + kStreamed;  // (beyond the last cache)
    plan.threads = 256;
    plan.blocks = ceil_div(P.vectors, 256);
    P.whole_blocks = 1;  // (a lane without a column has left)
    return MBT_OK;
  }
  // A workgroup takes 64 column vectors (256 bytes of a row) and up to 1024 threads' worth of chunks of time, a tile.  Where that makes fewer workgroups
  // than compute units, and
  //   - the walk is at least four tiles long, and eight columns a workgroup would not make it one tile or leave much to walk (2^21 steps in all): the
  //     axis is cut into segments over workgroups as well (64 columns x 65536 steps, float32 logit form: 25 us forward; with 16 columns a
  //     workgroup and fewer segments 32.  2000 columns x 2000 float32: backward 31 us, 40 in narrow workgroups)
  //   - otherwise: a workgroup takes fewer columns, down to 16, or 8 if only that makes the walk one tile (1000 lanes x 200: 8.1 -> 5.6 us; 512
  //     columns x 1000 bfloat16: forward 11 us, backward 17; in segments 21 and 26.  4000 columns 20 and 27, 26 and 35)
  int columns_log2 = 6;
  while (columns_log2 > 0 && (int64_t{1} << (columns_log2 - 1)) >= P.vectors) --columns_log2;
  const int chunks_wanted = log2_ceil(parallel);
  auto chunks_with = [&](int columns) {
    int chunks = chunks_wanted < 10 - columns ? chunks_wanted : 10 - columns;
    return chunks + columns < 6 ? 6 - columns : chunks;
  };
  auto tile_with = [&](int columns) { return (int64_t{1} << chunks_with(columns)) * chunk; };
  auto blocks_with = [&](int columns) { return ceil_div(P.vectors, int64_t{1} << columns); };
  const bool narrow = steps <= tile_with(3) && steps * P.vectors <= (int64_t{1} << 21);
  if (blocks_with(columns_log2) < 128 && steps >= 4 * tile_with(columns_log2) && !narrow) {
    const int64_t tile = tile_with(columns_log2), most = ceil_div(steps, tile);
    int64_t want = 256 / blocks_with(columns_log2);
    want = want < most ? want : most;
    P.segment = ceil_div(ceil_div(steps, want), tile) * tile;
    P.segments = static_cast<int32_t>(ceil_div(steps, P.segment));
  } else {
    while (columns_log2 > 3 && blocks_with(columns_log2) < 256 && (columns_log2 > 4 || steps > tile_with(columns_log2))) --columns_log2;
  }
  const int64_t chunks = int64_t{1} << chunks_with(columns_log2), columns = int64_t{1} << columns_log2;
  P.lanes_log2 = columns_log2;
  P.column_blocks = blocks_with(columns_log2);
  P.whole_blocks = P.vectors % columns == 0;
  plan.which = base + kJoined;
  plan.threads = static_cast<unsigned>(chunks * columns);
  plan.blocks = P.column_blocks * P.segments;
  plan.lds = static_cast<size_t>(plan.threads / 64 + 1) * v * columns * sizeof(float2);
  if (P.segments > 1) plan.workspace = static_cast<uint64_t>(P.vectors) * v * P.segments * sizeof(float2);
  return MBT_OK;
}

int run(int device, const mbt_recurrence* r, bool backward, void* stream) {
  Plan plan;
  int rc = make_plan(r, backward, plan);
  if (rc != MBT_OK) return rc;
  if (plan.blocks > 0xffffffffll / plan.threads) return  // (a launch counts its threads in 32 bits)
      mbt_set_error(MBT_ERR_INVALID, "%llu x %llu sequences are more than one launch can walk", (unsigned long long)r->outer, (unsigned long long)r->inner);
  if (plan.workspace > 0 && (r->workspace == nullptr || r->workspace_bytes < plan.workspace))
    return mbt_set_error(MBT_ERR_INVALID, "the workspace has %llu bytes; %llu are needed (mbt_recurrence_workspace)",
                         (unsigned long long)(r->workspace == nullptr ? 0 : r->workspace_bytes), (unsigned long long)plan.workspace);
  if (reinterpret_cast<uintptr_t>(r->workspace) % sizeof(float2) != 0) return mbt_set_error(MBT_ERR_INVALID, "the workspace is not aligned to 8 bytes");
  if (backward && r->form != kGateConstant && r->grad_gate.data != nullptr && r->edge_steps == 0 && r->states.data == nullptr && plan.params.steps > plan.piece)
    return mbt_set_error(MBT_ERR_INVALID, "grad_gate needs states or edges");
  if (backward && r->edge_steps != 0 && plan.piece % r->edge_steps != 0)
    return mbt_set_error(MBT_ERR_INVALID, "edges %d steps apart: every %lld steps one is needed (mbt_recurrence_edge_steps)", r->edge_steps, (long long)plan.piece);
  DeviceScope scope;
  rc = scope.enter(device);
  if (rc != MBT_OK) return rc;
  plan.params.composites = static_cast<float2*>(r->workspace);
  auto launch = [&](int which) {
    const unsigned blocks = static_cast<unsigned>(plan.blocks);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (r->dtype == MBT_FLOAT32) return launch_recurrence<float>(plan.params, r->form, backward, which, blocks, plan.threads, plan.lds, s);
    if (r->dtype == MBT_BFLOAT16) return launch_recurrence<bfloat16>(plan.params, r->form, backward, which, blocks, plan.threads, plan.lds, s);
    return launch_recurrence<float16>(plan.params, r->form, backward, which, blocks, plan.threads, plan.lds, s);
  };
  if (plan.params.segments > 1) {
    rc = launch(plan.which - kJoined + kComposites);
    if (rc != MBT_OK) return rc;
  }
  return launch(plan.which);
}

}  // namespace
}  // namespace mbt_learning

extern "C" {

uint64_t mbt_recurrence_workspace(const mbt_recurrence* r, int backward) {
  mbt_learning::Plan plan;
  return mbt_learning::make_plan(r, backward != 0, plan) == MBT_OK ? plan.workspace : 0;
}

int32_t mbt_recurrence_edge_steps(const mbt_recurrence* r) {
  using namespace mbt_learning;
  Plan plan;
  if (make_plan(r, true, plan) != MBT_OK || dtype_size(r->dtype) != 2 || r->form == kGateConstant) return 0;
  return plan.params.steps > plan.piece ? static_cast<int32_t>(plan.piece) : 0;
}

int mbt_recurrence_forward(int device, const mbt_recurrence* r, void* stream) { return mbt_learning::run(device, r, false, stream); }

int mbt_recurrence_backward(int device, const mbt_recurrence* r, void* stream) { return mbt_learning::run(device, r, true, stream); }

int mbt_recurrence_step(int device, int dtype, int form, uint64_t rows, uint64_t columns, const float* state, const void* inputs, const void* gate,
                        const uint8_t* reset, int64_t reset_row_stride, int64_t reset_column_stride, void* out, float* new_state, void* stream) {
  using namespace mbt_learning;
  if (!dtype_known(dtype)) return mbt_set_error(MBT_ERR_INVALID, "dtype %d: float32, bfloat16 and float16 are known", dtype);
  if (form != kGateValue && form != kGateLogit) return mbt_set_error(MBT_ERR_INVALID, "a single step takes MBT_GATE_VALUE or MBT_GATE_LOGIT");
  if (state == nullptr || inputs == nullptr || gate == nullptr || out == nullptr || new_state == nullptr) return mbt_set_error(MBT_ERR_INVALID, "null argument");
  if (rows < 1 || columns < 1 || rows > (uint64_t{1} << 33) / columns) return mbt_set_error(MBT_ERR_INVALID, "rows x columns has to be within 1 .. 2^33");
  DeviceScope scope;
  int rc = scope.enter(device);
  if (rc != MBT_OK) return rc;
  const int64_t n = static_cast<int64_t>(rows * columns), width = static_cast<int64_t>(columns);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MBT_FLOAT32)
    return launch_recurrence_step<float>(state, inputs, gate, reset, width, reset_row_stride, reset_column_stride, out, new_state, n, form, s);
  if (dtype == MBT_BFLOAT16)
    return launch_recurrence_step<bfloat16>(state, inputs, gate, reset, width, reset_row_stride, reset_column_stride, out, new_state, n, form, s);
  return launch_recurrence_step<float16>(state, inputs, gate, reset, width, reset_row_stride, reset_column_stride, out, new_state, n, form, s);
}

}  // extern "C"
