// extern "C" entry points of libprism_moe.so (declared in include/prism_moe.h).
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <set>
#include <utility>

#include "common.cuh"
#include "internal.h"

namespace prism {

namespace {
thread_local char g_err[512] = "";
thread_local cudaEvent_t g_stage_events[kNumStageEvents] = {};
thread_local int g_num_stage_events = 0;
}

void record_stage(int slot, cudaStream_t st) {
  if (slot < g_num_stage_events && g_stage_events[slot]) cudaEventRecord(g_stage_events[slot], st);
}

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}

int cuda_status(cudaError_t e, const char* what) {
  set_error("%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
  return PRISM_MOE_ERR_CUDA;
}

namespace {
std::atomic<int> g_engine{PRISM_MOE_ENGINE_AUTO};
std::atomic<uint64_t> g_wait_ns{2000000000ull};        // 2 s: far above any legitimate wait
std::atomic<uint64_t> g_peer_wait_ns{10000000000ull};  // 10 s: peers may start a step late
std::mutex g_attr_mu;
std::set<std::pair<const void*, int>> g_attr_done;
__device__ int g_device_error;   // one on each device (prism_moe_device_error_word)
}  // namespace

int expert_engine_setting() { return g_engine.load(std::memory_order_relaxed); }
uint64_t wait_limit_ns() { return g_wait_ns.load(std::memory_order_relaxed); }
uint64_t peer_wait_limit_ns() { return g_peer_wait_ns.load(std::memory_order_relaxed); }

int ensure_smem_attr(const void* func, int bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "cudaGetDevice");
  std::lock_guard<std::mutex> lock(g_attr_mu);
  if (g_attr_done.count({func, dev})) return PRISM_MOE_OK;
  e = cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(MaxDynamicSharedMemorySize)");
  g_attr_done.insert({func, dev});
  return PRISM_MOE_OK;
}

int num_sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 1;
  return n > 0 ? n : 1;
}

namespace {

int check_device() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "cudaGetDevice");
  int major = 0, minor = 0;
  cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
  if (major != 10 || minor != 0) {
    set_error("libprism_moe targets sm_100a (B200); device %d is sm_%d%d", dev, major, minor);
    return PRISM_MOE_ERR_UNSUPPORTED;
  }
  return PRISM_MOE_OK;
}

bool dtype_ok(int dtype) { return dtype == PRISM_MOE_F32 || dtype == PRISM_MOE_BF16; }
int64_t elem_size(int dtype) { return dtype == PRISM_MOE_BF16 ? 2 : 4; }

struct BlockLayout {
  size_t err, ids, w, plan, counts, offsets, entry_row, xs, h, y, total, plan_bytes;
};

BlockLayout block_layout(int64_t T, int64_t H, int64_t I, int E, int k, int dtype) {
  BlockLayout L{};
  const int64_t N = T * k;
  const size_t es = static_cast<size_t>(elem_size(dtype));
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += align_up(bytes > 0 ? bytes : 1, 256);
    return at;
  };
  L.err = take(256);
  L.ids = take(sizeof(int64_t) * N);
  L.w = take(es * N);
  L.plan_bytes = dispatch_workspace_size(N, E, 1);
  L.plan = take(L.plan_bytes);
  L.counts = take(sizeof(int32_t) * E);
  L.offsets = take(sizeof(int32_t) * (E + 1));
  L.entry_row = take(sizeof(int32_t) * N);
  L.xs = take(es * N * H);
  L.h = take(expert_scratch_bytes(N, I, static_cast<int64_t>(es)));
  L.y = take(es * N * H);
  L.total = o;
  return L;
}

// 4-bit weights [n, k] of one matrix (or a stack): what the kernels need of them.
int check_w4(const char* what, const prism_moe_w4* w, int64_t k, int64_t n) {
  PRISM_CHECK_ARG(w && w->qweight && w->scales, "%s: null 4-bit weight", what);
  PRISM_CHECK_ARG(w->group_size == 32 || w->group_size == 64 || w->group_size == 128,
                  "%s: group_size %d is not 32, 64 or 128", what, w->group_size);
  PRISM_CHECK_ARG(k % w->group_size == 0, "%s: %lld inputs are not a multiple of group_size %d",
                  what, static_cast<long long>(k), w->group_size);
  PRISM_CHECK_ARG(n % 8 == 0, "%s: %lld outputs are not a multiple of 8", what,
                  static_cast<long long>(n));
  PRISM_CHECK_ARG(k < (int64_t(1) << 30) && n < (int64_t(1) << 30), "%s: matrix too large", what);
  PRISM_CHECK_ARG((reinterpret_cast<uintptr_t>(w->qweight) | reinterpret_cast<uintptr_t>(w->scales) |
                   reinterpret_cast<uintptr_t>(w->zeros)) % 16 == 0,
                  "%s: 4-bit weights must be 16-byte aligned", what);
  return PRISM_MOE_OK;
}

// The block's kernels read and write rows in 16-byte pieces.
int check_block_buffers(const char* what, const void* x, const void* out, const void* workspace,
                        const prism_moe_norm_epilogue* e) {
  uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out) |
                  reinterpret_cast<uintptr_t>(workspace);
  if (e)
    all |= reinterpret_cast<uintptr_t>(e->residual) | reinterpret_cast<uintptr_t>(e->norm_weight) |
           reinterpret_cast<uintptr_t>(e->residual_out);
  PRISM_CHECK_ARG(all % 16 == 0, "%s: buffers must be 16-byte aligned", what);
  // the residual is read again after ``out`` and ``residual_out`` have been written
  PRISM_CHECK_ARG(!e || (e->residual != out && e->residual != e->residual_out && e->residual_out != out),
                  "%s: residual, residual_out and out must be three buffers", what);
  return PRISM_MOE_OK;
}

size_t w4_scratch_bytes(int64_t rows, int64_t inter) {
  return align_up(static_cast<size_t>(2 * rows * inter), 256);
}

// gate_up with SwiGLU into ``h`` (bf16: the next product's operand type), then down.
int expert_swiglu_w4(const void* xs, int64_t rows, int64_t H, int64_t I,
                     const int32_t* seg_offsets, const int32_t* seg_expert, int nseg, int El,
                     const prism_moe_w4& gu, const prism_moe_w4& dn, void* y, void* h, int* err,
                     cudaStream_t st) {
  W4Problem p;
  p.x = xs;
  p.rows_cap = rows;
  p.K = H;
  p.n_out = I;
  p.swiglu = true;
  p.seg_offsets = seg_offsets;
  p.seg_expert = seg_expert;
  p.nseg = nseg;
  p.num_mats = El;
  p.w = gu;
  p.out = h;
  p.err = err;
  record_stage(3, st);
  if (int r = w4_product(p, st)) return r;
  record_stage(4, st);
  p.x = h;
  p.K = I;
  p.n_out = H;
  p.swiglu = false;
  p.w = dn;
  p.out = y;
  p.after_product = true;
  const int r = w4_product(p, st);
  record_stage(5, st);
  return r;
}

// Plan, gather, experts (dense, or 4-bit where ``q_gu`` is given) and combine for routed tokens. Errors
// go to ``err``, or to the workspace's first word where that is NULL.
int block_after_router(const void* x, const int64_t* ids, const void* w, int dtype, int64_t T,
                       int64_t H, int64_t I, int E, int k, const void* w_gate_up,
                       const void* w_down, const prism_moe_w4* q_gu, const prism_moe_w4* q_dn,
                       void* out, char* ws, const BlockLayout& L, int* err,
                       const prism_moe_norm_epilogue* epilogue, cudaStream_t st) {
  if (!err) err = reinterpret_cast<int*>(ws + L.err);
  int32_t* counts = reinterpret_cast<int32_t*>(ws + L.counts);
  int32_t* offsets = reinterpret_cast<int32_t*>(ws + L.offsets);
  int32_t* entry_row = reinterpret_cast<int32_t*>(ws + L.entry_row);
  void* xs = ws + L.xs;
  void* h = ws + L.h;
  void* y = ws + L.y;
  const int64_t N = T * k;
  record_stage(1, st);
  int r = build_plan(ids, T, k, E, 1, nullptr, nullptr, nullptr, counts, offsets, entry_row,
                     nullptr, ws + L.plan, L.plan_bytes, st, err);
  if (r) return r;
  record_stage(2, st);
  r = permute_rows(x, T, H * elem_size(dtype), k, entry_row, xs, st);
  if (r) return r;
  if (q_gu)
    r = expert_swiglu_w4(xs, N, H, I, offsets, nullptr, E, E, *q_gu, *q_dn, y, h, err, st);
  else if (dtype == PRISM_MOE_BF16)
    r = expert_swiglu_bf16(xs, N, H, I, offsets, nullptr, E, E, w_gate_up, w_down, y, h, err, st);
  else
    r = expert_swiglu_f32(static_cast<const float*>(xs), N, H, I, offsets, nullptr, E, E,
                          static_cast<const float*>(w_gate_up), static_cast<const float*>(w_down),
                          static_cast<float*>(y), static_cast<float*>(h), st);
  if (r) return r;
  CombineSource src{};
  if (epilogue) {
    src.residual = epilogue->residual;
    src.norm_weight = epilogue->norm_weight;
    src.residual_out = epilogue->residual_out;
    src.eps = epilogue->eps;
  }
  r = combine(y, dtype, entry_row, w, T, k, H, out, st, &src);
  record_stage(6, st);
  return r;
}

}  // namespace
}  // namespace prism

using namespace prism;

extern "C" {

int prism_moe_version(void) { return 100; }

const char* prism_moe_last_error(void) { return g_err; }

int prism_moe_route_topk(const void* logits, int dtype, int64_t num_tokens, int32_t num_experts,
                         int32_t top_k, int32_t renorm, int64_t* topk_ids, void* topk_weights,
                         int32_t* expert_counts, void* stream) {
  PRISM_CHECK_ARG(dtype_ok(dtype), "route_topk: unknown dtype %d", dtype);
  PRISM_CHECK_ARG(num_tokens >= 0, "route_topk: negative num_tokens");
  PRISM_CHECK_ARG(num_experts >= 1 && num_experts <= 1024, "route_topk: num_experts %d outside [1, 1024]",
                  num_experts);
  PRISM_CHECK_ARG(top_k >= 1 && top_k <= 32 && top_k <= num_experts,
                  "route_topk: top_k %d outside [1, min(num_experts, 32)]", top_k);
  PRISM_CHECK_ARG(num_tokens == 0 || (logits && topk_ids && topk_weights),
                  "route_topk: null pointer");
  if (int r = check_device()) return r;
  return route_topk(logits, dtype, num_tokens, num_experts, top_k, renorm, topk_ids, topk_weights,
                    expert_counts, static_cast<cudaStream_t>(stream));
}

int prism_moe_route_scored(const void* logits, int dtype, int64_t num_tokens, int32_t num_experts,
                           int32_t top_k, const prism_moe_router* router, int64_t* topk_ids,
                           void* topk_weights, int weights_dtype, int32_t* expert_counts,
                           void* stream) {
  PRISM_CHECK_ARG(dtype_ok(dtype) && dtype_ok(weights_dtype), "route_scored: unknown dtype %d / %d",
                  dtype, weights_dtype);
  PRISM_CHECK_ARG(num_tokens >= 0, "route_scored: negative num_tokens");
  PRISM_CHECK_ARG(router != nullptr, "route_scored: null router");
  PRISM_CHECK_ARG(num_experts >= 1 && num_experts <= 1024,
                  "route_scored: num_experts %d outside [1, 1024]", num_experts);
  PRISM_CHECK_ARG(router->scoring == PRISM_MOE_SCORE_SOFTMAX ||
                      router->scoring == PRISM_MOE_SCORE_SIGMOID,
                  "route_scored: unknown scoring %d", router->scoring);
  PRISM_CHECK_ARG(router->group_score == PRISM_MOE_GROUP_MAX ||
                      router->group_score == PRISM_MOE_GROUP_TOP2,
                  "route_scored: unknown group_score %d", router->group_score);
  const int groups = router->num_groups, keep = router->topk_groups;
  PRISM_CHECK_ARG(groups >= 1 && groups <= 32 && num_experts % groups == 0,
                  "route_scored: num_groups %d outside [1, 32] or no divisor of %d experts", groups,
                  num_experts);
  PRISM_CHECK_ARG(keep >= 1 && keep <= groups, "route_scored: topk_groups %d outside [1, %d]", keep,
                  groups);
  PRISM_CHECK_ARG(top_k >= 1 && top_k <= 32 && top_k <= keep * (num_experts / groups),
                  "route_scored: top_k %d outside [1, min(32, %d experts of %d groups)]", top_k,
                  keep * (num_experts / groups), keep);
  PRISM_CHECK_ARG(num_tokens == 0 || (logits && topk_ids && topk_weights),
                  "route_scored: null pointer");
  if (int r = check_device()) return r;
  return route_scored(logits, dtype, num_tokens, num_experts, top_k, *router, topk_ids,
                      topk_weights, weights_dtype, expert_counts,
                      static_cast<cudaStream_t>(stream));
}

size_t prism_moe_dispatch_workspace_size(int64_t num_tokens, int32_t top_k, int32_t num_experts,
                                         int32_t ep_size) {
  if (num_tokens < 0 || top_k < 1 || num_experts < 1 || ep_size < 1) return 0;
  return dispatch_workspace_size(num_tokens * top_k, num_experts, ep_size);
}

int prism_moe_build_dispatch_plan(const int64_t* topk_ids, int64_t num_tokens, int32_t top_k,
                                  int32_t num_experts, int32_t ep_size, int64_t* perm,
                                  int64_t* input_splits, int64_t* sorted_local_eid,
                                  int32_t* expert_counts, int32_t* expert_offsets,
                                  int32_t* entry_row, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  PRISM_CHECK_ARG(num_tokens >= 0 && top_k >= 1 && top_k <= 32, "build_dispatch_plan: bad shape");
  PRISM_CHECK_ARG(ep_size >= 1 && num_experts >= 1 && num_experts % ep_size == 0,
                  "num_experts must be divisible by ep_size");
  PRISM_CHECK_ARG(num_tokens == 0 || (topk_ids && workspace), "build_dispatch_plan: null pointer");
  if (int r = check_device()) return r;
  return build_plan(topk_ids, num_tokens, top_k, num_experts, ep_size, perm, input_splits,
                    sorted_local_eid, expert_counts, expert_offsets, entry_row, nullptr,
                    workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int prism_moe_permute_rows(const void* x, int dtype, int64_t num_tokens, int64_t hidden,
                           int32_t top_k, const int32_t* entry_row, void* x_sorted, void* stream) {
  PRISM_CHECK_ARG(dtype_ok(dtype), "permute_rows: unknown dtype %d", dtype);
  PRISM_CHECK_ARG(num_tokens >= 0 && hidden >= 1, "permute_rows: bad shape");
  PRISM_CHECK_ARG(num_tokens == 0 || (x && entry_row && x_sorted), "permute_rows: null pointer");
  PRISM_CHECK_ARG((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(x_sorted)) % 16 == 0,
                  "permute_rows: buffers must be 16-byte aligned");
  if (int r = check_device()) return r;
  return permute_rows(x, num_tokens, hidden * elem_size(dtype), top_k, entry_row, x_sorted,
                      static_cast<cudaStream_t>(stream));
}

size_t prism_moe_expert_workspace_size(int64_t rows_capacity, int64_t hidden, int64_t inter,
                                       int dtype) {
  (void)hidden;
  if (rows_capacity < 0 || inter < 1 || !dtype_ok(dtype)) return 0;
  return expert_scratch_bytes(rows_capacity, inter, elem_size(dtype));
}

int prism_moe_expert_swiglu(const void* x_sorted, int dtype, int64_t rows_capacity,
                            int64_t hidden, int64_t inter, const int32_t* seg_offsets,
                            const int32_t* seg_expert, int32_t num_segments,
                            int32_t num_local_experts, const void* w_gate_up, const void* w_down,
                            void* y, void* workspace, size_t workspace_bytes, int* device_error,
                            void* stream) {
  PRISM_CHECK_ARG(dtype_ok(dtype), "expert_swiglu: unknown dtype %d", dtype);
  PRISM_CHECK_ARG(rows_capacity >= 0 && hidden >= 1 && inter >= 1, "expert_swiglu: bad shape");
  PRISM_CHECK_ARG(num_segments >= 1 && num_local_experts >= 1, "expert_swiglu: no segments");
  PRISM_CHECK_ARG(workspace_bytes >= prism_moe_expert_workspace_size(rows_capacity, hidden, inter, dtype),
                  "expert_swiglu: workspace too small");
  PRISM_CHECK_ARG(rows_capacity == 0 || (x_sorted && seg_offsets && w_gate_up && w_down && y && workspace),
                  "expert_swiglu: null pointer");
  if (int r = check_device()) return r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows_capacity == 0) return PRISM_MOE_OK;
  if (dtype == PRISM_MOE_BF16)
    return expert_swiglu_bf16(x_sorted, rows_capacity, hidden, inter, seg_offsets, seg_expert,
                              num_segments, num_local_experts, w_gate_up, w_down, y, workspace,
                              device_error, st);
  return expert_swiglu_f32(static_cast<const float*>(x_sorted), rows_capacity, hidden, inter,
                           seg_offsets, seg_expert, num_segments, num_local_experts,
                           static_cast<const float*>(w_gate_up), static_cast<const float*>(w_down),
                           static_cast<float*>(y), static_cast<float*>(workspace), st);
}

int prism_moe_linear_w4(const void* x, int64_t rows, int64_t in_features, int64_t out_features,
                        const prism_moe_w4* weight, void* y, int* device_error, void* stream) {
  PRISM_CHECK_ARG(rows >= 0 && in_features >= 1 && out_features >= 1, "linear_w4: bad shape");
  PRISM_CHECK_ARG(rows < (int64_t(1) << 31), "linear_w4: too many rows");
  if (int r = check_w4("linear_w4", weight, in_features, out_features)) return r;
  PRISM_CHECK_ARG(rows == 0 || (x && y), "linear_w4: null pointer");
  PRISM_CHECK_ARG((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % 16 == 0,
                  "linear_w4: buffers must be 16-byte aligned");
  const uintptr_t x0 = reinterpret_cast<uintptr_t>(x), y0 = reinterpret_cast<uintptr_t>(y);
  PRISM_CHECK_ARG(x0 + 2 * rows * in_features <= y0 || y0 + 2 * rows * out_features <= x0 || rows == 0,
                  "linear_w4: y overlaps x");
  if (int r = check_device()) return r;
  if (rows == 0) return PRISM_MOE_OK;
  W4Problem p;
  p.x = x;
  p.rows_cap = rows;
  p.K = in_features;
  p.n_out = out_features;
  p.w = *weight;
  p.out = y;
  p.err = device_error;
  return w4_product(p, static_cast<cudaStream_t>(stream));
}

size_t prism_moe_expert_w4_workspace_size(int64_t rows_capacity, int64_t inter) {
  if (rows_capacity < 0 || inter < 1) return 0;
  return w4_scratch_bytes(rows_capacity, inter);
}

int prism_moe_expert_swiglu_w4(const void* x_sorted, int64_t rows_capacity, int64_t hidden,
                               int64_t inter, const int32_t* seg_offsets,
                               const int32_t* seg_expert, int32_t num_segments,
                               int32_t num_local_experts, const prism_moe_w4* w_gate_up,
                               const prism_moe_w4* w_down, void* y, void* workspace,
                               size_t workspace_bytes, int* device_error, void* stream) {
  PRISM_CHECK_ARG(rows_capacity >= 0 && hidden >= 1 && inter >= 1, "expert_swiglu_w4: bad shape");
  PRISM_CHECK_ARG(rows_capacity < (int64_t(1) << 31), "expert_swiglu_w4: rows_capacity too large");
  PRISM_CHECK_ARG(num_segments >= 1 && num_segments <= kMaxW4Segments,
                  "expert_swiglu_w4: segments %d outside [1, %d]", num_segments, kMaxW4Segments);
  PRISM_CHECK_ARG(num_local_experts >= 1, "expert_swiglu_w4: no experts");
  if (int r = check_w4("expert_swiglu_w4", w_gate_up, hidden, 2 * inter)) return r;
  if (int r = check_w4("expert_swiglu_w4", w_down, inter, hidden)) return r;
  PRISM_CHECK_ARG(workspace_bytes >= w4_scratch_bytes(rows_capacity, inter),
                  "expert_swiglu_w4: workspace too small");
  PRISM_CHECK_ARG(rows_capacity == 0 || (x_sorted && y && workspace),
                  "expert_swiglu_w4: null pointer");
  PRISM_CHECK_ARG(seg_offsets || num_segments == 1,
                  "expert_swiglu_w4: without seg_offsets all rows are one segment, not %d",
                  num_segments);
  PRISM_CHECK_ARG((reinterpret_cast<uintptr_t>(x_sorted) | reinterpret_cast<uintptr_t>(y) |
                   reinterpret_cast<uintptr_t>(workspace)) % 16 == 0,
                  "expert_swiglu_w4: buffers must be 16-byte aligned");
  if (int r = check_device()) return r;
  if (rows_capacity == 0) return PRISM_MOE_OK;
  return expert_swiglu_w4(x_sorted, rows_capacity, hidden, inter, seg_offsets, seg_expert,
                          num_segments, num_local_experts, *w_gate_up, *w_down, y, workspace,
                          device_error, static_cast<cudaStream_t>(stream));
}

int prism_moe_combine(const void* expert_out, int dtype, const int32_t* entry_row,
                      const void* topk_weights, int64_t num_tokens, int32_t top_k, int64_t hidden,
                      void* out, void* stream) {
  PRISM_CHECK_ARG(dtype_ok(dtype), "combine: unknown dtype %d", dtype);
  PRISM_CHECK_ARG(num_tokens >= 0 && hidden >= 1, "combine: bad shape");
  PRISM_CHECK_ARG(num_tokens == 0 || (expert_out && topk_weights && out), "combine: null pointer");
  PRISM_CHECK_ARG((reinterpret_cast<uintptr_t>(expert_out) | reinterpret_cast<uintptr_t>(out)) % 16 == 0,
                  "combine: buffers must be 16-byte aligned");
  if (int r = check_device()) return r;
  return combine(expert_out, dtype, entry_row, topk_weights, num_tokens, top_k, hidden, out,
                 static_cast<cudaStream_t>(stream));
}

size_t prism_moe_block_workspace_size(int64_t num_tokens, int64_t hidden, int64_t inter,
                                      int32_t num_experts, int32_t top_k, int dtype) {
  if (num_tokens < 0 || hidden < 1 || inter < 1 || num_experts < 1 || top_k < 1 || !dtype_ok(dtype))
    return 0;
  return block_layout(num_tokens, hidden, inter, num_experts, top_k, dtype).total;
}

int prism_moe_block_forward_norm(const void* x, const void* router_logits, int dtype,
                                 int64_t num_tokens, int64_t hidden, int64_t inter,
                                 int32_t num_experts, int32_t top_k, int32_t renorm,
                                 const void* w_gate_up, const void* w_down, void* out,
                                 int64_t* topk_ids, void* topk_weights, void* workspace,
                                 size_t workspace_bytes, void* stream,
                                 const prism_moe_norm_epilogue* epilogue) {
  PRISM_CHECK_ARG(dtype_ok(dtype), "block_forward: unknown dtype %d", dtype);
  PRISM_CHECK_ARG(num_tokens >= 0 && hidden >= 1 && inter >= 1, "block_forward: bad shape");
  PRISM_CHECK_ARG(num_experts >= 1 && num_experts <= 1024, "block_forward: num_experts %d outside [1, 1024]",
                  num_experts);
  PRISM_CHECK_ARG(top_k >= 1 && top_k <= 32 && top_k <= num_experts,
                  "block_forward: top_k %d outside [1, min(num_experts, 32)]", top_k);
  const BlockLayout L = block_layout(num_tokens, hidden, inter, num_experts, top_k, dtype);
  PRISM_CHECK_ARG(workspace && workspace_bytes >= L.total,
                  "block_forward: workspace too small (%zu < %zu)", workspace_bytes, L.total);
  PRISM_CHECK_ARG(num_tokens == 0 || (x && router_logits && w_gate_up && w_down && out),
                  "block_forward: null pointer");
  PRISM_CHECK_ARG(!epilogue || (epilogue->residual && epilogue->norm_weight &&
                                epilogue->residual_out && epilogue->eps >= 0.f),
                  "block_forward: incomplete norm epilogue");
  if (int r = check_block_buffers("block_forward", x, out, workspace, epilogue)) return r;
  if (int r = check_device()) return r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (num_tokens == 0) return PRISM_MOE_OK;
  char* ws = static_cast<char*>(workspace);
  int64_t* ids = topk_ids ? topk_ids : reinterpret_cast<int64_t*>(ws + L.ids);
  void* w = topk_weights ? topk_weights : static_cast<void*>(ws + L.w);
  record_stage(0, st);
  int r = route_topk(router_logits, dtype, num_tokens, num_experts, top_k, renorm, ids, w, nullptr, st);
  if (r) return r;
  return block_after_router(x, ids, w, dtype, num_tokens, hidden, inter, num_experts, top_k,
                            w_gate_up, w_down, nullptr, nullptr, out, ws, L, nullptr, epilogue, st);
}

int prism_moe_block_forward_routed(const void* x, const int64_t* topk_ids,
                                   const void* topk_weights, int dtype, int64_t num_tokens,
                                   int64_t hidden, int64_t inter, int32_t num_experts,
                                   int32_t top_k, const void* w_gate_up, const void* w_down,
                                   const prism_moe_w4* q_gate_up, const prism_moe_w4* q_down,
                                   void* out, void* workspace, size_t workspace_bytes,
                                   void* stream, const prism_moe_norm_epilogue* epilogue) {
  return prism_moe_block_forward_routed_reporting(x, topk_ids, topk_weights, dtype, num_tokens, hidden,
                                                  inter, num_experts, top_k, w_gate_up, w_down,
                                                  q_gate_up, q_down, out, workspace, workspace_bytes,
                                                  nullptr, stream, epilogue);
}

int prism_moe_block_forward_routed_reporting(
    const void* x, const int64_t* topk_ids, const void* topk_weights, int dtype, int64_t num_tokens,
    int64_t hidden, int64_t inter, int32_t num_experts, int32_t top_k, const void* w_gate_up,
    const void* w_down, const prism_moe_w4* q_gate_up, const prism_moe_w4* q_down, void* out,
    void* workspace, size_t workspace_bytes, int* device_error, void* stream,
    const prism_moe_norm_epilogue* epilogue) {
  PRISM_CHECK_ARG(dtype_ok(dtype), "block_forward_routed: unknown dtype %d", dtype);
  PRISM_CHECK_ARG(num_tokens >= 0 && hidden >= 1 && inter >= 1, "block_forward_routed: bad shape");
  PRISM_CHECK_ARG(num_experts >= 1 && num_experts <= 1024,
                  "block_forward_routed: num_experts %d outside [1, 1024]", num_experts);
  PRISM_CHECK_ARG(top_k >= 1 && top_k <= 32 && top_k <= num_experts,
                  "block_forward_routed: top_k %d outside [1, min(num_experts, 32)]", top_k);
  const bool w4 = q_gate_up || q_down;
  PRISM_CHECK_ARG(w4 ? (!w_gate_up && !w_down) : (w_gate_up && w_down),
                  "block_forward_routed: give either dense or 4-bit expert weights");
  if (w4) {
    PRISM_CHECK_ARG(dtype == PRISM_MOE_BF16,
                    "block_forward_routed: 4-bit experts take bf16 activations");
    if (int r = check_w4("block_forward_routed", q_gate_up, hidden, 2 * inter)) return r;
    if (int r = check_w4("block_forward_routed", q_down, inter, hidden)) return r;
  }
  const BlockLayout L = block_layout(num_tokens, hidden, inter, num_experts, top_k, dtype);
  PRISM_CHECK_ARG(workspace && workspace_bytes >= L.total,
                  "block_forward_routed: workspace too small (%zu < %zu)", workspace_bytes, L.total);
  PRISM_CHECK_ARG(num_tokens == 0 || (x && topk_ids && topk_weights && out),
                  "block_forward_routed: null pointer");
  PRISM_CHECK_ARG(!epilogue || (epilogue->residual && epilogue->norm_weight &&
                                epilogue->residual_out && epilogue->eps >= 0.f),
                  "block_forward_routed: incomplete norm epilogue");
  if (int r = check_block_buffers("block_forward_routed", x, out, workspace, epilogue)) return r;
  if (int r = check_device()) return r;
  if (num_tokens == 0) return PRISM_MOE_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  record_stage(0, st);
  return block_after_router(x, topk_ids, topk_weights, dtype, num_tokens, hidden, inter,
                            num_experts, top_k, w_gate_up, w_down, q_gate_up, q_down, out,
                            static_cast<char*>(workspace), L, device_error, epilogue, st);
}

int prism_moe_block_forward(const void* x, const void* router_logits, int dtype,
                            int64_t num_tokens, int64_t hidden, int64_t inter,
                            int32_t num_experts, int32_t top_k, int32_t renorm,
                            const void* w_gate_up, const void* w_down, void* out,
                            int64_t* topk_ids, void* topk_weights, void* workspace,
                            size_t workspace_bytes, void* stream) {
  return prism_moe_block_forward_norm(x, router_logits, dtype, num_tokens, hidden, inter,
                                      num_experts, top_k, renorm, w_gate_up, w_down, out,
                                      topk_ids, topk_weights, workspace, workspace_bytes, stream,
                                      nullptr);
}

int prism_moe_rmsnorm(const void* x, const void* residual, const void* weight, float eps,
                      int dtype, int64_t num_tokens, int64_t hidden, void* out,
                      void* residual_out, void* stream) {
  PRISM_CHECK_ARG(dtype_ok(dtype), "rmsnorm: unknown dtype %d", dtype);
  PRISM_CHECK_ARG(num_tokens >= 0 && hidden >= 1, "rmsnorm: bad shape");
  PRISM_CHECK_ARG(eps >= 0.f, "rmsnorm: negative eps");
  PRISM_CHECK_ARG(num_tokens == 0 || (x && weight && out), "rmsnorm: null pointer");
  PRISM_CHECK_ARG((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                   reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(out) |
                   reinterpret_cast<uintptr_t>(residual_out)) % 16 == 0,
                  "rmsnorm: buffers must be 16-byte aligned");
  if (int r = check_device()) return r;
  return rmsnorm(x, residual, weight, eps, dtype, num_tokens, hidden, out, residual_out,
                 static_cast<cudaStream_t>(stream));
}

int prism_moe_profile_events(void* const* events, int32_t count) {
  PRISM_CHECK_ARG(count >= 0 && count <= kNumStageEvents, "profile_events: count %d outside [0, %d]",
                  count, kNumStageEvents);
  PRISM_CHECK_ARG(count == 0 || events != nullptr, "profile_events: null events");
  for (int i = 0; i < kNumStageEvents; ++i)
    g_stage_events[i] = i < count ? static_cast<cudaEvent_t>(events[i]) : nullptr;
  g_num_stage_events = count;
  return PRISM_MOE_OK;
}

int prism_moe_set_expert_engine(int engine) {
  PRISM_CHECK_ARG(engine >= PRISM_MOE_ENGINE_AUTO && engine <= PRISM_MOE_ENGINE_PAIR,
                  "set_expert_engine: unknown engine %d", engine);
  g_engine.store(engine, std::memory_order_relaxed);
  return PRISM_MOE_OK;
}

int prism_moe_set_wait_limits(int64_t wait_ns, int64_t peer_wait_ns) {
  PRISM_CHECK_ARG(wait_ns >= 0 && peer_wait_ns >= 0, "set_wait_limits: negative limit");
  PRISM_CHECK_ARG(wait_ns <= 60000000000ll && peer_wait_ns <= 60000000000ll,
                  "set_wait_limits: limits above 60 s are not accepted");
  g_wait_ns.store(wait_ns > 0 ? static_cast<uint64_t>(wait_ns) : 2000000000ull,
                  std::memory_order_relaxed);
  g_peer_wait_ns.store(peer_wait_ns > 0 ? static_cast<uint64_t>(peer_wait_ns) : 10000000000ull,
                       std::memory_order_relaxed);
  return PRISM_MOE_OK;
}

int prism_moe_device_error_word(int** word) {
  PRISM_CHECK_ARG(word != nullptr, "device_error_word: null pointer");
  if (int r = check_device()) return r;
  void* at = nullptr;
  PRISM_CUDA(cudaGetSymbolAddress(&at, g_device_error));
  *word = static_cast<int*>(at);
  return PRISM_MOE_OK;
}

int prism_moe_read_device_error(int* device_error, void* stream) {
  PRISM_CHECK_ARG(device_error != nullptr, "read_device_error: null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int v = 0;
  PRISM_CUDA(cudaMemcpyAsync(&v, device_error, sizeof(int), cudaMemcpyDeviceToHost, st));
  PRISM_CUDA(cudaStreamSynchronize(st));
  if (v != 0) {
    PRISM_CUDA(cudaMemsetAsync(device_error, 0, sizeof(int), st));
    PRISM_CUDA(cudaStreamSynchronize(st));
    set_error("a kernel recorded device status %d", v);
    return v;
  }
  return PRISM_MOE_OK;
}

}  // extern "C"
