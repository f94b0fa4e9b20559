// Thin torch extension over the C ABI (include/cwarp_rnnt_b200.h): the replacement of the reference's cwarp_cuda.cpp.
// It owns tensors, the device guard and the current stream; all arithmetic lives in libcwarp_rnnt_b200.so.
//
// Exports the reference module's three functions with the reference's argument order and result shapes
// (cwarp_cuda.cpp:138-153) for callers of `cwarp_rnnt._C`, plus the fused entry points the autograd function uses.
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "cwarp_rnnt_b200.h"

namespace {

// Same wording as the reference's checks (cwarp_cuda.cpp:46-52).
#define CHECK_CUDA(x) TORCH_CHECK(x.device().is_cuda(), #x " must be a CUDA tensor")
#define CHECK_CONTIGUOUS(x) TORCH_CHECK(x.is_contiguous(), #x " must be contiguous")
#define CHECK_TYPE(x, T) TORCH_CHECK(x.scalar_type() == T, #x " must be " #T)
#define CHECK_INPUT(x, T) \
    CHECK_CUDA(x);        \
    CHECK_CONTIGUOUS(x);  \
    CHECK_TYPE(x, T)

int dtype_code(const torch::Tensor &x)
{
    switch (x.scalar_type()) {
    case torch::ScalarType::Float: return CWRNNT_F32;
    case torch::ScalarType::Half: return CWRNNT_F16;
    case torch::ScalarType::BFloat16: return CWRNNT_BF16;
    case torch::ScalarType::Double: return CWRNNT_F64;
    default: TORCH_CHECK(false, "xs must be float32, float16, bfloat16 or float64, got ", x.scalar_type());
    }
    return -1;
}

torch::ScalarType cost_type(const torch::Tensor &x)
{
    return x.scalar_type() == torch::ScalarType::Double ? torch::ScalarType::Double : torch::ScalarType::Float;
}

void check_status(int st, const char *what)
{
    if (st == CWRNNT_OK) return;
    std::string msg = std::string(what) + ": " + cwrnnt_status_string(st);
    if (st == CWRNNT_ERR_LAUNCH) msg += std::string(" (") + cwrnnt_last_error() + ")";
    TORCH_CHECK(false, msg);
}

cwrnnt_problem describe(const torch::Tensor &xs, const torch::Tensor &lx, const torch::Tensor &ys, int64_t blank,
                        int64_t flags, int64_t mean_denominator)
{
    TORCH_CHECK(xs.dim() == 2, "xs must be 2-D [sum_i T_i*(U_i+1), V]");
    TORCH_CHECK(ys.dim() == 2 && ys.size(0) == lx.size(0), "ys must be [N, Umax]");
    cwrnnt_problem p{};
    p.n_rows = xs.size(0);
    p.V = static_cast<int32_t>(xs.size(1));
    p.B = static_cast<int32_t>(lx.size(0));
    p.y_stride = static_cast<int32_t>(ys.size(1));
    p.max_u = static_cast<int32_t>(ys.size(1));
    p.blank = static_cast<int32_t>(blank);
    p.dtype = dtype_code(xs);
    p.flags = static_cast<int32_t>(flags);
    p.mean_denominator = static_cast<int32_t>(mean_denominator);
    return p;
}

void check_inputs(const torch::Tensor &xs, const torch::Tensor &lx, const torch::Tensor &ys, const torch::Tensor &ly)
{
    CHECK_CONTIGUOUS(xs);
    CHECK_CUDA(xs);
    CHECK_INPUT(lx, torch::ScalarType::Int);
    CHECK_INPUT(ys, torch::ScalarType::Int);
    CHECK_INPUT(ly, torch::ScalarType::Int);
    TORCH_CHECK(lx.device() == xs.device() && ly.device() == xs.device() && ys.device() == xs.device(),
                "xs, lx, ys, ly must live on the same device");
    TORCH_CHECK(lx.dim() == 1 && ly.dim() == 1 && lx.size(0) == ly.size(0), "lx and ly must be [N]");
}

torch::Tensor make_workspace(const cwrnnt_problem &p, const torch::Tensor &like)
{
    const int64_t bytes = cwrnnt_workspace_bytes(&p);
    TORCH_CHECK(bytes >= 0, "invalid problem: check blank in [0,V), label length <= ", CWRNNT_MAX_COLUMNS - 1);
    return torch::empty({bytes}, like.options().dtype(torch::kUInt8));
}

cwrnnt_stream_t current_stream()
{
    return reinterpret_cast<cwrnnt_stream_t>(at::cuda::getCurrentCUDAStream().stream());
}

const int32_t *i32(const torch::Tensor &t) { return t.numel() ? t.data_ptr<int32_t>() : nullptr; }

// ---------------------------------------------------------------------------------------------- fused entry points

// Forward. Returns (costs [N], loss [] (zero unless a reduce flag is set), workspace bytes).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> rnnt_forward(const torch::Tensor &xs, const torch::Tensor &lx,
                                                                     const torch::Tensor &ys, const torch::Tensor &ly,
                                                                     int64_t blank, int64_t flags,
                                                                     int64_t mean_denominator)
{
    check_inputs(xs, lx, ys, ly);
    const c10::cuda::CUDAGuard guard(xs.device());
    cwrnnt_problem p = describe(xs, lx, ys, blank, flags, mean_denominator);
    auto ws = make_workspace(p, xs);
    auto costs = torch::empty({lx.size(0)}, xs.options().dtype(cost_type(xs)));
    // written by the kernels whenever a reduction is asked for on a non-empty batch (NaN on invalid lengths)
    auto loss = ((flags & (CWRNNT_REDUCE_MEAN | CWRNNT_REDUCE_SUM)) && lx.size(0) > 0) ? torch::empty({}, costs.options())
                                                                   : torch::zeros({}, costs.options());
    check_status(cwrnnt_forward(&p, xs.data_ptr(), i32(lx), i32(ly), i32(ys), ws.data_ptr(), ws.numel(),
                                costs.data_ptr(), loss.data_ptr(), current_stream()),
                 "cwrnnt_forward");
    return {costs, loss, ws};
}

// Backward. grad_costs: [] or [1] (gradient of the reduced loss) or [N] (per-sequence), costs dtype.
torch::Tensor rnnt_backward(const torch::Tensor &xs, const torch::Tensor &lx, const torch::Tensor &ys,
                            const torch::Tensor &ly, int64_t blank, int64_t flags, int64_t mean_denominator,
                            const torch::Tensor &workspace, const torch::Tensor &grad_costs)
{
    check_inputs(xs, lx, ys, ly);
    CHECK_CUDA(grad_costs);
    const c10::cuda::CUDAGuard guard(xs.device());
    cwrnnt_problem p = describe(xs, lx, ys, blank, flags, mean_denominator);
    auto gc = grad_costs.to(cost_type(xs)).contiguous();
    TORCH_CHECK(gc.numel() == 1 || gc.numel() == lx.size(0), "grad_costs must have 1 or N elements");
    auto gx = torch::empty_like(xs);
    check_status(cwrnnt_backward(&p, xs.data_ptr(), i32(lx), i32(ly), i32(ys), workspace.data_ptr(), gc.data_ptr(),
                                 gc.numel() == 1 ? 0 : 1, gx.data_ptr(), current_stream()),
                 "cwrnnt_backward");
    return gx;
}

// Side streams of the pipelined step: one set per device and host thread (a pipe serves one call at a time), created
// on first use and kept for the life of the thread's process.
cwrnnt_pipe *pipe_of(int device_index)
{
    static thread_local std::vector<cwrnnt_pipe *> pipes;
    if (device_index >= static_cast<int>(pipes.size())) pipes.resize(device_index + 1, nullptr);
    if (!pipes[device_index]) check_status(cwrnnt_pipe_create(&pipes[device_index]), "cwrnnt_pipe_create");
    return pipes[device_index];
}

// Forward and gradient in one pipelined call, for an upstream gradient of 1 (scaled later by rnnt_scale_grad if the
// real one differs). Returns (costs [N], loss [], workspace bytes, grad_x like xs).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>
rnnt_loss_grad(const torch::Tensor &xs, const torch::Tensor &lx, const torch::Tensor &ys, const torch::Tensor &ly,
               int64_t blank, int64_t flags, int64_t mean_denominator, int64_t groups)
{
    check_inputs(xs, lx, ys, ly);
    const c10::cuda::CUDAGuard guard(xs.device());
    cwrnnt_problem p = describe(xs, lx, ys, blank, flags, mean_denominator);
    auto ws = make_workspace(p, xs);
    auto costs = torch::empty({lx.size(0)}, xs.options().dtype(cost_type(xs)));
    // written by the kernels whenever a reduction is asked for on a non-empty batch (NaN on invalid lengths)
    auto loss = ((flags & (CWRNNT_REDUCE_MEAN | CWRNNT_REDUCE_SUM)) && lx.size(0) > 0) ? torch::empty({}, costs.options())
                                                                   : torch::zeros({}, costs.options());
    auto gx = torch::empty_like(xs);
    check_status(cwrnnt_loss_grad(pipe_of(xs.get_device()), &p, xs.data_ptr(), i32(lx), i32(ly), i32(ys),
                                  ws.data_ptr(), ws.numel(), costs.data_ptr(), loss.data_ptr(), nullptr, 0,
                                  gx.data_ptr(), nullptr, 0, nullptr, static_cast<int32_t>(groups), current_stream()),
                 "cwrnnt_loss_grad");
    return {costs, loss, ws, gx};
}

// grad_x *= factor in place; factor holds one element of the costs dtype on the same device.
void rnnt_scale_grad(torch::Tensor grad_x, const torch::Tensor &factor)
{
    CHECK_CONTIGUOUS(grad_x);
    CHECK_CUDA(grad_x);
    CHECK_CUDA(factor);
    TORCH_CHECK(grad_x.dim() == 2 && factor.numel() == 1, "grad_x must be 2-D and factor a single element");
    const c10::cuda::CUDAGuard guard(grad_x.device());
    cwrnnt_problem p{};
    p.n_rows = grad_x.size(0);
    p.V = static_cast<int32_t>(grad_x.size(1));
    p.dtype = dtype_code(grad_x);
    auto f = factor.to(cost_type(grad_x)).contiguous();
    check_status(cwrnnt_scale_grad(&p, grad_x.data_ptr(), f.data_ptr(), current_stream()), "cwrnnt_scale_grad");
}

// Input validation ahead of the heavy kernels: [status bits, first bad sequence, max(lx), max(ly)]; one short sync.
std::vector<int64_t> rnnt_validate(const torch::Tensor &lx, const torch::Tensor &ys, const torch::Tensor &ly,
                                   int64_t n_rows, int64_t V)
{
    CHECK_INPUT(lx, torch::ScalarType::Int);
    CHECK_INPUT(ys, torch::ScalarType::Int);
    CHECK_INPUT(ly, torch::ScalarType::Int);
    TORCH_CHECK(ys.dim() == 2 && ys.size(0) == lx.size(0) && ly.size(0) == lx.size(0), "ys must be [N, Umax]");
    const c10::cuda::CUDAGuard guard(lx.device());
    cwrnnt_problem p{};
    p.n_rows = n_rows;
    p.V = static_cast<int32_t>(V);
    p.B = static_cast<int32_t>(lx.size(0));
    p.y_stride = p.max_u = static_cast<int32_t>(ys.size(1));
    auto scratch = torch::empty({4}, lx.options());
    int32_t st[4] = {0, 0, 0, 0};
    check_status(cwrnnt_validate(&p, i32(lx), i32(ly), i32(ys), scratch.data_ptr(), st, current_stream()),
                 "cwrnnt_validate");
    return {st[0], st[1], st[2], st[3]};
}

// The same validation queued without waiting: returns the four words as a pinned host tensor that is filled once the
// current stream has passed this point. The caller records an event, queues the loss kernels, then waits on the event.
torch::Tensor rnnt_validate_begin(const torch::Tensor &lx, const torch::Tensor &ys, const torch::Tensor &ly,
                                  int64_t n_rows, int64_t V)
{
    CHECK_INPUT(lx, torch::ScalarType::Int);
    CHECK_INPUT(ys, torch::ScalarType::Int);
    CHECK_INPUT(ly, torch::ScalarType::Int);
    TORCH_CHECK(ys.dim() == 2 && ys.size(0) == lx.size(0) && ly.size(0) == lx.size(0), "ys must be [N, Umax]");
    const c10::cuda::CUDAGuard guard(lx.device());
    cwrnnt_problem p{};
    p.n_rows = n_rows;
    p.V = static_cast<int32_t>(V);
    p.B = static_cast<int32_t>(lx.size(0));
    p.y_stride = p.max_u = static_cast<int32_t>(ys.size(1));
    auto scratch = torch::empty({4}, lx.options());  // freed stream-ordered by the caching allocator
    auto out = torch::empty({4}, torch::TensorOptions().dtype(torch::kInt32).pinned_memory(true));
    check_status(cwrnnt_validate_async(&p, i32(lx), i32(ly), i32(ys), scratch.data_ptr(), out.data_ptr<int32_t>(),
                                       current_stream()),
                 "cwrnnt_validate_async");
    return out;
}

// Device status words of a workspace: synchronises the current stream. [bits, first bad sequence, rows, 0].
std::vector<int64_t> rnnt_status(const torch::Tensor &workspace)
{
    CHECK_CUDA(workspace);
    const c10::cuda::CUDAGuard guard(workspace.device());
    int32_t st[4] = {0, 0, 0, 0};
    check_status(cwrnnt_read_status(workspace.data_ptr(), st, current_stream()), "cwrnnt_read_status");
    return {st[0], st[1], st[2], st[3]};
}

// Padded [N, T, U+1, V] -> compact [n_rows, V] (n_rows = sum T_n*(U_n+1), computed by the caller) and back.
torch::Tensor pack_padded(const torch::Tensor &padded, const torch::Tensor &lx, const torch::Tensor &ly,
                          int64_t n_rows)
{
    CHECK_CUDA(padded);
    CHECK_CONTIGUOUS(padded);
    CHECK_INPUT(lx, torch::ScalarType::Int);
    CHECK_INPUT(ly, torch::ScalarType::Int);
    TORCH_CHECK(padded.dim() == 4 && padded.size(0) == lx.size(0), "padded must be [N, T, U+1, V]");
    const c10::cuda::CUDAGuard guard(padded.device());
    cwrnnt_problem p{};
    p.n_rows = n_rows;
    p.V = static_cast<int32_t>(padded.size(3));
    p.B = static_cast<int32_t>(padded.size(0));
    p.y_stride = p.max_u = static_cast<int32_t>(padded.size(2) - 1);
    p.dtype = dtype_code(padded);
    auto scratch = torch::empty({cwrnnt_scatter_scratch_bytes(p.B)}, padded.options().dtype(torch::kUInt8));
    auto out = torch::empty({n_rows, padded.size(3)}, padded.options());
    check_status(cwrnnt_pack_padded(&p, padded.data_ptr(), static_cast<int32_t>(padded.size(1)),
                                    static_cast<int32_t>(padded.size(2)), i32(lx), i32(ly), scratch.data_ptr(),
                                    scratch.numel(), out.data_ptr(), current_stream()),
                 "cwrnnt_pack_padded");
    return out;
}

torch::Tensor unpack_padded(const torch::Tensor &compact, const torch::Tensor &lx, const torch::Tensor &ly,
                            int64_t T, int64_t Up)
{
    CHECK_CUDA(compact);
    CHECK_INPUT(lx, torch::ScalarType::Int);
    CHECK_INPUT(ly, torch::ScalarType::Int);
    TORCH_CHECK(compact.dim() == 2, "compact must be [n_rows, V]");
    const c10::cuda::CUDAGuard guard(compact.device());
    auto c = compact.contiguous();
    cwrnnt_problem p{};
    p.n_rows = c.size(0);
    p.V = static_cast<int32_t>(c.size(1));
    p.B = static_cast<int32_t>(lx.size(0));
    p.y_stride = p.max_u = static_cast<int32_t>(Up - 1);
    p.dtype = dtype_code(c);
    auto scratch = torch::empty({cwrnnt_scatter_scratch_bytes(p.B)}, c.options().dtype(torch::kUInt8));
    auto out = torch::empty({lx.size(0), T, Up, c.size(1)}, c.options());
    check_status(cwrnnt_unpack_padded(&p, c.data_ptr(), static_cast<int32_t>(T), static_cast<int32_t>(Up), i32(lx),
                                      i32(ly), scratch.data_ptr(), scratch.numel(), out.data_ptr(), current_stream()),
                 "cwrnnt_unpack_padded");
    return out;
}

// -------------------------------------------------------------------------------------- operators on rows of logits

using OptTensor = std::optional<torch::Tensor>;

void *ptr(const OptTensor &t) { return t && t->numel() ? t->data_ptr() : nullptr; }

// x [rows, V] with unit column stride; rows may lie further apart.
cwrnnt_rows describe_rows(const torch::Tensor &x, int64_t n_list, int64_t top_k, double temperature)
{
    CHECK_CUDA(x);
    TORCH_CHECK(x.dim() == 2 && x.size(1) >= 1, "x must be [rows, V] with at least one column");
    TORCH_CHECK(x.size(1) == 1 || x.stride(1) == 1, "x must have unit stride along its columns");
    TORCH_CHECK(x.size(1) <= INT32_MAX - 64, "too many columns");
    TORCH_CHECK(x.size(0) < 2 || x.stride(0) >= x.size(1), "rows of x overlap");
    TORCH_CHECK(n_list <= CWRNNT_MAX_LIST && top_k <= CWRNNT_MAX_LIST, "at most ", CWRNNT_MAX_LIST,
                " targets, top entries or teacher entries of a row");
    TORCH_CHECK(top_k >= 0 && top_k <= x.size(1), "top_k must lie in [0, V]");
    cwrnnt_rows p{};
    p.n_rows = x.size(0);
    p.V = static_cast<int32_t>(x.size(1));
    p.x_stride = x.size(0) < 2 ? x.size(1) : x.stride(0);
    p.grad_stride = x.size(1);
    p.temperature = temperature;
    p.dtype = dtype_code(x);
    p.n_list = static_cast<int32_t>(n_list);
    p.top_k = static_cast<int32_t>(top_k);
    return p;
}

// [rows, n] int32 / costs-type companion of x on the same device, contiguous.
void check_companion(const torch::Tensor &t, const torch::Tensor &x, torch::ScalarType type, const char *name)
{
    TORCH_CHECK(t.device() == x.device(), name, " must live on the device of x");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.scalar_type() == type, name, " must be ", type);
    TORCH_CHECK(t.size(0) == x.size(0), name, " must have one row for each row of x");
}

// Returns (log_probs [R,P]?, entropy [R]?, top_log_probs [R,k]?, top_indices [R,k]?, stats [R,2]?).
std::tuple<OptTensor, OptTensor, OptTensor, OptTensor, OptTensor>
token_scores(const torch::Tensor &x, const OptTensor &targets, int64_t top_k, bool entropy, double temperature,
             bool keep)
{
    const cwrnnt_rows p = describe_rows(x, targets ? targets->size(1) : 0, top_k, temperature);
    if (targets) check_companion(*targets, x, torch::ScalarType::Int, "targets");
    const c10::cuda::CUDAGuard guard(x.device());
    const auto costs = x.options().dtype(cost_type(x));
    OptTensor lp, ent, top, index, stats;
    if (targets) lp = torch::empty({p.n_rows, p.n_list}, costs);
    if (entropy) ent = torch::empty({p.n_rows}, costs);
    if (top_k > 0) {
        top = torch::empty({p.n_rows, p.top_k}, costs);
        index = torch::empty({p.n_rows, p.top_k}, x.options().dtype(torch::kInt32));
    }
    if (keep) stats = torch::empty({p.n_rows, 2}, costs);
    check_status(cwrnnt_token_scores(&p, x.data_ptr(), static_cast<const int32_t *>(ptr(targets)), ptr(lp), ptr(ent),
                                     ptr(top), static_cast<int32_t *>(ptr(index)), ptr(stats),
                                     current_stream()),
                 "cwrnnt_token_scores");
    return {lp, ent, top, index, stats};
}

torch::Tensor token_scores_backward(const torch::Tensor &x, const OptTensor &targets, const OptTensor &index,
                                    const torch::Tensor &stats, const OptTensor &entropy, const OptTensor &g_lp,
                                    const OptTensor &g_ent, const OptTensor &g_top, double temperature)
{
    const cwrnnt_rows p = describe_rows(x, targets ? targets->size(1) : 0, index ? index->size(1) : 0, temperature);
    const c10::cuda::CUDAGuard guard(x.device());
    const auto type = cost_type(x);
    for (const OptTensor *t : {&g_lp, &g_ent, &g_top})
        if (*t) check_companion(**t, x, type, "an upstream gradient");
    auto gx = torch::empty({x.size(0), x.size(1)}, x.options());
    check_status(cwrnnt_token_scores_backward(&p, x.data_ptr(), static_cast<const int32_t *>(ptr(targets)),
                                              static_cast<const int32_t *>(ptr(index)), stats.data_ptr(),
                                              ptr(entropy), ptr(g_lp), ptr(g_ent), ptr(g_top), gx.data_ptr(),
                                              current_stream()),
                 "cwrnnt_token_scores_backward");
    return gx;
}

// Returns (row_loss [R]?, loss []?, grad_x [R,V]?). `made`: the gradient for an upstream gradient of 1, to be made anew in
// its place if that is something else.
std::tuple<OptTensor, OptTensor, OptTensor> distill(const torch::Tensor &x, const torch::Tensor &teacher,
                                                    const torch::Tensor &indices, const OptTensor &weight,
                                                    const OptTensor &upstream, bool tail, double temperature,
                                                    double scale, bool want_rows, bool want_loss, bool want_grad,
                                                    const OptTensor &made = {})
{
    TORCH_CHECK(teacher.dim() == 2 && indices.dim() == 2 && teacher.size(1) == indices.size(1) && indices.size(1) > 0,
                "teacher values and indices must both be [rows, K], K >= 1");
    const cwrnnt_rows p = describe_rows(x, indices.size(1), 0, temperature);
    const auto type = cost_type(x);
    check_companion(teacher, x, type, "teacher values");
    check_companion(indices, x, torch::ScalarType::Int, "indices");
    if (weight) check_companion(*weight, x, type, "weight");
    if (upstream)
        TORCH_CHECK(upstream->device() == x.device() && upstream->scalar_type() == type && upstream->is_contiguous() &&
                        (upstream->numel() == 1 || upstream->numel() == x.size(0)),
                    "an upstream gradient must have 1 or N elements");
    const c10::cuda::CUDAGuard guard(x.device());
    const auto costs = x.options().dtype(type);
    OptTensor rows, loss, gx, ws;
    if (want_rows) rows = torch::empty({p.n_rows}, costs);
    if (want_loss) {
        loss = torch::empty({}, costs);
        ws = torch::empty({cwrnnt_distill_workspace_bytes(&p)}, x.options().dtype(torch::kUInt8));
    }
    if (want_grad) gx = made ? *made : torch::empty({x.size(0), x.size(1)}, x.options());
    const int32_t stride = made ? CWRNNT_UPSTREAM_UNLESS_ONE : upstream && upstream->numel() > 1 ? 1 : 0;
    check_status(cwrnnt_distill(&p, tail ? 1 : 0, x.data_ptr(), teacher.data_ptr(),
                                static_cast<const int32_t *>(indices.data_ptr()), ptr(weight), ptr(upstream), stride, scale, ptr(ws), ws ? ws->numel() : 0,
                                ptr(rows), ptr(loss), ptr(gx), current_stream()),
                 "cwrnnt_distill");
    return {rows, loss, gx};
}

// ------------------------------------------------------------------------------------------------- linear layers

// A matrix with unit column stride as the C ABI reads it where it lies; copied where its rows overlap, or where TMA would
// have to start off a 16-byte boundary.
torch::Tensor readable(const torch::Tensor &m)
{
    const bool rows_ok = m.size(0) < 2 || m.stride(0) >= m.size(1);
    const bool columns_ok = m.size(1) < 2 || m.stride(1) == 1;
    const int64_t ld = m.size(0) < 2 ? m.size(1) : m.stride(0);
    if (!rows_ok || !columns_ok) return m.clone(torch::MemoryFormat::Contiguous);
    if (ld % 8 == 0 && reinterpret_cast<uintptr_t>(m.data_ptr()) % 16 != 0)
        return m.clone(torch::MemoryFormat::Contiguous);
    return m;
}
int64_t leading(const torch::Tensor &m) { return m.size(0) < 2 ? m.size(1) : m.stride(0); }

cwrnnt_linear describe_linear(const torch::Tensor &x, const torch::Tensor &weight, const OptTensor &bias,
                              int64_t activation)
{
    CHECK_CUDA(x);
    TORCH_CHECK(x.dim() == 2 && weight.dim() == 2 && x.size(1) == weight.size(1) && x.size(1) > 0 && weight.size(0) > 0,
                "x must be [rows, n_in] and weight [n_out, n_in]");
    TORCH_CHECK(x.scalar_type() == torch::ScalarType::Half || x.scalar_type() == torch::ScalarType::BFloat16,
                "x must be float16 or bfloat16, got ", x.scalar_type());
    TORCH_CHECK(weight.scalar_type() == x.scalar_type() && weight.device() == x.device(),
                "weight must have the type and device of x");
    TORCH_CHECK(x.size(1) <= (1 << 24) && weight.size(0) <= (1 << 24) && x.size(0) <= INT32_MAX - 1023,
                "a side of the product is too long");
    if (bias)
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0) && bias->scalar_type() == x.scalar_type() &&
                        bias->device() == x.device() && bias->is_contiguous(),
                    "bias must be [n_out], contiguous, of the type and device of x");
    cwrnnt_linear p{};
    p.n_rows = x.size(0);
    p.n_in = static_cast<int32_t>(x.size(1));
    p.n_out = static_cast<int32_t>(weight.size(0));
    p.x_stride = leading(x);
    p.w_stride = leading(weight);
    p.g_stride = weight.size(0);
    p.dtype = dtype_code(x);
    p.activation = static_cast<int32_t>(activation);
    return p;
}

torch::Tensor linear_forward(const torch::Tensor &x_, const torch::Tensor &weight_, const OptTensor &bias,
                             const OptTensor &residual_, int64_t activation)
{
    CHECK_CUDA(x_);
    CHECK_CUDA(weight_);
    TORCH_CHECK(x_.dim() == 2 && weight_.dim() == 2, "x must be [rows, n_in] and weight [n_out, n_in]");
    const c10::cuda::CUDAGuard guard(x_.device());
    const auto x = readable(x_), weight = readable(weight_);
    const cwrnnt_linear p = describe_linear(x, weight, bias, activation);
    OptTensor residual = residual_;
    if (residual && residual->dim() == 2) residual = readable(*residual);
    if (residual)
        TORCH_CHECK(residual->dim() == 2 && residual->size(0) == p.n_rows && residual->size(1) == p.n_out &&
                        residual->scalar_type() == x.scalar_type() && residual->device() == x.device() &&
                        residual->is_contiguous(),
                    "residual must be [rows, n_out], contiguous, of the type and device of x");
    const int64_t bytes = cwrnnt_linear_workspace_bytes(&p, residual ? CWRNNT_LINEAR_FORWARD_RESIDUAL : CWRNNT_LINEAR_FORWARD);
    TORCH_CHECK(bytes >= 0, "invalid linear layer");
    auto ws = torch::empty({bytes}, x.options().dtype(torch::kUInt8));
    auto y = torch::empty({x.size(0), weight.size(0)}, x.options());
    check_status(cwrnnt_linear_forward(&p, x.data_ptr(), weight.data_ptr(), ptr(bias), ptr(residual), ws.data_ptr(),
                                       bytes, y.data_ptr(), current_stream()),
                 "cwrnnt_linear_forward");
    return y;
}

// Returns (grad_x?, grad_weight?, grad_bias?).
std::tuple<OptTensor, OptTensor, OptTensor> linear_backward(const torch::Tensor &x_, const torch::Tensor &weight_,
                                                            const OptTensor &bias, const torch::Tensor &grad_y,
                                                            int64_t activation, bool want_x, bool want_weight,
                                                            bool want_bias)
{
    CHECK_CUDA(x_);
    const c10::cuda::CUDAGuard guard(x_.device());
    const auto x = readable(x_), weight = readable(weight_), g = readable(grad_y);
    cwrnnt_linear p = describe_linear(x, weight, bias, activation);
    TORCH_CHECK(g.dim() == 2 && g.size(0) == p.n_rows && g.size(1) == p.n_out && g.scalar_type() == x.scalar_type() &&
                    g.device() == x.device(),
                "the upstream gradient must be [rows, n_out], of the type and device of x");
    p.g_stride = leading(g);
    const int64_t bytes = cwrnnt_linear_workspace_bytes(&p, CWRNNT_LINEAR_BACKWARD);
    TORCH_CHECK(bytes >= 0, "invalid linear layer");
    auto ws = torch::empty({bytes}, x.options().dtype(torch::kUInt8));
    OptTensor gx, gw, gb;
    if (want_x) gx = torch::empty({x.size(0), x.size(1)}, x.options());
    if (want_weight) gw = torch::empty({weight.size(0), weight.size(1)}, x.options());
    if (want_bias) gb = torch::empty({weight.size(0)}, x.options());
    check_status(cwrnnt_linear_backward(&p, x.data_ptr(), weight.data_ptr(), ptr(bias), g.data_ptr(), ws.data_ptr(),
                                        bytes, ptr(gx), ptr(gw), ptr(gb), current_stream()),
                 "cwrnnt_linear_backward");
    return {gx, gw, gb};
}

// ----------------------------------------------------------------------- the operators above as autograd functions
// (In C++, so that a small step does not spend its time in the interpreter.) None of them is differentiable twice: a
// gradient that was computed with create_graph raises when it is differentiated.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

variable_list once_differentiable(variable_list grads, const char *name)
{
    if (!at::GradMode::is_enabled()) return grads;
    auto refuse = std::make_shared<torch::autograd::DelayedError>(
        std::string(name) + " is not differentiable twice", static_cast<int64_t>(grads.size()));
    for (auto &g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    return (*refuse)(std::move(grads));
}
OptTensor some(const torch::Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// None of them has a forward-mode derivative either. A tensor with a tangent need not require a gradient, so the autograd
// functions may not see it, and the tangent would be dropped and read as zero.
void refuse_tangent(const OptTensor &t, const char *name)
{
    TORCH_CHECK(!(t && t->defined() && t->_fw_grad(0).defined()), name, " has no forward-mode derivative");
}

class TokenScoresFn : public torch::autograd::Function<TokenScoresFn> {
public:
    // outputs: those of (log_probs, entropy, top_log_probs, top_indices) that were asked for
    static variable_list forward(AutogradContext *ctx, const torch::Tensor &x, const OptTensor &targets, int64_t top_k,
                                 bool entropy, double temperature)
    {
        auto [lp, ent, top, index, stats] = token_scores(x, targets, top_k, entropy, temperature, true);
        ctx->save_for_backward({x, targets.value_or(torch::Tensor()), index.value_or(torch::Tensor()), *stats,
                                ent.value_or(torch::Tensor())});
        ctx->saved_data["temperature"] = temperature;
        ctx->set_materialize_grads(false);
        if (index) ctx->mark_non_differentiable({*index});
        variable_list out;
        for (const OptTensor *t : {&lp, &ent, &top, &index})
            if (*t) out.push_back(**t);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        OptTensor up[3];  // in the order of the outputs
        size_t at = 0;
        const bool have[3] = {saved[1].defined(), saved[4].defined(), saved[2].defined()};
        bool any = false;
        for (int i = 0; i < 3; ++i) {
            if (!have[i]) continue;
            if (grads[at].defined()) up[i] = grads[at].detach().contiguous(), any = true;
            ++at;
        }
        variable_list out(5);
        if (any)
            out[0] = token_scores_backward(saved[0].detach(), some(saved[1]), some(saved[2]), saved[3], some(saved[4]),
                                           up[0], up[1], up[2], ctx->saved_data["temperature"].toDouble());
        return once_differentiable(std::move(out), "token_scores");
    }
};

std::tuple<OptTensor, OptTensor, OptTensor, OptTensor> token_scores_ad(const torch::Tensor &x, const OptTensor &targets,
                                                                       int64_t top_k, bool entropy, double temperature)
{
    refuse_tangent(x, "token_scores");
    if (!(at::GradMode::is_enabled() && x.requires_grad())) {
        auto [lp, ent, top, index, stats] = token_scores(x, targets, top_k, entropy, temperature, false);
        return {lp, ent, top, index};
    }
    auto out = TokenScoresFn::apply(x, targets, top_k, entropy, temperature);
    size_t at = 0;
    auto next = [&](bool wanted) { return wanted ? OptTensor(out[at++]) : OptTensor(); };
    auto lp = next(targets.has_value()), ent = next(entropy), top = next(top_k > 0), index = next(top_k > 0);
    return {lp, ent, top, index};
}

// The capture that the current stream is in, 0: none.
int64_t current_capture()
{
    if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) return 0;
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    C10_CUDA_CHECK(cudaStreamGetCaptureInfo(at::cuda::getCurrentCUDAStream(), &status, &id));
    return static_cast<int64_t>(id);
}

class DistillFn : public torch::autograd::Function<DistillFn> {
public:
    static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &x, const torch::Tensor &teacher,
                                 const torch::Tensor &indices, const OptTensor &weight, bool tail, double temperature,
                                 double scale, bool reduced, bool eager)
    {
        auto [rows, loss, grad] =
            distill(x, teacher, indices, weight, {}, tail, temperature, scale, !reduced, reduced, reduced && eager);
        ctx->save_for_backward({x, teacher, indices, weight.value_or(torch::Tensor())});
        ctx->saved_data["tail"] = tail;
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["scale"] = scale;
        if (grad) ctx->saved_data["grad"] = *grad;
        const c10::cuda::CUDAGuard guard(x.device());
        ctx->saved_data["capture"] = current_capture();
        return reduced ? *loss : *rows;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        variable_list out(9);
        const auto g = grads[0].detach();
        auto make = [&](const OptTensor &made) {
            const auto saved = ctx->get_saved_variables();
            return *std::get<2>(distill(saved[0].detach(), saved[1], saved[2], some(saved[3]), g.contiguous(),
                                        ctx->saved_data["tail"].toBool(), ctx->saved_data["temperature"].toDouble(),
                                        ctx->saved_data["scale"].toDouble(), false, false, true, made));
        };
        const auto eager = ctx->saved_data.find("grad");
        if (eager != ctx->saved_data.end() && ctx->saved_data["capture"].toInt() == current_capture()) {
            // computed during forward for an upstream gradient of 1; handed over once (a second backward over a
            // retained graph recomputes it below, and so does one that is captured without its forward, or in a graph
            // of its own: replayed by itself, it would scale the one gradient again and again)
            out[0] = eager->second.toTensor();
            ctx->saved_data.erase(eager);
            // Of a mean over many rows float16 keeps few digits of a gradient and none below 2^-25 (a token of probability
            // 1e-2 of 300 000 rows); a loss scale comes too late for them. So that gradient is made anew unless the
            // factor is 1. The other types have the range, and their one more rounding is half a step.
            if (out[0].scalar_type() == torch::ScalarType::Half)
                out[0] = make(out[0]);
            else if (out[0].numel())
                rnnt_scale_grad(out[0], g);
        } else {
            out[0] = make({});
        }
        return once_differentiable(std::move(out), "distill_loss");
    }
};

torch::Tensor distill_ad(const torch::Tensor &x, const torch::Tensor &teacher, const torch::Tensor &indices,
                         const OptTensor &weight, bool tail, double temperature, double scale, bool reduced, bool eager)
{
    refuse_tangent(x, "distill_loss");
    if (at::GradMode::is_enabled() && x.requires_grad())
        return DistillFn::apply(x, teacher, indices, weight, tail, temperature, scale, reduced, eager);
    auto [rows, loss, grad] =
        distill(x, teacher, indices, weight, {}, tail, temperature, scale, !reduced, reduced, false);
    return reduced ? *loss : *rows;
}

class LinearFn : public torch::autograd::Function<LinearFn> {
public:
    static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &x, const torch::Tensor &weight,
                                 const OptTensor &bias, const OptTensor &residual, int64_t activation)
    {
        ctx->save_for_backward({x, weight, bias.value_or(torch::Tensor())});
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["residual"] = residual.has_value();
        return linear_forward(x, weight, bias, residual, activation);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        variable_list out(5);
        const auto saved = ctx->get_saved_variables();
        const auto g = grads[0].detach();
        // (edges are counted over the tensors that were given: the bias is the third if there is one)
        const bool want[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                              saved[2].defined() && ctx->needs_input_grad(2)};
        if (want[0] || want[1] || want[2]) {
            const OptTensor bias = saved[2].defined() ? OptTensor(saved[2].detach()) : OptTensor();
            auto [gx, gw, gb] = linear_backward(saved[0].detach(), saved[1].detach(), bias, g,
                                                ctx->saved_data["activation"].toInt(), want[0], want[1], want[2]);
            if (gx) out[0] = *gx;
            if (gw) out[1] = *gw;
            if (gb) out[2] = *gb;
        }
        if (ctx->saved_data["residual"].toBool()) out[3] = g;
        return once_differentiable(std::move(out), "fused_linear");
    }
};

torch::Tensor linear_ad(const torch::Tensor &x, const torch::Tensor &weight, const OptTensor &bias,
                        const OptTensor &residual, int64_t activation)
{
    for (const OptTensor &t : {OptTensor(x), OptTensor(weight), bias, residual}) refuse_tangent(t, "fused_linear");
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad()) ||
                                       (residual && residual->requires_grad())))
        return LinearFn::apply(x, weight, bias, residual, activation);
    return linear_forward(x, weight, bias, residual, activation);
}

// ------------------------------------------------------------------- the reference module's functions, same shapes

// cwarp_cuda.cpp:84-108. xs are log-probabilities. Returns (costs [N], grads [STU,2], alphas, betas [N,Tmax,Umax+1]).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>
compact_rnnt_loss_forward(const torch::Tensor xs, const torch::Tensor lx, const torch::Tensor ys,
                          const torch::Tensor ly, const int blank)
{
    check_inputs(xs, lx, ys, ly);
    TORCH_CHECK(xs.scalar_type() == torch::ScalarType::Float || xs.scalar_type() == torch::ScalarType::Double,
                "the reference-shaped entry points take float32 or float64 log-probabilities");
    const c10::cuda::CUDAGuard guard(xs.device());
    cwrnnt_problem p = describe(xs, lx, ys, blank, 0, 0);
    auto ws = make_workspace(p, xs);
    auto costs = torch::empty({lx.size(0)}, xs.options());
    check_status(cwrnnt_forward(&p, xs.data_ptr(), i32(lx), i32(ly), i32(ys), ws.data_ptr(), ws.numel(),
                                costs.data_ptr(), nullptr, current_stream()),
                 "cwrnnt_forward");
    auto grads = torch::empty({xs.size(0), 2}, xs.options());
    check_status(cwrnnt_pair_grads(&p, xs.data_ptr(), i32(lx), i32(ly), i32(ys), ws.data_ptr(), grads.data_ptr(),
                                   current_stream()),
                 "cwrnnt_pair_grads");
    // padded debug outputs need max T on the host, like the reference (cwarp_cuda_rnnt_kernel.cu:395-396)
    const int64_t t_max = lx.numel() ? lx.max().item<int64_t>() : 0;
    const int64_t u_max1 = ys.size(1) + 1;
    auto alphas = torch::empty({lx.size(0), t_max, u_max1}, xs.options());
    auto betas = torch::empty_like(alphas);
    check_status(cwrnnt_export_alpha_beta(&p, i32(lx), i32(ly), ws.data_ptr(), static_cast<int32_t>(t_max),
                                          static_cast<int32_t>(u_max1), alphas.data_ptr(), betas.data_ptr(),
                                          current_stream()),
                 "cwrnnt_export_alpha_beta");
    return {costs, grads, alphas, betas};
}

// cwarp_cuda.cpp:58-82. Costs only.
torch::Tensor compact_rnnt_loss(const torch::Tensor xs, const torch::Tensor lx, const torch::Tensor ys,
                                const torch::Tensor ly, const int blank)
{
    check_inputs(xs, lx, ys, ly);
    TORCH_CHECK(xs.scalar_type() == torch::ScalarType::Float || xs.scalar_type() == torch::ScalarType::Double,
                "the reference-shaped entry points take float32 or float64 log-probabilities");
    const c10::cuda::CUDAGuard guard(xs.device());
    cwrnnt_problem p = describe(xs, lx, ys, blank, CWRNNT_COSTS_ONLY, 0);
    auto ws = make_workspace(p, xs);
    auto costs = torch::empty({lx.size(0)}, xs.options());
    check_status(cwrnnt_forward(&p, xs.data_ptr(), i32(lx), i32(ly), i32(ys), ws.data_ptr(), ws.numel(),
                                costs.data_ptr(), nullptr, current_stream()),
                 "cwrnnt_forward");
    return costs;
}

// cwarp_cuda.cpp:110-136. grad_in [STU,2] is NOT modified (the reference scales it in place).
torch::Tensor compact_rnnt_loss_backward(torch::Tensor grad_in, const torch::Tensor grad_costs,
                                         const torch::Tensor labels, const torch::Tensor lx, const torch::Tensor ly,
                                         const int blank, const int V)
{
    CHECK_CUDA(grad_costs);
    CHECK_CUDA(grad_in);
    CHECK_INPUT(labels, torch::ScalarType::Int);
    CHECK_INPUT(lx, torch::ScalarType::Int);
    CHECK_INPUT(ly, torch::ScalarType::Int);
    TORCH_CHECK(grad_in.dim() == 2 && grad_in.size(1) == 2, "grad_in must be [STU, 2]");
    TORCH_CHECK(grad_in.scalar_type() == torch::ScalarType::Float || grad_in.scalar_type() == torch::ScalarType::Double,
                "grad_in must be float32 or float64");
    const c10::cuda::CUDAGuard guard(grad_in.device());
    auto g = grad_in.contiguous();
    auto gc = grad_costs.to(g.scalar_type()).contiguous();
    TORCH_CHECK(gc.numel() == lx.size(0), "grad_costs must be [N]");
    cwrnnt_problem p{};
    p.n_rows = g.size(0);
    p.V = V;
    p.B = static_cast<int32_t>(lx.size(0));
    p.y_stride = p.max_u = static_cast<int32_t>(labels.size(1));
    p.blank = blank;
    p.dtype = g.scalar_type() == torch::ScalarType::Double ? CWRNNT_F64 : CWRNNT_F32;
    auto scratch = torch::empty({cwrnnt_scatter_scratch_bytes(p.B)}, g.options().dtype(torch::kUInt8));
    auto dense = torch::empty({g.size(0), static_cast<int64_t>(V)}, g.options());
    check_status(cwrnnt_scatter_backward(&p, g.data_ptr(), gc.data_ptr(), i32(lx), i32(ly), i32(labels),
                                         scratch.data_ptr(), scratch.numel(), dense.data_ptr(), current_stream()),
                 "cwrnnt_scatter_backward");
    return dense;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("_cwarp_rnnt_forward", &compact_rnnt_loss_forward,
          "Transducer loss forward for compact layout (reference shapes): (costs, grads[STU,2], alphas, betas).");
    m.def("_cwarp_rnnt_backward", &compact_rnnt_loss_backward,
          "Transducer loss backward for compact layout (reference shapes): dense [STU,V] gradient.");
    m.def("_cwarp_rnnt_loss", &compact_rnnt_loss, "Transducer costs without gradients.");
    m.def("_rnnt_forward", &rnnt_forward, "Fused forward: (costs, loss, workspace).");
    m.def("_rnnt_backward", &rnnt_backward, "Fused backward: gradient w.r.t. xs.");
    m.def("_rnnt_loss_grad", &rnnt_loss_grad,
          "Pipelined forward + gradient for an upstream gradient of 1: (costs, loss, workspace, grad_x).");
    m.def("_rnnt_scale_grad", &rnnt_scale_grad, "In-place grad_x *= factor (device scalar); free when the factor is 1.");
    m.def("_rnnt_validate", &rnnt_validate,
          "Validates lengths, row count and labels: [bits, first bad sequence, max lx, max ly] (one short sync).");
    m.def("_rnnt_validate_begin", &rnnt_validate_begin,
          "Queues the validation and returns a pinned int32[4] tensor filled once the current stream gets there.");
    m.def("_rnnt_status", &rnnt_status, "Status words of a workspace (synchronises).");
    m.def("_pack_padded", &pack_padded, "Padded [N,T,U+1,V] -> compact [n_rows,V].");
    m.def("_unpack_padded", &unpack_padded, "Compact [n_rows,V] -> zero-padded [N,T,U+1,V].");
    m.def("_token_scores", &token_scores_ad,
          "Scores of logits rows: (log_probs, entropy, top_log_probs, top_indices), differentiable.");
    m.def("_distill", &distill_ad, "Distillation from a teacher's top entries: the loss, or one per row; differentiable.");
    m.def("_linear", &linear_ad, "act(x W^T + bias) + residual on the tensor cores, differentiable.");
    m.attr("MAX_LIST") = static_cast<int>(CWRNNT_MAX_LIST);
    m.attr("FUSED_LOG_SOFTMAX") = static_cast<int>(CWRNNT_FUSED_LOG_SOFTMAX);
    m.attr("COSTS_ONLY") = static_cast<int>(CWRNNT_COSTS_ONLY);
    m.attr("REDUCE_MEAN") = static_cast<int>(CWRNNT_REDUCE_MEAN);
    m.attr("REDUCE_SUM") = static_cast<int>(CWRNNT_REDUCE_SUM);
    m.attr("AVERAGE_FRAMES") = static_cast<int>(CWRNNT_AVERAGE_FRAMES);
    m.attr("ST_BAD_LENGTH") = static_cast<int>(CWRNNT_ST_BAD_LENGTH);
    m.attr("ST_ROW_MISMATCH") = static_cast<int>(CWRNNT_ST_ROW_MISMATCH);
    m.attr("ST_BAD_LABEL") = static_cast<int>(CWRNNT_ST_BAD_LABEL);
    m.attr("ST_FWD_BWD_GAP") = static_cast<int>(CWRNNT_ST_FWD_BWD_GAP);
}
