// Host side of the operators around the language-model head: argument checks, workspaces and
// launches of distill.hip, adapters.hip and logits.hip.  Python (ops/distill.py and its
// neighbours) checks shapes with errors of its own; what a kernel relies on is checked here again.
#include "lm_ops.h"

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <vector>

extern "C" {
int distill_splits(long N, int V);
void launch_distill_fwd(int, const void*, long, const void*, long, int, const void*, long, int,
                        const long*, int, float*, float*, float*, float*, float*, long, int,
                        float, float,
                        hipStream_t);
void launch_distill_bwd(int, const void*, long, const void*, long, int, const void*, long, int,
                        const long*, int, const float*, const float*, const float*, void*, long,
                        int, float, float, hipStream_t);
}

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

// The current stream of the tensors' own device (the caller holds a DeviceGuard on it).
hipStream_t stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int type_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return 0;
        case at::kHalf: return 1;
        case at::kFloat: return 2;
        default: break;
    }
    TORCH_CHECK(false, name, " must be bf16, fp16 or fp32, got ", t.scalar_type());
}

bool wide_index(const Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, name,
                " must be int32 or int64");
    return t.scalar_type() == at::kLong;
}

void check_on(const Tensor& t, const Tensor& ref, const char* name) {
    TORCH_CHECK(t.device() == ref.device(), name, " must be on ", ref.device(), ", got ",
                t.device());
}

void check_launch(const char* name) {
    const hipError_t e = hipGetLastError();
    TORCH_CHECK(e == hipSuccess, name, ": ", hipGetErrorString(e));
}

// Rows of any stride with neighbouring elements side by side; anything else is copied.
Tensor rows_of(const Tensor& t) {
    return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous();
}
long row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct Distill {
    Tensor z, index, teacher, target;
    long N;
    int V, K, type, ttype, index64;
    const long* tp;

    Distill(const Tensor& logits, const Tensor& idx, const Tensor& t, const OptTensor& y) {
        TORCH_CHECK(logits.is_cuda(), "logits must be on GPU");
        TORCH_CHECK(logits.dim() == 2 && idx.dim() == 2 && t.dim() == 2 &&
                        idx.size(0) == logits.size(0) && t.size(0) == logits.size(0) &&
                        idx.size(1) == t.size(1),
                    "distill: logits (N, V), teacher_index and teacher_logits (N, K)");
        TORCH_CHECK(logits.size(1) >= 1 && logits.size(1) <= (1 << 30) &&
                        t.size(1) <= (1 << 30),
                    "distill: V and K must be below 2^30, V at least 1");
        check_on(idx, logits, "teacher_index");
        check_on(t, logits, "teacher_logits");
        type = type_of(logits, "logits");
        ttype = type_of(t, "teacher_logits");
        index64 = wide_index(idx, "teacher_index");
        z = rows_of(logits);
        index = rows_of(idx);
        teacher = rows_of(t);
        N = z.size(0);
        V = (int)z.size(1);
        K = (int)t.size(1);
        tp = nullptr;
        if (y.has_value()) {
            TORCH_CHECK(y->dim() == 1 && y->size(0) == N && y->scalar_type() == at::kLong,
                        "distill: targets must be (N,) int64");
            check_on(*y, logits, "targets");
            target = y->contiguous();
            tp = (const long*)target.data_ptr();
        }
    }
};

// -> (loss, 1 / counted rows, stats (N, 8) fp32; the last two for the backward pass)
std::vector<Tensor> distill_fwd(Tensor logits, Tensor index, Tensor teacher, OptTensor targets,
                                double alpha, double tau) {
    const Distill d(logits, index, teacher, targets);
    const c10::DeviceGuard guard(logits.device());
    const auto f32 = logits.options().dtype(at::kFloat);
    const int splits = distill_splits(d.N, d.V);
    auto loss = at::empty({}, f32), inv = at::empty({}, f32), stats = at::empty({d.N, 8}, f32);
    auto work = at::empty({d.N * (2 + 3 * (long)splits)}, f32);
    float* rows = (float*)work.data_ptr();
    launch_distill_fwd(d.type, d.z.data_ptr(), row_stride(d.z), d.index.data_ptr(),
                       row_stride(d.index), d.index64, d.teacher.data_ptr(),
                       row_stride(d.teacher), d.ttype, d.tp, d.K, rows + 2 * d.N,
                       (float*)stats.data_ptr(), rows, (float*)loss.data_ptr(),
                       (float*)inv.data_ptr(), d.N, d.V, (float)alpha, (float)tau, stream_of(logits));
    check_launch("distill_fwd");
    return {loss, inv, stats};
}

Tensor distill_bwd(Tensor logits, Tensor index, Tensor teacher, OptTensor targets, Tensor stats,
                   Tensor inv, Tensor grad, double alpha, double tau) {
    const Distill d(logits, index, teacher, targets);
    const c10::DeviceGuard guard(logits.device());
    TORCH_CHECK(stats.is_contiguous() && stats.numel() == d.N * 8 && inv.numel() == 1,
                "distill_bwd: stats and inv as distill_fwd returned them");
    check_on(grad, logits, "grad");
    const Tensor g = grad.to(at::kFloat).contiguous();
    TORCH_CHECK(g.numel() == 1, "distill_bwd: the gradient of the loss is one number");
    auto dz = at::empty({d.N, (long)d.V}, logits.options());
    if (d.N == 0) return dz;
    launch_distill_bwd(d.type, d.z.data_ptr(), row_stride(d.z), d.index.data_ptr(),
                       row_stride(d.index), d.index64, d.teacher.data_ptr(),
                       row_stride(d.teacher), d.ttype, d.tp, d.K,
                       (const float*)stats.data_ptr(), (const float*)inv.data_ptr(),
                       (const float*)g.data_ptr(), dz.data_ptr(), d.N, d.V, (float)alpha,
                       (float)tau, stream_of(logits));
    check_launch("distill_bwd");
    return dz;
}

}  // namespace

void register_lm_ops(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("distill_fwd", &distill_fwd, "distillation from a teacher's top logits: loss, stats",
          py::arg("logits"), py::arg("index"), py::arg("teacher"), py::arg("targets") = py::none(),
          py::arg("alpha"), py::arg("tau"));
    m.def("distill_bwd", &distill_bwd, "gradient of distill_fwd", py::arg("logits"),
          py::arg("index"), py::arg("teacher"), py::arg("targets") = py::none(), py::arg("stats"),
          py::arg("inv"), py::arg("grad"), py::arg("alpha"), py::arg("tau"));
}
