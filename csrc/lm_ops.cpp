// Host side of the operators around the language-model head: argument checks, workspaces and
// launches of distill.hip, adapters.hip and logits.hip.  Python (ops/distill.py and its
// neighbours) checks shapes with errors of its own; what a kernel relies on is checked here again.
#include "lm_ops.h"

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <algorithm>
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
void launch_adjust(int, const void*, long, void*, const void*, long, int, int, const void*, int,
                   const void*, int, const float*, float, const float*, float, const float*,
                   float, const void*, long, int, const float*, long, int, const unsigned*, long,
                   long, int, hipStream_t);
int lowrank_rp(int R);
int lowrank_splits(const long* counts, int S, long T, int K);
int lowrank_outer_shift(const long* counts, int S, long T, int NP);
int lowrank_outer_tiles(const long* counts, int S, long T, int shift);
void launch_shrink(int, int, const void*, long, const void*, int, int, const int*, const int*,
                   const int*, const long*, int, int, long, const float*, float, void*, float*,
                   hipStream_t);
void launch_expand(int, int, const void*, long, void*, long, const void*, const void*, int, int,
                   const int*, const int*, const int*, const long*, int, int, long, hipStream_t);
void launch_outer(int, int, const void*, long, int, const void*, float*, const int*, const int*,
                  const int*, const long*, int, int, long, int, void*, int, int, hipStream_t);
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

// ------------------------------------------------------------------ logits of a decode step
// A per-request number as a (B,) tensor; the scalar beside it is used where there is none.
Tensor per_row(const OptTensor& t, const Tensor& logits, const char* name) {
    if (!t.has_value()) return Tensor();
    TORCH_CHECK(t->dim() == 1 && t->size(0) == logits.size(0), name, " must be (B,)");
    check_on(*t, logits, name);
    return t->to(at::kFloat).contiguous();
}
const float* float_ptr(const Tensor& t) { return t.defined() ? (const float*)t.data_ptr() : nullptr; }

Tensor adjust(Tensor logits, OptTensor history, OptTensor lengths, OptTensor prompts,
              OptTensor repetition, double repetition_all, OptTensor presence,
              double presence_all, OptTensor frequency, double frequency_all,
              OptTensor bias_index, OptTensor bias, OptTensor allowed) {
    TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "logits must be (B, V) on GPU");
    const long B = logits.size(0), V = logits.size(1);
    TORCH_CHECK(V <= (1 << 30), "logits: V must be at most 2^30");
    const c10::DeviceGuard guard(logits.device());
    const int type = type_of(logits, "logits");
    const Tensor z = rows_of(logits);
    Tensor h, len, pre, bi, bv, ok;
    int h64 = 0, l64 = 0, p64 = 0, i64 = 0;
    if (history.has_value()) {
        TORCH_CHECK(history->dim() == 2 && history->size(0) == B &&
                        history->size(1) <= (1 << 30),
                    "history must be (B, L)");
        check_on(*history, logits, "history");
        h64 = wide_index(*history, "history");
        h = rows_of(*history);
        auto per_request = [&](const OptTensor& t, Tensor& to, int& wide, const char* name) {
            if (!t.has_value()) return;
            TORCH_CHECK(t->dim() == 1 && t->size(0) == B, name, " must be (B,)");
            check_on(*t, logits, name);
            wide = wide_index(*t, name);
            to = t->contiguous();
        };
        per_request(lengths, len, l64, "lengths");
        per_request(prompts, pre, p64, "prompt_lengths");
    }
    const Tensor rep = per_row(repetition, logits, "repetition"),
                 pres = per_row(presence, logits, "presence"),
                 freq = per_row(frequency, logits, "frequency");
    if (bias_index.has_value()) {
        TORCH_CHECK(bias.has_value() && bias_index->dim() == 2 && bias_index->size(0) == B &&
                        bias->sizes() == bias_index->sizes() && bias->size(1) <= (1 << 30),
                    "bias_index and bias must be (B, K)");
        check_on(*bias_index, logits, "bias_index");
        check_on(*bias, logits, "bias");
        i64 = wide_index(*bias_index, "bias_index");
        bi = rows_of(*bias_index);
        bv = rows_of(bias->to(at::kFloat));
    }
    if (allowed.has_value()) {
        TORCH_CHECK(allowed->dim() == 2 && allowed->size(0) == B &&
                        allowed->size(1) == (V + 31) / 32 && allowed->scalar_type() == at::kInt,
                    "allowed must be (B, ceil(V / 32)) int32");
        check_on(*allowed, logits, "allowed");
        ok = rows_of(*allowed);
    }
    auto out = at::empty({B, V}, logits.options());
    if (B == 0 || V == 0) return out;
    auto ptr = [](const Tensor& t) -> const void* { return t.defined() ? t.data_ptr() : nullptr; };
    auto stride = [](const Tensor& t) { return t.defined() ? row_stride(t) : 0; };
    // an empty list has no data: it is no list
    const bool past = h.defined() && h.size(1) > 0, some = bi.defined() && bi.size(1) > 0;
    launch_adjust(type, z.data_ptr(), row_stride(z), out.data_ptr(), past ? ptr(h) : nullptr,
                  stride(h), past ? (int)h.size(1) : 0, h64, ptr(len), l64, ptr(pre), p64,
                  float_ptr(rep), (float)repetition_all, float_ptr(pres), (float)presence_all,
                  float_ptr(freq), (float)frequency_all, some ? ptr(bi) : nullptr, stride(bi),
                  i64, some ? float_ptr(bv) : nullptr, stride(bv), some ? (int)bi.size(1) : 0,
                  (const unsigned*)ptr(ok), stride(ok), B, (int)V, stream_of(logits));
    check_launch("adjust_logits");
    return out;
}

// ------------------------------------------------------------------ low-rank adapters
// Rows grouped by adapter (ops/adapters.py: AdapterRows), and what every launch takes of them.
struct Grouped {
    Tensor order, segs, adapter, scale;
    std::vector<long> counts;
    int S, Bn, L, K, M, R, type;
    long T, N;
    float scale_all;

    Grouped(const Tensor& x, const Tensor& y, const Tensor& a, const Tensor& b, Tensor order_,
            Tensor segs_, Tensor adapter_, std::vector<int64_t> counts_, const OptTensor& scale_,
            double all)
        : order(order_), segs(segs_), adapter(adapter_), counts(counts_.begin(), counts_.end()),
          scale_all((float)all) {
        TORCH_CHECK(x.is_cuda() && x.dim() == 2 && y.dim() == 2 && x.size(0) == y.size(0),
                    "lowrank: x (N, K) and y (N, M) on GPU");
        TORCH_CHECK(a.dim() == 3 && b.dim() == 3 && a.size(0) == b.size(0) &&
                        a.size(2) == b.size(1) && a.size(1) == x.size(1) &&
                        b.size(2) == y.size(1),
                    "lowrank: a (L, K, R), b (L, R, M)");
        TORCH_CHECK(a.is_contiguous() && b.is_contiguous(), "lowrank: a and b contiguous");
        for (const Tensor* t : {&y, &a, &b}) {
            check_on(*t, x, "lowrank: every tensor");
            TORCH_CHECK(t->scalar_type() == x.scalar_type(), "lowrank: one type for all");
        }
        for (const Tensor* t : {&order, &segs, &adapter}) {
            check_on(*t, x, "lowrank: the grouped rows");
            TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous(), "lowrank: rows int32");
        }
        type = type_of(x, "x");
        TORCH_CHECK(type != 2, "lowrank: bf16 or fp16");
        L = (int)a.size(0);
        K = (int)a.size(1);
        R = (int)a.size(2);
        M = (int)b.size(2);
        N = x.size(0);
        Bn = (int)order.numel();
        S = (int)counts.size();
        TORCH_CHECK(R >= 1 && R <= 128 && K >= 1 && M >= 1 && K < (1 << 30) && M < (1 << 30),
                    "lowrank: a rank of 1 to 128");
        TORCH_CHECK(segs.numel() == 4l * S && adapter.numel() == Bn && Bn > 0 && N % Bn == 0,
                    "lowrank: N rows of Bn columns");
        T = N / Bn;
        long sum = 0;
        for (long c : counts) sum += c;
        TORCH_CHECK(sum == Bn && N < (1l << 31) && N / 64 * ((std::max(K, M) + 127) / 128) <
                        (1l << 31), "lowrank: too many rows");
        if (scale_.has_value()) {
            TORCH_CHECK(scale_->numel() == L && scale_->dim() == 1, "lowrank: scale (L,)");
            check_on(*scale_, x, "scale");
            scale = scale_->to(at::kFloat).contiguous();
        }
    }
    const int* ip(const Tensor& t) const { return (const int*)t.data_ptr(); }

    // v (N, RP) = s x W, W (L, K, R) or, contraction contiguous, (L, R, K)
    Tensor shrink(const Tensor& x, const Tensor& w, bool kcont, hipStream_t st) const {
        const int k = (int)x.size(1), splits = lowrank_splits(counts.data(), S, T, k);
        auto v = at::empty({N, (long)lowrank_rp(R)}, x.options());
        Tensor part;
        if (splits > 1)
            part = at::empty({(long)splits * N * lowrank_rp(R)}, x.options().dtype(at::kFloat));
        launch_shrink(type, kcont, x.data_ptr(), row_stride(x), w.data_ptr(), k, R, ip(order),
                      ip(segs), ip(adapter), counts.data(), S, Bn, T, float_ptr(scale), scale_all,
                      v.data_ptr(), splits > 1 ? (float*)part.data_ptr() : nullptr, st);
        check_launch("lowrank shrink");
        return v;
    }
    // out = base + v W, W (L, R, M) or, rank contiguous, (L, M, R)
    void expand(const Tensor& base, Tensor& out, const Tensor& v, const Tensor& w, bool rcont,
                hipStream_t st) const {
        launch_expand(type, rcont, base.defined() ? base.data_ptr() : nullptr,
                      base.defined() ? row_stride(base) : 0, out.data_ptr(), row_stride(out),
                      v.data_ptr(), w.data_ptr(), (int)out.size(1), R, ip(order), ip(segs),
                      ip(adapter), counts.data(), S, Bn, T, st);
        check_launch("lowrank expand");
    }
    // sum over an adapter's rows of p^T q: (L, R, NP) or, rank contiguous, (L, NP, R)
    Tensor outer(const Tensor& p, const Tensor& q, bool rcont, hipStream_t st) const {
        const int np = (int)p.size(1), shift = lowrank_outer_shift(counts.data(), S, T, np);
        const long tiles = lowrank_outer_tiles(counts.data(), S, T, shift);
        auto part = at::empty({tiles * lowrank_rp(R) * ((np + 127) / 128 * 128)},
                              p.options().dtype(at::kFloat));
        auto out = rcont ? at::empty({L, np, R}, p.options()) : at::empty({L, R, np}, p.options());
        launch_outer(type, rcont, p.data_ptr(), row_stride(p), np, q.data_ptr(),
                     (float*)part.data_ptr(), ip(order), ip(segs), ip(adapter), counts.data(), S,
                     Bn, T, shift, out.data_ptr(), R, L, st);
        check_launch("lowrank outer");
        return out;
    }
};

// -> (out, v); out is y itself where `inplace`
std::vector<Tensor> lowrank_fwd(Tensor y, Tensor x, Tensor a, Tensor b, Tensor order, Tensor segs,
                                Tensor adapter, std::vector<int64_t> counts, OptTensor scale,
                                double scale_all, bool inplace) {
    const c10::DeviceGuard guard(x.device());
    const Grouped g(x, y, a, b, order, segs, adapter, counts, scale, scale_all);
    const hipStream_t st = stream_of(x);
    const Tensor xr = rows_of(x), yr = inplace ? y : rows_of(y);
    TORCH_CHECK(yr.size(1) <= 1 || yr.stride(1) == 1, "lowrank: y's rows must be contiguous");
    Tensor out = inplace ? y : at::empty({g.N, (long)g.M}, y.options());
    Tensor v = g.shrink(xr, a, false, st);
    g.expand(yr, out, v, b, false, st);
    return {out, v};
}

std::vector<OptTensor> lowrank_bwd(Tensor dy, Tensor x, Tensor a, Tensor b, Tensor v, Tensor order,
                                   Tensor segs, Tensor adapter, std::vector<int64_t> counts,
                                   OptTensor scale, double scale_all, bool need_x, bool need_a,
                                   bool need_b) {
    const c10::DeviceGuard guard(x.device());
    const Grouped g(x, dy, a, b, order, segs, adapter, counts, scale, scale_all);
    const hipStream_t st = stream_of(x);
    TORCH_CHECK(v.dim() == 2 && v.size(0) == g.N && v.size(1) == lowrank_rp(g.R) &&
                    v.is_contiguous() && v.scalar_type() == x.scalar_type(),
                "lowrank_bwd: v as lowrank_fwd returned it");
    check_on(v, x, "v");
    const Tensor xr = rows_of(x), dr = rows_of(dy);
    OptTensor dx, da, db;
    if (need_x || need_a) {
        const Tensor u = g.shrink(dr, b, true, st);
        if (need_x) {
            Tensor out = at::empty({g.N, (long)g.K}, x.options());
            g.expand(Tensor(), out, u, a, true, st);
            dx = out;
        }
        if (need_a) da = g.outer(xr, u, true, st);
    }
    if (need_b) db = g.outer(dr, v, false, st);
    return {dx, da, db};
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
    m.def("adjust_logits", &adjust, "penalties, biases and masks on decode logits",
          py::arg("logits"), py::arg("history"), py::arg("lengths"), py::arg("prompt_lengths"),
          py::arg("repetition"), py::arg("repetition_all"), py::arg("presence"),
          py::arg("presence_all"), py::arg("frequency"), py::arg("frequency_all"),
          py::arg("bias_index"), py::arg("bias"), py::arg("allowed"));
    m.def("lowrank_fwd", &lowrank_fwd, "y + s x A B by rows' adapters", py::arg("y"),
          py::arg("x"), py::arg("a"), py::arg("b"), py::arg("order"), py::arg("segs"),
          py::arg("adapter"), py::arg("counts"), py::arg("scale") = py::none(),
          py::arg("scale_all") = 1.0, py::arg("inplace") = false);
    m.def("lowrank_bwd", &lowrank_bwd, "gradients of lowrank_fwd", py::arg("dy"), py::arg("x"),
          py::arg("a"), py::arg("b"), py::arg("v"), py::arg("order"), py::arg("segs"),
          py::arg("adapter"), py::arg("counts"), py::arg("scale") = py::none(),
          py::arg("scale_all") = 1.0, py::arg("need_x") = true, py::arg("need_a") = true,
          py::arg("need_b") = true);
}
