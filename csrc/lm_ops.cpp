// Host side of the operators around the language-model head: argument checks, workspaces and
// launches of distill.hip, adapters.hip and logits.hip.  Tensors on the GPU are checked here alone,
// with the errors that Python (ops/distill.py and its neighbours) raises for the reference: the
// checks there take as long as a launch (logits of one row 9.7 us a call with them, 6.7 without).
#include "lm_ops.h"

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <vector>

extern "C" {
int distill_in_registers(int V);
void launch_distill_fwd(int, const void*, long, const void*, long, int, const void*, long, int,
                        const long*, int, void*, float*, float*, float*, void*, long, int, float,
                        float, float, hipStream_t);
void launch_distill_bwd(int, const void*, long, const void*, long, int, const void*, long, int,
                        const long*, int, const void*, const float*, const float*, void*, int,
                        long, int, float, float, hipStream_t);
void launch_adjust(int, const void*, long, void*, const void*, long, int, int, const void*, int,
                   const void*, int, const float*, float, const float*, float, const float*,
                   float, const void*, long, int, const float*, long, int, const unsigned*, long,
                   long, int, hipStream_t);
int lowrank_width(int R);
int lowrank_row(int type, int R);
int lowrank_splits(const long* counts, int S, long T, int K, int alone);
int lowrank_outer_columns(const long* counts, int S, long T, int NP, int R, int with_u);
int lowrank_outer_shift(const long* counts, int S, long T, int strips, int columns, int R);
int lowrank_few(const long* counts, int S, long T);
void launch_expand_few(int, const void*, long, void*, long, const float*, const void*, int, int,
                       const int*, const int*, const int*, const long*, int, int, long,
                       const float*, float, int, hipStream_t);
int lowrank_outer_whole(const long* counts, int S, long T, int shift);
int lowrank_outer_tiles(const long* counts, int S, long T, int shift);
int lowrank_one_reading(int R);
void launch_shrink(int, int, const void*, long, long, const void*, long, int, int, const int*,
                   const int*, const int*, const long*, int, int, long, const float*, float,
                   void*, float*, int, hipStream_t);
void launch_shrink_sum(int, int, const int*, const int*, const int*, int, int, long, const float*,
                       float, void*, const float*, int, hipStream_t);
void launch_expand(int, int, const void*, long, long, void*, long, const void*, const void*, long,
                   int, int, const int*, const int*, const int*, const long*, int, int, long,
                   hipStream_t);
void launch_outer(int, int, const void*, long, long, int, const void*, float*, const void*, long,
                  float*, const int*, const int*, const int*, const long*, int, int, long, int,
                  int, int, void*, int, int, hipStream_t);
}

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

// A refusal of an argument, Python's ValueError.
#define REQUIRE(cond, ...) \
    if (!(cond)) throw pybind11::value_error(c10::str(__VA_ARGS__))

// The current stream of the tensors' own device (the caller holds a DeviceGuard on it).
hipStream_t stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// The capture that the stream is in, 0 for none.
int64_t capture_of(hipStream_t st) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo(st, &status, &id) != hipSuccess) {
        (void)hipGetLastError();        // the default stream, while another one is captured
        return 0;
    }
    return status == hipStreamCaptureStatusActive ? (int64_t)id : 0;
}

int type_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return 0;
        case at::kHalf: return 1;
        case at::kFloat: return 2;
        default: break;
    }
    REQUIRE(false, name, " must be bf16, fp16 or fp32, got ", t.scalar_type());
    return -1;
}

bool wide_index(const Tensor& t, const char* name) {
    REQUIRE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, name,
            " must be int32 or int64");
    return t.scalar_type() == at::kLong;
}

void check_on(const Tensor& t, const Tensor& ref, const char* name) {
    REQUIRE(t.device() == ref.device(), name, " must be on ", ref.device(), ", got ", t.device());
}

void check_launch(const char* name) {
    const hipError_t e = hipGetLastError();
    TORCH_CHECK(e == hipSuccess, name, ": ", hipGetErrorString(e));
}

// Forward-mode derivatives: a result without its tangent would make a wrong sum with others.
void check_no_tangent(const char* name, std::initializer_list<OptTensor> inputs) {
    for (const OptTensor& t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.has_value() || !t->defined() || !t->_fw_grad(0).defined(),
                                    name, " has no forward-mode derivative");
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
        REQUIRE(logits.is_cuda() && logits.dim() == 2, "logits must be (N, V) on GPU, got ",
                logits.sizes());
        REQUIRE(idx.dim() == 2 && idx.size(0) == logits.size(0) && t.sizes() == idx.sizes(),
                "teacher_index and teacher_logits must be (N=", logits.size(0), ", K), got ",
                idx.sizes(), ", ", t.sizes());
        REQUIRE(logits.size(1) >= 1 && logits.size(1) <= (1 << 30) && t.size(1) <= (1 << 30),
                "V and K must be below 2^30, V at least 1");
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
        REQUIRE(N < (1l << 32) / (V > 8192 ? 1024 : 256), "too many rows");
        tp = nullptr;
        if (y.has_value()) {
            REQUIRE(y->dim() == 1 && y->size(0) == N && y->scalar_type() == at::kLong,
                    "targets must be (N=", N, ",) int64");
            check_on(*y, logits, "targets");
            target = y->contiguous();
            tp = (const long*)target.data_ptr();
        }
    }
};

// The gradient is written with the loss where that can be; the backward pass then only looks
// whether it is scaled (csrc/distill.hip).
struct DistillLoss : public torch::autograd::Function<DistillLoss> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, Tensor logits, Tensor index,
                          Tensor teacher, OptTensor targets, double alpha, double tau,
                          double weight, bool need) {
        const Distill d(logits, index, teacher, targets);
        const c10::DeviceGuard guard(logits.device());
        const auto f32 = logits.options().dtype(at::kFloat);
        auto loss = at::empty({}, f32), inv = at::empty({}, f32), stats = at::empty({d.N, 8}, f32);
        auto rows = at::empty({d.N}, f32);
        Tensor dz;
        if (need && d.N > 0 && distill_in_registers(d.V))
            dz = at::empty({d.N, (long)d.V}, logits.options());
        launch_distill_fwd(d.type, d.z.data_ptr(), row_stride(d.z), d.index.data_ptr(),
                           row_stride(d.index), d.index64, d.teacher.data_ptr(),
                           row_stride(d.teacher), d.ttype, d.tp, d.K, stats.data_ptr(),
                           (float*)rows.data_ptr(), (float*)loss.data_ptr(),
                           (float*)inv.data_ptr(), dz.defined() ? dz.data_ptr() : nullptr, d.N,
                           d.V, (float)alpha, (float)tau, (float)weight, stream_of(logits));
        check_launch("distill_loss");
        if (need) {
            ctx->save_for_backward({logits, index, teacher, targets.value_or(Tensor()), stats,
                                    inv});
            ctx->saved_data["alpha"] = alpha;
            ctx->saved_data["tau"] = tau;
            if (dz.defined()) {
                ctx->saved_data["dz"] = dz;
                ctx->saved_data["capture"] = capture_of(stream_of(logits));
            }
        }
        return loss;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "distill_loss is differentiable once");
        const auto v = ctx->get_saved_variables();
        const Tensor &logits = v[0], &g = grads[0];
        torch::autograd::variable_list out(8);
        if (!g.defined()) return out;
        const Distill d(logits, v[1], v[2], v[3].defined() ? OptTensor(v[3]) : OptTensor());
        const c10::DeviceGuard guard(logits.device());
        // Handed out once: a second backward pass over a kept graph computes its own.  So does a
        // captured one whose forward is not in the same capture: it is replayed without it.
        const auto had = ctx->saved_data.find("dz");
        const bool done = had != ctx->saved_data.end() &&
                          ctx->saved_data["capture"].toInt() == capture_of(stream_of(logits));
        if (done) {
            out[0] = had->second.toTensor();
            ctx->saved_data.erase(had);
        } else {
            out[0] = at::empty({d.N, (long)d.V}, logits.options());
        }
        if (d.N > 0)
            launch_distill_bwd(d.type, d.z.data_ptr(), row_stride(d.z), d.index.data_ptr(),
                               row_stride(d.index), d.index64, d.teacher.data_ptr(),
                               row_stride(d.teacher), d.ttype, d.tp, d.K, v[4].data_ptr(),
                               (const float*)v[5].data_ptr(), (const float*)g.data_ptr(),
                               out[0].data_ptr(), done, d.N, d.V,
                               (float)ctx->saved_data["alpha"].toDouble(),
                               (float)ctx->saved_data["tau"].toDouble(), stream_of(logits));
        check_launch("distill_loss backward");
        return out;
    }
};

Tensor distill_loss(Tensor logits, Tensor index, Tensor teacher, OptTensor targets, double alpha,
                    double tau, double weight) {
    const bool need = at::GradMode::is_enabled() && logits.requires_grad();
    if (teacher.scalar_type() == at::kDouble) teacher = teacher.to(at::kFloat);
    if (teacher.requires_grad()) teacher = teacher.detach();
    return DistillLoss::apply(logits, index, teacher, targets, alpha, tau, weight, need);
}

// ------------------------------------------------------------------ logits of a decode step
// A per-request number as a (B,) tensor; the scalar beside it is used where there is none.
Tensor per_row(const OptTensor& t, const Tensor& logits, const char* name) {
    if (!t.has_value()) return Tensor();
    REQUIRE(t->dim() == 1 && t->size(0) == logits.size(0) && t->is_floating_point(), name,
            " must be a number or (B=", logits.size(0), ",) floating");
    check_on(*t, logits, name);
    return t->to(at::kFloat).contiguous();
}
const float* float_ptr(const Tensor& t) {
    return t.defined() ? (const float*)t.data_ptr() : nullptr;
}

Tensor adjust(Tensor logits, OptTensor history, OptTensor lengths, OptTensor prompts,
              OptTensor repetition, double repetition_all, OptTensor presence,
              double presence_all, OptTensor frequency, double frequency_all,
              OptTensor bias_index, OptTensor bias, OptTensor allowed) {
    REQUIRE(logits.is_cuda() && logits.dim() == 2, "logits must be (B, V) on GPU, got ",
            logits.sizes());
    const long B = logits.size(0), V = logits.size(1);
    REQUIRE(V <= (1 << 30) && B * ((V + 2047) / 2048) < (1l << 24),
            "logits: V at most 2^30, and fewer than 2^24 parts of 2048 columns");
    check_no_tangent("adjust_logits", {logits, repetition, presence, frequency, bias});
    const at::NoGradGuard off;
    const c10::DeviceGuard guard(logits.device());
    const int type = type_of(logits, "logits");
    const Tensor z = rows_of(logits);
    Tensor h, len, pre, bi, bv, ok;
    int h64 = 0, l64 = 0, p64 = 0, i64 = 0;
    if (history.has_value()) {
        REQUIRE(history->dim() == 2 && history->size(0) == B && history->size(1) <= (1 << 30),
                "history must be (B=", B, ", L), got ", history->sizes());
        check_on(*history, logits, "history");
        h64 = wide_index(*history, "history");
        h = rows_of(*history);
        auto per_request = [&](const OptTensor& t, Tensor& to, int& wide, const char* name) {
            if (!t.has_value()) return;
            REQUIRE(t->dim() == 1 && t->size(0) == B, name, " must be (B=", B, ",)");
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
        REQUIRE(bias.has_value() && bias_index->dim() == 2 && bias_index->size(0) == B &&
                    bias->sizes() == bias_index->sizes() && bias->size(1) <= (1 << 30) &&
                    bias->is_floating_point(),
                "bias_index must be (B=", B, ", K) and bias floating of the same shape");
        check_on(*bias_index, logits, "bias_index");
        check_on(*bias, logits, "bias");
        i64 = wide_index(*bias_index, "bias_index");
        bi = rows_of(*bias_index);
        bv = rows_of(bias->to(at::kFloat));
    }
    if (allowed.has_value()) {
        REQUIRE(allowed->dim() == 2 && allowed->size(0) == B &&
                    allowed->size(1) == (V + 31) / 32 && allowed->scalar_type() == at::kInt,
                "allowed must be (B=", B, ", ", (V + 31) / 32, ") int32");
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
// Elements of the storage from the tensor's first on: the kernels read eight at a time, past a
// row's end if need be but never past this.  Where there are not even eight, in a copy.
long room_of(const Tensor& t) {
    return (long)(t.storage().nbytes() / t.element_size()) - t.storage_offset();
}
Tensor readable(const Tensor& t) {
    if (!t.defined() || room_of(t) >= 8) return t;
    Tensor copy = at::zeros({t.numel() + 8}, t.options()).narrow(0, 0, t.numel()).view(t.sizes());
    return copy.copy_(t);
}

// A tensor of any leading shape as rows; a contiguous one without asking for a view.
struct Matrix {
    Tensor t;
    long cols = 0, stride = 0, room = 8;

    Matrix() = default;         // none
    Matrix(const Tensor& any, long rows, long n) : t(any), cols(n), stride(n) {
        if (!any.is_contiguous()) {
            t = rows_of(any.reshape({rows, n}));
            stride = row_stride(t);
        }
        if (room_of(t) < 8) {
            t = readable(t.reshape({rows, n}));
            stride = n;
        }
        room = room_of(t);
    }
    // A contiguous result: written, so as it is, whatever lies behind it.
    static Matrix result(const Tensor& out, long n) {
        Matrix m;
        m.t = out;
        m.cols = m.stride = n;
        return m;
    }
    void* data() const { return t.defined() ? t.data_ptr() : nullptr; }
};

// Rows grouped by adapter (ops/adapters.py: AdapterRows), and what every launch takes of them.
struct Grouped {
    Tensor order, segs, adapter, scale;
    std::vector<long> counts;
    int S, Bn, L, K, M, R, type;
    long T, N;
    int groups;         // adapters that have rows
    float scale_all;

    Grouped(const Tensor& x, const Tensor& y, const Tensor& a, const Tensor& b, Tensor order_,
            Tensor segs_, Tensor adapter_, std::vector<int64_t> counts_, int64_t groups_,
            const OptTensor& scale_, double all)
        : order(order_), segs(segs_), adapter(adapter_), counts(counts_.begin(), counts_.end()),
          groups((int)groups_), scale_all((float)all) {
        REQUIRE(a.dim() == 3 && b.dim() == 3 && a.size(0) == b.size(0) && a.size(2) == b.size(1),
                "a must be (L, K, R) and b (L, R, M), got ", a.sizes(), ", ", b.sizes());
        REQUIRE(a.size(2) >= 1 && a.size(2) <= 128, "rank must be in [1, 128], got ", a.size(2));
        REQUIRE(x.is_cuda() && x.dim() >= 2 && x.dim() == y.dim() &&
                    x.sizes().slice(0, x.dim() - 1) == y.sizes().slice(0, y.dim() - 1) &&
                    a.size(1) == x.size(-1) && b.size(2) == y.size(-1),
                "x must be (..., B, ", a.size(1), ") and y (..., B, ", b.size(2), "), got ",
                x.sizes(), ", ", y.sizes());
        for (const Tensor* t : {&y, &a, &b}) {
            check_on(*t, x, "every tensor");
            REQUIRE(t->scalar_type() == x.scalar_type(),
                    "y, x, a and b must have one floating type");
        }
        type = type_of(x, "x");
        REQUIRE(type != 2, "x must be bf16 or fp16");
        L = (int)a.size(0);
        K = (int)a.size(1);
        R = (int)a.size(2);
        M = (int)b.size(2);
        if (scale_.has_value()) {
            REQUIRE(scale_->dim() == 1 && scale_->size(0) == L && scale_->is_floating_point(),
                    "scale must be a number or (L=", L, ",) floating");
            REQUIRE(!scale_->requires_grad(), "scale gets no gradient: detach it");
            check_on(*scale_, x, "scale");
            scale = scale_->to(at::kFloat).contiguous();
        }
        Bn = (int)order.numel();
        S = (int)counts.size();
        REQUIRE(Bn == x.size(-2), "rows must be AdapterRows of ", x.size(-2), " columns");
        for (const Tensor* t : {&order, &segs, &adapter}) {
            check_on(*t, x, "rows");
            TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous(), "lowrank: rows int32");
        }
        // The rows may end with the call, or with the backward pass, and with a stream that is not
        // theirs still at work: their memory waits for it.
        const c10::impl::VirtualGuardImpl device(x.device().type());
        const auto stream = device.getStream(x.device());
        const Tensor* last = nullptr;
        for (const Tensor* t : {&order, &segs, &adapter}) {     // parts of one storage, as a rule
            if (!last || !t->is_alias_of(*last))
                device.recordDataPtrOnStream(t->storage().data_ptr(), stream);
            last = t;
        }
        TORCH_CHECK(a.is_contiguous() && b.is_contiguous(), "lowrank: a and b contiguous");
        TORCH_CHECK(x.numel() > 0 && y.numel() > 0, "lowrank: no rows");
        N = x.numel() / K;
        REQUIRE(K < (1 << 30) && M < (1 << 30), "rows of fewer than 2^30 elements");
        TORCH_CHECK(segs.numel() == 4l * S && adapter.numel() == Bn && N % Bn == 0,
                    "lowrank: N rows of Bn columns");
        T = N / Bn;
        long sum = 0;
        for (long c : counts) sum += c;
        TORCH_CHECK(groups <= S && groups >= S - 1 && sum == Bn, "lowrank: groups");
        REQUIRE(N < (1l << 31), "too many rows");
        check_grid(N / 64 + S, 256);                            // shrink
        check_grid((N / 256 + S) * ((M + 255) / 256), 256);     // expand, also of few rows
    }
    // A launch holds fewer than 2^32 threads.
    static void check_grid(long blocks, long threads) {
        REQUIRE(blocks * threads < (1l << 32), "too many rows or adapters for one launch");
    }
    const int* ip(const Tensor& t) const { return (const int*)t.data_ptr(); }

    // v = s x W, N rows of fp32 numbers in parts (csrc/adapters.hip); W (L, K, R) or, contraction
    // contiguous, (L, R, K)
    Tensor shrink(const Matrix& x, const Tensor& w_, bool kcont, hipStream_t st) const {
        const Tensor w = readable(w_);
        const int k = (int)x.cols, splits = lowrank_splits(counts.data(), S, T, k, 4);
        auto v = at::empty({N, (long)lowrank_row(type, R)}, w.options());
        Tensor part;
        if (splits > 1)
            part = at::empty({(long)splits * N * lowrank_width(R)}, w.options().dtype(at::kFloat));
        launch_shrink(type, kcont, x.data(), x.stride, x.room, w.data_ptr(), room_of(w), k, R,
                      ip(order), ip(segs), ip(adapter), counts.data(), S, Bn, T, float_ptr(scale),
                      scale_all, v.data_ptr(), splits > 1 ? (float*)part.data_ptr() : nullptr,
                      splits, st);
        if (splits > 1) sum(v, (const float*)part.data_ptr(), splits, st);
        check_launch("lowrank shrink");
        return v;
    }
    void sum(Tensor& v, const float* part, int splits, hipStream_t st) const {
        launch_shrink_sum(type, R, ip(order), ip(segs), ip(adapter), S, Bn, T, float_ptr(scale),
                          scale_all, v.data_ptr(), part, splits, st);
    }
    // out = base + s x A B of a few rows an adapter, in two launches
    void few(const Matrix& base, const Matrix& out, const Matrix& x, const Tensor& a_,
             const Tensor& b, hipStream_t st) const {
        const Tensor a = readable(a_);
        const int splits = lowrank_splits(counts.data(), S, T, K, 0);
        auto part = at::empty({(long)splits * N * lowrank_width(R)}, a.options().dtype(at::kFloat));
        launch_shrink(type, 0, x.data(), x.stride, x.room, a.data_ptr(), room_of(a), K, R,
                      ip(order), ip(segs), ip(adapter), counts.data(), S, Bn, T, float_ptr(scale),
                      scale_all, nullptr, (float*)part.data_ptr(), splits, st);
        launch_expand_few(type, base.data(), base.stride, out.data(), out.stride,
                          (const float*)part.data_ptr(), b.data_ptr(), M, R, ip(order), ip(segs),
                          ip(adapter), counts.data(), S, Bn, T, float_ptr(scale), scale_all,
                          splits, st);
        check_launch("lowrank few");
    }
    // out = base + v W, W (L, R, M) or, rank contiguous, (L, M, R)
    void expand(const Matrix& base, const Matrix& out, const Tensor& v, const Tensor& w_,
                bool rcont, hipStream_t st) const {
        const Tensor w = readable(w_);
        check_grid((N / 256 + S) * ((out.cols + 255) / 256), 256);
        launch_expand(type, rcont, base.data(), base.stride, base.room, out.data(), out.stride,
                      v.data_ptr(), w.data_ptr(), room_of(w), (int)out.cols, R, ip(order),
                      ip(segs), ip(adapter), counts.data(), S, Bn, T, st);
        check_launch("lowrank expand");
    }
    // sum over an adapter's rows of p^T q: (L, R, NP) or, rank contiguous, (L, NP, R).  With w
    // (L, R, NP) also `u` = s p w^T, from the same reading of p.
    Tensor outer(const Matrix& p, const Tensor& q, bool rcont, hipStream_t st,
                 const Tensor& w_ = Tensor(), Tensor* u = nullptr) const {
        const Tensor w = readable(w_);
        const int np = (int)p.cols, width = lowrank_width(R);
        const int columns = lowrank_outer_columns(counts.data(), S, T, np, R, u != nullptr);
        const int strips = (np + columns - 1) / columns;
        const int shift = lowrank_outer_shift(counts.data(), S, T, strips, columns, R);
        const long tiles = lowrank_outer_tiles(counts.data(), S, T, shift);
        const bool whole = lowrank_outer_whole(counts.data(), S, T, shift);
        check_grid(tiles * strips, 256);
        check_grid((long)L * R * ((np + 1023) / 1024), 256);    // its sum
        if (u) check_grid(N, width / 4);
        // one workspace: the gradient's parts, u's shares and a row for what belongs to no row
        const long parts = whole ? 0 : tiles * width * strips * columns;
        auto work = at::empty({parts + (u ? (strips * N + 1) * width : 0)},
                              q.options().dtype(at::kFloat));
        float* part = (float*)work.data_ptr();
        const std::vector<int64_t> size = rcont ? std::vector<int64_t>{L, np, R}
                                                : std::vector<int64_t>{L, R, np};
        // an adapter without rows has no tile to write its zeros
        auto out = whole && groups < L ? at::zeros(size, p.t.options())
                                       : at::empty(size, p.t.options());
        launch_outer(type, rcont, p.data(), p.stride, p.room, np, q.data_ptr(),
                     part, u ? w.data_ptr() : nullptr, u ? room_of(w) : 8,
                     u ? part + parts : nullptr, ip(order), ip(segs), ip(adapter),
                     counts.data(), S, Bn, T, shift, columns, whole, out.data_ptr(), R, L, st);
        if (u) {
            *u = at::empty({N, (long)lowrank_row(type, R)}, q.options());
            sum(*u, part + parts, strips, st);
        }
        check_launch("lowrank outer");
        return out;
    }
};

// y + s x A B, y and x of any leading shape over rows of Bn columns; `v`, where it is asked for,
// is x A for the backward pass.
Tensor lowrank_forward(const Grouped& g, const Tensor& y, const Tensor& x, const Tensor& a,
                       const Tensor& b, bool inplace, Tensor* v) {
    const hipStream_t st = stream_of(x);
    Tensor out = inplace ? y : at::empty(y.sizes(), y.options());
    const Matrix base(y, g.N, g.M), xr(x, g.N, g.K);
    const Matrix rows = Matrix::result(out, g.M);
    if (!v && lowrank_few(g.counts.data(), g.S, g.T)) {
        g.few(base, rows, xr, a, b, st);
        return out;
    }
    const Tensor made = g.shrink(xr, a, false, st);
    g.expand(base, rows, made, b, false, st);
    if (v) *v = made;
    return out;
}

struct LowRankAdd : public torch::autograd::Function<LowRankAdd> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, Tensor y, Tensor x, Tensor a,
                          Tensor b, Tensor order, Tensor segs, Tensor adapter,
                          std::vector<int64_t> counts, int64_t groups, OptTensor scale,
                          double scale_all) {
        const c10::DeviceGuard guard(x.device());
        const Grouped g(x, y, a, b, order, segs, adapter, counts, groups, scale, scale_all);
        Tensor v, out = lowrank_forward(g, y, x, a, b, false, &v);
        ctx->save_for_backward({x, a, b, v, order, segs, adapter, scale.value_or(Tensor())});
        ctx->saved_data["counts"] = counts;
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["scale"] = scale_all;
        ctx->saved_data["need"] = std::vector<bool>{y.requires_grad(), x.requires_grad(),
                                                    a.requires_grad(), b.requires_grad()};
        return out;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "lowrank_add is differentiable once");
        torch::autograd::variable_list out(11);
        const Tensor& dy = grads[0];
        if (!dy.defined()) return out;
        const auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &a = s[1], &b = s[2], &v = s[3];
        const c10::DeviceGuard guard(x.device());
        const Grouped g(x, dy, a, b, s[4], s[5], s[6], ctx->saved_data["counts"].toIntVector(),
                        ctx->saved_data["groups"].toInt(),
                        s[7].defined() ? OptTensor(s[7]) : OptTensor(),
                        ctx->saved_data["scale"].toDouble());
        const hipStream_t st = stream_of(x);
        const auto need = ctx->saved_data["need"].toBoolList();
        const bool need_u = need[1] || need[2];
        if (need[0]) out[0] = dy;
        if (!need_u && !need[3]) return out;
        const Matrix dr(dy, g.N, g.M);
        Tensor u;
        if (need[3] && need_u && lowrank_one_reading(g.R)) {
            out[3] = g.outer(dr, v, false, st, b, &u);
        } else {
            if (need[3]) out[3] = g.outer(dr, v, false, st);
            if (need_u) u = g.shrink(dr, b, true, st);
        }
        if (need[1]) {
            out[1] = at::empty(x.sizes(), x.options());
            g.expand(Matrix(), Matrix::result(out[1], g.K), u, a, true, st);
        }
        if (need[2]) out[2] = g.outer(Matrix(x, g.N, g.K), u, true, st);
        return out;
    }
};

Tensor lowrank_add(Tensor y, Tensor x, Tensor a, Tensor b, Tensor order, Tensor segs,
                   Tensor adapter, std::vector<int64_t> counts, int64_t groups, OptTensor scale,
                   double scale_all, bool inplace, int64_t adapters) {
    REQUIRE(a.dim() >= 1 && a.size(0) == adapters, "rows are of ", adapters, " adapters, a is ",
            a.sizes());
    check_no_tangent("lowrank_add", {y, x, a, b, scale});
    if (!inplace && at::GradMode::is_enabled() &&
        (y.requires_grad() || x.requires_grad() || a.requires_grad() || b.requires_grad()))
        return LowRankAdd::apply(y, x, a.contiguous(), b.contiguous(), order, segs, adapter,
                                 counts, groups, scale, scale_all);
    const at::NoGradGuard off;
    const c10::DeviceGuard guard(x.device());
    const Tensor ac = a.contiguous(), bc = b.contiguous();
    const Grouped g(x, y, ac, bc, order, segs, adapter, counts, groups, scale, scale_all);
    REQUIRE(!inplace || y.is_contiguous(), "y must be contiguous");
    // autograd has to see that y is another one now
    if (inplace && !y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
    return lowrank_forward(g, y, x, ac, bc, inplace, nullptr);
}

}  // namespace

void register_lm_ops(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("distill_loss", &distill_loss, "distillation from a teacher's top logits",
          py::arg("logits"), py::arg("index"), py::arg("teacher"), py::arg("targets"),
          py::arg("alpha"), py::arg("tau"), py::arg("weight"));
    m.def("adjust_logits", &adjust, "penalties, biases and masks on decode logits",
          py::arg("logits"), py::arg("history"), py::arg("lengths"), py::arg("prompt_lengths"),
          py::arg("repetition"), py::arg("repetition_all"), py::arg("presence"),
          py::arg("presence_all"), py::arg("frequency"), py::arg("frequency_all"),
          py::arg("bias_index"), py::arg("bias"), py::arg("allowed"));
    m.def("lowrank_add", &lowrank_add, "y + s x A B by rows' adapters", py::arg("y"),
          py::arg("x"), py::arg("a"), py::arg("b"), py::arg("order"), py::arg("segs"),
          py::arg("adapter"), py::arg("counts"), py::arg("groups"),
          py::arg("scale"), py::arg("scale_all"), py::arg("inplace"), py::arg("adapters"));
}
