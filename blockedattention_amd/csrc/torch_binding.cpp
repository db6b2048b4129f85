// torch extension `blockAttention`: the reference's operator surface
// (csrc/sparseBlockedAttention.cpp:118-136) on top of the C ABI in
// include/blocked_attention.h.  Host code only; compiled by the host compiler.
//
//   sparseBlockedGEMM(mat1, mat2, mat1Accum?, mat2Accum?, outAccum?, MList?, NList?, KList?,
//                     transpose1, transpose2) -> Tensor [H, Dout]
//   sparseBlockedSoftmax(src, rowList?, colList?, srcAccum?) -> Tensor [H, Dsrc]
//
// Additions that keep the reference behaviour when left at their defaults:
//   sparseBlockedSoftmaxScaled(src, rowList, colList, srcAccum?, scale)
//   sparseBlockedGEMMSoftmax(mat1, mat2, ..., scale, out_fp32)   fused pair, forward only
//   pagedResize, pagedAppend, pagedAttention, pagedTree, pagedTreeAttention, pagedKeep, pagedFork, pagedCopy
//                                                                paged key-value cache, forward only; no schedule, no
//                                                                host synchronisation
//
// Every precondition the reference leaves to assert() is a TORCH_CHECK here.
// The tensors are used as device memory only; all work happens in
// libblockedattn_hip.so on the current HIP stream.  Scheduling costs one host
// synchronisation: reading the plan summary, which carries Dout (needed to
// allocate the result) and the device-side metadata verdict.  The layers and
// heads of a model call these operators many times with the SAME metadata
// tensors, so the last few schedules are kept, keyed by the identity and the
// version counter of every metadata tensor: a repeated call launches its
// kernels at once.  set_schedule_cache(0) turns that off (needed only by a
// caller that rewrites metadata tensors behind PyTorch's back, through raw
// pointers, which the version counters cannot see).
#include <array>
#include <deque>
#include <map>
#include <memory>
#include <mutex>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <c10/core/InferenceMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "blocked_attention.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void *current_stream(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check_status(int st, const char *what) {
    TORCH_CHECK(st == BA_OK, what, ": ", ba_status_string(st), " (status ", st, ")");
}

int dtype_code(const Tensor &t, const char *name) {
    switch (t.scalar_type()) {
        case at::kHalf: return BA_F16;
        case at::kBFloat16: return BA_BF16;
        case at::kFloat: return BA_F32;
        case at::kDouble: return BA_F64;
        case at::kByte: return BA_U8;
        case at::kChar: return BA_I8;
        case at::kShort: return BA_I16;
        case at::kInt: return BA_I32;
        case at::kLong: return BA_I64;
        default: TORCH_CHECK(false, name, ": dtype ", t.scalar_type(), " is not supported");
    }
    return -1;
}

void check_data(const Tensor &t, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void check_meta(const Tensor &t, const char *name, const Tensor &like, int64_t n) {
    check_data(t, name);
    TORCH_CHECK(t.scalar_type() == at::kLong, name, " must be int64");
    TORCH_CHECK(t.device() == like.device(), name, " must be on the same device as the data");
    TORCH_CHECK(t.dim() == 1 && t.numel() == n, name, " must be 1-D with ", n, " entries, got ", t.sizes());
}

int64_t leading(const Tensor &t) {
    int64_t h = 1;
    for (int64_t d = 0; d + 1 < t.dim(); ++d) h *= t.size(d);
    return h;
}

struct Schedule;
// Schedules derived from one schedule (permuted shapes for the two GEMMs of the backward pass), made on first
// use and shared by every copy of the schedule, so that they live and die with its cache entry.
struct Derived {
    std::mutex mu;
    std::shared_ptr<Schedule> grad1, grad2;
    Tensor summary;                                 // of this schedule, as the tensor that autograd nodes keep
};

struct Schedule {
    Tensor accum1, accum2, accumOut, M, N, K;
    Tensor plan;
    ba_plan_info info;
    std::shared_ptr<Derived> derived;
};

// ---------------------------------------------------------------- schedule cache
struct ScheduleKey {
    int kind = 0;                                   // 0 GEMM, 1 softmax
    int device = -1;
    std::array<const void *, 6> impl{};             // TensorImpl of each metadata tensor (nullptr: not given)
    std::array<int64_t, 6> version{};
    bool cacheable = true;
    bool operator==(const ScheduleKey &o) const {
        return kind == o.kind && device == o.device && impl == o.impl && version == o.version;
    }
};

ScheduleKey make_key(int kind, const Tensor &like, std::initializer_list<const OptTensor *> metas) {
    ScheduleKey k;
    k.kind = kind;
    k.device = like.device().index();
    size_t i = 0;
    for (const OptTensor *m : metas) {
        if (m->has_value() && (*m)->defined()) {
            if ((*m)->is_inference()) k.cacheable = false;      // no version counter to watch
            else { k.impl[i] = (*m)->unsafeGetTensorImpl(); k.version[i] = (int64_t)(*m)->_version(); }
        }
        ++i;
    }
    return k;
}

struct ScheduleCache {
    std::mutex mu;
    std::deque<std::pair<ScheduleKey, Schedule>> entries;       // most recent first; entries keep their tensors alive
    size_t capacity = 8;
    int64_t hits = 0, misses = 0;
};
ScheduleCache &cache() {
    static ScheduleCache c;
    return c;
}

bool cache_lookup(const ScheduleKey &key, Schedule &out) {
    ScheduleCache &c = cache();
    std::lock_guard<std::mutex> lock(c.mu);
    if (c.capacity == 0 || !key.cacheable) return false;
    for (auto it = c.entries.begin(); it != c.entries.end(); ++it) {
        if (it->first == key) {
            out = it->second;
            if (it != c.entries.begin()) {
                auto e = *it;
                c.entries.erase(it);
                c.entries.push_front(std::move(e));
            }
            ++c.hits;
            return true;
        }
    }
    ++c.misses;
    return false;
}

void cache_store(const ScheduleKey &key, const Schedule &s) {
    ScheduleCache &c = cache();
    std::lock_guard<std::mutex> lock(c.mu);
    if (c.capacity == 0 || !key.cacheable) return;
    c.entries.emplace_front(key, s);
    while (c.entries.size() > c.capacity) c.entries.pop_back();
}

void set_schedule_cache(int64_t capacity) {
    TORCH_CHECK(capacity >= 0 && capacity <= 1024, "schedule cache capacity must be in [0, 1024]");
    ScheduleCache &c = cache();
    std::lock_guard<std::mutex> lock(c.mu);
    c.capacity = (size_t)capacity;
    while (c.entries.size() > c.capacity) c.entries.pop_back();
}

std::vector<int64_t> schedule_cache_stats() {
    ScheduleCache &c = cache();
    std::lock_guard<std::mutex> lock(c.mu);
    return {c.hits, c.misses, (int64_t)c.entries.size(), (int64_t)c.capacity};
}

// Where a scheduler launch hands its summaries to the host: BA_MAILBOX_BYTES of pinned, GPU-writable memory per
// plan (up to three) and calling thread (allocated at the thread's first schedule, kept for the life of the process) and a ticket that
// changes with every use.  The host then spins on the ticket instead of copying and synchronising the stream.
struct Mailbox {
    void *mem = nullptr;
    uint32_t ticket = 0;
    Mailbox() {
        if (hipHostMalloc(&mem, 3 * BA_MAILBOX_BYTES, hipHostMallocCoherent | hipHostMallocMapped | hipHostMallocPortable) != hipSuccess) mem = nullptr;
        else memset(mem, 0, 3 * BA_MAILBOX_BYTES);
    }
};
Mailbox &mailbox() {
    static thread_local Mailbox m;
    return m;
}

// The three metadata cases of the reference (cpp:17-44), resolved on the device.
Schedule schedule_gemm(const Tensor &like, const OptTensor &a1, const OptTensor &a2, const OptTensor &aO,
                       const OptTensor &M, const OptTensor &N, const OptTensor &K, bool use_cache = true,
                       bool train = false) {
    const bool have_accum = a1.has_value() && a2.has_value() && aO.has_value();
    const bool have_lists = M.has_value() && N.has_value() && K.has_value();
    TORCH_CHECK(have_accum || have_lists,
                "sparseBlockedGEMM needs either (mat1Accum, mat2Accum, outAccum) or (MList, NList, KList)");
    Schedule s;
    const ScheduleKey key = make_key(0, like, {&a1, &a2, &aO, &M, &N, &K});
    if (use_cache && cache_lookup(key, s)) return s;
    // A schedule made in inference mode may serve a call that saves its tensors for a backward pass.
    c10::InferenceMode normal_tensors(false);
    s.derived = std::make_shared<Derived>();
    int64_t nseg;
    int mode;
    const auto opts = at::TensorOptions().dtype(at::kLong).device(like.device());
    if (have_lists) {
        nseg = M->numel();
        check_meta(*M, "MList", like, nseg); check_meta(*N, "NList", like, nseg); check_meta(*K, "KList", like, nseg);
        s.M = *M; s.N = *N; s.K = *K;
    }
    if (have_accum) {
        nseg = a1->numel() - 1;
        TORCH_CHECK(nseg >= 0, "prefix sums need at least one entry");
        check_meta(*a1, "mat1Accum", like, nseg + 1); check_meta(*a2, "mat2Accum", like, nseg + 1);
        check_meta(*aO, "outAccum", like, nseg + 1);
        if (have_lists) TORCH_CHECK(s.M.numel() == nseg, "lists and prefix sums disagree on the segment count");
        s.accum1 = *a1; s.accum2 = *a2; s.accumOut = *aO;
    }
    if (have_lists && have_accum) {
        mode = BA_META_GIVEN;
    } else if (have_lists) {
        mode = BA_META_FROM_LISTS;
        s.accum1 = at::empty({nseg + 1}, opts); s.accum2 = at::empty({nseg + 1}, opts);
        s.accumOut = at::empty({nseg + 1}, opts);
    } else {
        mode = BA_META_FROM_ACCUM;
        s.M = at::empty({nseg}, opts); s.N = at::empty({nseg}, opts); s.K = at::empty({nseg}, opts);
    }
    const size_t bytes = ba_plan_bytes(nseg);
    s.plan = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(like.device()));
    void *stream = current_stream(like);
    Mailbox &mb = mailbox();
    int st;
    if (mb.mem) {
        const uint32_t ticket = ++mb.ticket ? mb.ticket : ++mb.ticket;       // never 0, the mailbox's first content
        int64_t *const m = s.M.data_ptr<int64_t>(), *const n = s.N.data_ptr<int64_t>(), *const k = s.K.data_ptr<int64_t>();
        int64_t *const o1 = s.accum1.data_ptr<int64_t>(), *const o2 = s.accum2.data_ptr<int64_t>(),
                *const oO = s.accumOut.data_ptr<int64_t>();
        if (train) {
            // the backward products' plans in the same launch (the same verdict and summaries as if made one by one)
            auto g1 = std::make_shared<Schedule>(), g2 = std::make_shared<Schedule>();
            g1->plan = at::empty_like(s.plan); g2->plan = at::empty_like(s.plan);
            g1->derived = std::make_shared<Derived>(); g2->derived = std::make_shared<Derived>();
            check_status(ba_plan_gemm_train_notify(s.plan.data_ptr(), g1->plan.data_ptr(), g2->plan.data_ptr(), bytes, nseg,
                                                   mode, m, n, k, o1, o2, oO, mb.mem, ticket, stream),
                         "ba_plan_gemm_train_notify");
            st = ba_plan_wait(mb.mem, ticket, &s.info, 60 * 1000 * 1000);
            char *const mem = static_cast<char *>(mb.mem);
            const int st1 = ba_plan_wait(mem + BA_MAILBOX_BYTES, ticket, &g1->info, 60 * 1000 * 1000);
            const int st2 = ba_plan_wait(mem + 2 * BA_MAILBOX_BYTES, ticket, &g2->info, 60 * 1000 * 1000);
            if (st1 == BA_OK) s.derived->grad1 = std::move(g1);      // else the backward pass makes it, and reports
            if (st2 == BA_OK) s.derived->grad2 = std::move(g2);
        } else {
            check_status(ba_plan_gemm_notify(s.plan.data_ptr(), bytes, nseg, mode, m, n, k, o1, o2, oO, mb.mem, ticket, stream),
                         "ba_plan_gemm_notify");
            st = ba_plan_wait(mb.mem, ticket, &s.info, 60 * 1000 * 1000);
        }
    } else {
        check_status(ba_plan_gemm(s.plan.data_ptr(), bytes, nseg, mode, s.M.data_ptr<int64_t>(),
                                  s.N.data_ptr<int64_t>(), s.K.data_ptr<int64_t>(), s.accum1.data_ptr<int64_t>(),
                                  s.accum2.data_ptr<int64_t>(), s.accumOut.data_ptr<int64_t>(), stream),
                     "ba_plan_gemm");
        st = ba_plan_read(s.plan.data_ptr(), &s.info, stream);
    }
    TORCH_CHECK(st != BA_ERR_BAD_METADATA, "segment metadata rejected: ", s.info.bad_segments,
                " segment(s) have negative, oversized or inconsistent shapes / prefix sums");
    check_status(st, "ba_plan_read");
    if (use_cache) cache_store(key, s);
    return s;
}

Schedule schedule_softmax(const Tensor &like, const Tensor &rows, const Tensor &cols, const OptTensor &accum) {
    Schedule s;
    const OptTensor rows_o(rows), cols_o(cols), none;
    const ScheduleKey key = make_key(1, like, {&rows_o, &cols_o, &accum, &none, &none, &none});
    if (cache_lookup(key, s)) return s;
    c10::InferenceMode normal_tensors(false);
    s.derived = std::make_shared<Derived>();
    const int64_t nseg = rows.numel();
    check_meta(rows, "rowList", like, nseg); check_meta(cols, "colList", like, nseg);
    s.M = rows; s.N = cols;
    if (accum.has_value()) {
        check_meta(*accum, "srcAccum", like, nseg + 1);
        s.accumOut = *accum;
    } else {
        s.accumOut = at::empty({nseg + 1}, at::TensorOptions().dtype(at::kLong).device(like.device()));
    }
    const size_t bytes = ba_plan_bytes(nseg);
    s.plan = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(like.device()));
    void *stream = current_stream(like);
    Mailbox &mb = mailbox();
    int st;
    if (mb.mem) {
        const uint32_t ticket = ++mb.ticket ? mb.ticket : ++mb.ticket;
        check_status(ba_plan_softmax_notify(s.plan.data_ptr(), bytes, nseg, rows.data_ptr<int64_t>(), cols.data_ptr<int64_t>(),
                                            s.accumOut.data_ptr<int64_t>(), accum.has_value() ? 1 : 0, mb.mem, ticket, stream),
                     "ba_plan_softmax_notify");
        st = ba_plan_wait(mb.mem, ticket, &s.info, 60 * 1000 * 1000);
    } else {
        check_status(ba_plan_softmax(s.plan.data_ptr(), bytes, nseg, rows.data_ptr<int64_t>(), cols.data_ptr<int64_t>(),
                                     s.accumOut.data_ptr<int64_t>(), accum.has_value() ? 1 : 0, stream),
                     "ba_plan_softmax");
        st = ba_plan_read(s.plan.data_ptr(), &s.info, stream);
    }
    TORCH_CHECK(st != BA_ERR_BAD_METADATA, "segment metadata rejected: ", s.info.bad_segments,
                " segment(s) have negative or oversized shapes or a prefix sum too small for them");
    check_status(st, "ba_plan_read");
    cache_store(key, s);
    return s;
}

// sparseBlockedGEMMLaunch (h:18; GEMM.cu:985-1033): result is always [H, Dout] in mat1's dtype.
Tensor gemm_launch(const Tensor &mat1, const Tensor &mat2, Schedule &s, bool t1, bool t2) {
    check_data(mat1, "mat1"); check_data(mat2, "mat2");
    TORCH_CHECK(mat1.scalar_type() == mat2.scalar_type(), "mat1 and mat2 must have the same dtype, got ",
                mat1.scalar_type(), " and ", mat2.scalar_type());
    TORCH_CHECK(mat1.device() == mat2.device(), "mat1 and mat2 must be on the same device");
    TORCH_CHECK(mat1.dim() >= 1 && mat2.dim() >= 1, "mat1 and mat2 need a last dimension");
    TORCH_CHECK(mat1.size(-1) == s.info.Dm1, "mat1.size(-1) = ", mat1.size(-1), " but the segments need ", s.info.Dm1);
    TORCH_CHECK(mat2.size(-1) == s.info.Dm2, "mat2.size(-1) = ", mat2.size(-1), " but the segments need ", s.info.Dm2);
    const int64_t H = leading(mat1);
    TORCH_CHECK(leading(mat2) == H, "mat1 and mat2 disagree on the number of heads");
    const int dt = dtype_code(mat1, "sparseBlockedGEMM");
    Tensor out = at::empty({H, s.info.Dout}, mat1.options());
    check_status(ba_varlen_gemm(s.plan.data_ptr(), &s.info, s.info.nseg, dt, mat1.data_ptr(), mat2.data_ptr(), out.data_ptr(), H,
                                s.info.Dm1, s.info.Dm2, s.info.Dout, t1, t2, current_stream(mat1)),
                 "ba_varlen_gemm");
    return out;
}

// The schedule of one of the two backward products of s (permuted metadata, given in both forms), made once and
// kept with s: it lives and dies with the forward schedule and takes no slot of the cache.
Schedule &derived_schedule(const Schedule &s, std::shared_ptr<Schedule> Derived::*slot, const Tensor &like,
                           const Tensor &a1, const Tensor &a2, const Tensor &aO, const Tensor &rows, const Tensor &cols,
                           const Tensor &reduce) {
    TORCH_CHECK(s.derived, "internal: schedule without a holder for derived schedules");
    std::lock_guard<std::mutex> lock(s.derived->mu);
    std::shared_ptr<Schedule> &p = (*s.derived).*slot;
    if (!p)
        p = std::make_shared<Schedule>(schedule_gemm(like, OptTensor(a1), OptTensor(a2), OptTensor(aO), OptTensor(rows),
                                                     OptTensor(cols), OptTensor(reduce), /*use_cache=*/false));
    return *p;
}

// What an autograd node keeps of a schedule from its forward to its backward pass: two tensors, the plan and a copy of
// its summary, saved like the operands (a capsule or raw bytes in the node's other data would shut it out of compiled
// autograd, which hashes those).  The copy is made once and shared by the nodes of the schedule.
void keep_schedule(variable_list &saved, const Schedule &s) {
    std::lock_guard<std::mutex> lock(s.derived->mu);
    Tensor &summary = s.derived->summary;
    if (!summary.defined()) {
        c10::InferenceMode normal_tensors(false);
        summary = at::empty({(int64_t)sizeof(ba_plan_info)}, at::TensorOptions().dtype(at::kByte).device(at::kCPU));
        memcpy(summary.data_ptr(), &s.info, sizeof(ba_plan_info));
    }
    saved.push_back(s.plan);
    saved.push_back(summary);
}
// The schedule of saved[at] and saved[at + 1].  Saved-tensor hooks may have put them anywhere (a summary that comes back
// on the GPU is copied once more); what is not a plan and its summary any longer is refused.
Schedule kept_schedule(const variable_list &saved, size_t at, const Tensor &like) {
    Schedule s;
    s.plan = saved[at];
    const Tensor info = saved[at + 1].is_cpu() ? saved[at + 1] : saved[at + 1].to(at::kCPU);
    TORCH_CHECK(info.scalar_type() == at::kByte && info.is_contiguous() && info.numel() == (int64_t)sizeof(ba_plan_info),
                "backward: the saved summary of the plan came back as ", info.toString(), info.sizes());
    memcpy(&s.info, info.data_ptr(), sizeof(ba_plan_info));
    check_data(s.plan, "backward: the saved plan");
    TORCH_CHECK(s.plan.scalar_type() == at::kByte && s.plan.device() == like.device() && s.info.nseg >= 0 &&
                    s.plan.numel() == (int64_t)ba_plan_bytes(s.info.nseg) && ((uintptr_t)s.plan.data_ptr() & 15) == 0,
                "backward: the saved plan came back as ", s.plan.toString(), s.plan.sizes());
    return s;
}
// An operand or result that comes back for the backward pass (through whatever hooks there are), `last` elements a head.
void check_kept(const Tensor &t, const char *name, const Tensor &like, int64_t H, int64_t last) {
    check_data(t, name);
    TORCH_CHECK(t.device() == like.device() && t.dim() >= 1 && t.size(-1) == last && leading(t) == H, "backward: the saved ", name,
                " came back as ", t.toString(), t.sizes(), ", not ", H, " x ", last);
}

class SparseBlockedGEMM : public torch::autograd::Function<SparseBlockedGEMM> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &mat1, const Tensor &mat2, const OptTensor &a1,
                                 const OptTensor &a2, const OptTensor &aO, const OptTensor &M, const OptTensor &N,
                                 const OptTensor &K, bool t1, bool t2, bool train) {
        check_data(mat1, "mat1"); check_data(mat2, "mat2");
        c10::hip::HIPGuardMasqueradingAsCUDA guard(mat1.device());
        Schedule s = schedule_gemm(mat1, a1, a2, aO, M, N, K, /*use_cache=*/true, train);
        variable_list keep{mat1, mat2, s.accum1, s.accum2, s.accumOut, s.M, s.N, s.K};
        if (train) {
            std::lock_guard<std::mutex> lock(s.derived->mu);
            if (s.derived->grad1 && s.derived->grad2) {
                keep_schedule(keep, *s.derived->grad1);
                keep_schedule(keep, *s.derived->grad2);
            }
        }
        ctx->save_for_backward(keep);
        ctx->saved_data["transpose1"] = t1;
        ctx->saved_data["transpose2"] = t2;
        return {gemm_launch(mat1, mat2, s, t1, t2)};
    }

    // dA = dS B and dB = dS^T A as two more varlen GEMMs with permuted metadata
    // (cpp:52-72); like the reference, the gradient layouts are those of the
    // untransposed forward.
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor grad = grads[0].contiguous();
        c10::hip::HIPGuardMasqueradingAsCUDA guard(grad.device());
        const Tensor mat1 = saved[0].to(grad.scalar_type()), mat2 = saved[1].to(grad.scalar_type());
        const Tensor &a1 = saved[2], &a2 = saved[3], &aO = saved[4], &M = saved[5], &N = saved[6], &K = saved[7];
        const bool t1 = ctx->saved_data["transpose1"].toBool(), t2 = ctx->saved_data["transpose2"].toBool();
        Tensor g1, g2;
        // dS and the saved operands are read as they lie: the products whose reduction runs over N or M take the
        // kernels for any layout and reduction length (two launches, like the reference)
        Schedule s1, s2;
        if (saved.size() > 8) {
            s1 = kept_schedule(saved, 8, grad);
            s2 = kept_schedule(saved, 10, grad);
        } else {                                       // the forward's schedule was made by a call without gradients
            const Schedule fwd = schedule_gemm(grad, a1, a2, aO, M, N, K);
            s1 = derived_schedule(fwd, &Derived::grad1, grad, aO, a2, a1, M, K, N);
            s2 = derived_schedule(fwd, &Derived::grad2, grad, aO, a1, a2, N, K, M);
        }
        const int64_t heads = leading(grad);
        check_kept(mat1, "mat1", grad, heads, s2.info.Dm2);
        check_kept(mat2, "mat2", grad, heads, s1.info.Dm2);
        // batches of short segments: both products as ONE launch where the library offers it (layouts of the
        // untransposed forward), else one call each
        bool done = false;
        if (!t1 && !t2 && grad.dim() >= 1 && grad.size(-1) == s1.info.Dm1 && grad.size(-1) == s2.info.Dm1 &&
            (grad.scalar_type() == at::kHalf || grad.scalar_type() == at::kBFloat16)) {
            g1 = at::empty({heads, s1.info.Dout}, grad.options());
            g2 = at::empty({heads, s2.info.Dout}, grad.options());
            const int st = ba_varlen_gemm_two(dtype_code(grad, "sparseBlockedGEMM backward"), heads, s1.plan.data_ptr(), &s1.info,
                                              grad.data_ptr(), mat2.data_ptr(), g1.data_ptr(), s1.info.Dm1, s1.info.Dm2,
                                              s1.info.Dout, s2.plan.data_ptr(), &s2.info, grad.data_ptr(), mat1.data_ptr(),
                                              g2.data_ptr(), s2.info.Dm1, s2.info.Dm2, s2.info.Dout, current_stream(grad));
            if (st == BA_OK) done = true;
            else if (st != BA_ERR_UNSUPPORTED) check_status(st, "ba_varlen_gemm_two");
        }
        if (!done) {
            g1 = gemm_launch(grad, mat2, s1, false, !t2);
            g2 = gemm_launch(grad, mat1, s2, true, !t1);
        }
        return {g1.view_as(saved[0]), g2.view_as(saved[1]), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(),
                Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

class SparseBlockedSoftmax : public torch::autograd::Function<SparseBlockedSoftmax> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &src, const OptTensor &rows,
                                 const OptTensor &cols, const OptTensor &accum, double scale) {
        TORCH_CHECK(rows.has_value() && cols.has_value(), "sparseBlockedSoftmax needs rowList and colList");
        check_data(src, "src");
        c10::hip::HIPGuardMasqueradingAsCUDA guard(src.device());
        Schedule s = schedule_softmax(src, *rows, *cols, accum);
        TORCH_CHECK(src.dim() >= 1 && src.size(-1) == s.info.Dout, "src.size(-1) = ", src.size(-1),
                    " but the segments need ", s.info.Dout);
        const int64_t H = leading(src);
        const int dt = dtype_code(src, "sparseBlockedSoftmax");
        Tensor out = at::empty({H, s.info.Dout}, src.options());
        check_status(ba_blocked_softmax(s.plan.data_ptr(), &s.info, s.info.nseg, dt, src.data_ptr(), out.data_ptr(), H,
                                        s.info.Dout, (float)scale, current_stream(src)),
                     "ba_blocked_softmax");
        // (the metadata only so that a change of it between the passes is refused by its version counter)
        variable_list keep{out, s.accumOut, s.M, s.N};
        keep_schedule(keep, s);
        ctx->save_for_backward(keep);
        ctx->saved_data["scale"] = scale;
        return {out};
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor grad = grads[0].contiguous();
        c10::hip::HIPGuardMasqueradingAsCUDA guard(grad.device());
        const Tensor y = saved[0].to(grad.scalar_type());
        const Schedule s = kept_schedule(saved, 4, grad);
        const int64_t H = leading(grad);
        check_kept(grad, "gradient", grad, H, s.info.Dout); check_kept(y, "result", grad, H, s.info.Dout);
        Tensor dx = at::empty_like(y);
        check_status(ba_blocked_softmax_backward(s.plan.data_ptr(), &s.info, s.info.nseg,
                                                 dtype_code(y, "softmax backward"),
                                                 y.data_ptr(), grad.data_ptr(), dx.data_ptr(), H, s.info.Dout,
                                                 (float)ctx->saved_data["scale"].toDouble(), current_stream(y)),
                     "ba_blocked_softmax_backward");
        return {dx, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// ------------------------------------------------------------------ the ops
Tensor sparseBlockedGEMM_op(const Tensor &mat1, const Tensor &mat2, const OptTensor &mat1Accum,
                            const OptTensor &mat2Accum, const OptTensor &outAccum, const OptTensor &MList,
                            const OptTensor &NList, const OptTensor &KList, bool transpose1, bool transpose2) {
    const bool train = at::GradMode::is_enabled() && (mat1.requires_grad() || mat2.requires_grad());
    return SparseBlockedGEMM::apply(mat1, mat2, mat1Accum, mat2Accum, outAccum, MList, NList, KList, transpose1,
                                    transpose2, train)[0];
}

Tensor sparseBlockedSoftmax_op(const Tensor &src, const OptTensor &rowList, const OptTensor &colList,
                               const OptTensor &srcAccum) {
    return SparseBlockedSoftmax::apply(src, rowList, colList, srcAccum, 1.0)[0];
}

Tensor sparseBlockedSoftmaxScaled_op(const Tensor &src, const OptTensor &rowList, const OptTensor &colList,
                                     const OptTensor &srcAccum, double scale) {
    return SparseBlockedSoftmax::apply(src, rowList, colList, srcAccum, scale)[0];
}

// Fused softmax(scale * A_g B_g^T): forward only, scores never leave registers.
Tensor sparseBlockedGEMMSoftmax_op(const Tensor &mat1, const Tensor &mat2, const OptTensor &mat1Accum,
                                   const OptTensor &mat2Accum, const OptTensor &outAccum, const OptTensor &MList,
                                   const OptTensor &NList, const OptTensor &KList, double scale, bool out_fp32) {
    check_data(mat1, "mat1"); check_data(mat2, "mat2");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(mat1.device());
    TORCH_CHECK(mat1.scalar_type() == mat2.scalar_type(), "mat1 and mat2 must have the same dtype");
    TORCH_CHECK(mat1.scalar_type() == at::kHalf || mat1.scalar_type() == at::kBFloat16,
                "the fused GEMM + softmax takes fp16 or bf16 operands");
    TORCH_CHECK(mat1.device() == mat2.device(), "mat1 and mat2 must be on the same device");
    Schedule s = schedule_gemm(mat1, mat1Accum, mat2Accum, outAccum, MList, NList, KList);
    TORCH_CHECK(mat1.size(-1) == s.info.Dm1 && mat2.size(-1) == s.info.Dm2,
                "operand sizes do not match the segments: need ", s.info.Dm1, " and ", s.info.Dm2);
    const int64_t H = leading(mat1);
    TORCH_CHECK(leading(mat2) == H, "mat1 and mat2 disagree on the number of heads");
    Tensor out = at::empty({H, s.info.Dout}, out_fp32 ? mat1.options().dtype(at::kFloat) : mat1.options());
    check_status(ba_gemm_softmax(s.plan.data_ptr(), &s.info, s.info.nseg, dtype_code(mat1, "fused"), mat1.data_ptr(),
                                 mat2.data_ptr(), out.data_ptr(), out_fp32 ? BA_F32 : dtype_code(mat1, "fused"), H,
                                 s.info.Dm1, s.info.Dm2, s.info.Dout, (float)scale, current_stream(mat1)),
                 "ba_gemm_softmax");
    return out;
}

// softmax(scale * Q_g K_g^T) V_g in one pass, the probabilities never written.  Q is the M x K operand of the segments,
// K and V are both N x K; the result is [H, Dm1].  With lse, the rows' sums for the backward pass too.
Tensor attention_launch(const Tensor &q, const Tensor &k, const Tensor &v, Schedule &s, double scale, Tensor *lse) {
    TORCH_CHECK(q.size(-1) == s.info.Dm1 && k.size(-1) == s.info.Dm2 && v.size(-1) == s.info.Dm2,
                "operand sizes do not match the segments: need ", s.info.Dm1, " (q) and ", s.info.Dm2, " (k, v)");
    TORCH_CHECK(s.info.max_K <= 128, "the one-pass attention takes head dimensions up to 128, got ", s.info.max_K);
    const int64_t H = leading(q);
    TORCH_CHECK(leading(k) == H && leading(v) == H, "q, k and v disagree on the number of heads");
    Tensor out = at::empty({H, s.info.Dm1}, q.options());
    const int dt = dtype_code(q, "attention");
    void *stream = current_stream(q);
    if (!lse) {
        check_status(ba_varlen_attention(s.plan.data_ptr(), &s.info, s.info.nseg, dt, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                         out.data_ptr(), H, s.info.Dm1, s.info.Dm2, s.info.Dout, (float)scale, stream),
                     "ba_varlen_attention");
        return out;
    }
    *lse = at::empty({H, ba_attention_rows(&s.info, s.info.Dm1)}, q.options().dtype(at::kFloat));
    check_status(ba_varlen_attention_train(s.plan.data_ptr(), &s.info, s.info.nseg, dt, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                           out.data_ptr(), lse->data_ptr<float>(), H, s.info.Dm1, s.info.Dm2, s.info.Dout,
                                           (float)scale, stream),
                 "ba_varlen_attention_train");
    return out;
}

Schedule attention_schedule(const Tensor &q, const Tensor &k, const Tensor &v, const OptTensor &a1, const OptTensor &a2,
                            const OptTensor &aO, const OptTensor &M, const OptTensor &N, const OptTensor &K) {
    TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
                "q, k and v must have the same dtype");
    TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16,
                "the one-pass attention takes fp16 or bf16 operands");
    TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), "q, k and v must be on the same device");
    return schedule_gemm(q, a1, a2, aO, M, N, K);
}

// Differentiable form.  Between the passes it keeps the operands, the result, the rows' sums and the plan with its
// summary: nothing of the size M x N, and the backward pass schedules nothing.  As with the operators this stands in
// for, the result may be changed in place before the backward pass.
class SparseBlockedAttention : public torch::autograd::Function<SparseBlockedAttention> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const OptTensor &a1,
                                 const OptTensor &a2, const OptTensor &aO, const OptTensor &M, const OptTensor &N,
                                 const OptTensor &K, double scale) {
        Schedule s = attention_schedule(q, k, v, a1, a2, aO, M, N, K);
        Tensor lse;
        Tensor out = attention_launch(q, k, v, s, scale, &lse);
        // The result is kept without its version counter, so that a caller may write on it; `watch`, an empty tensor with
        // that counter, tells the backward pass, which then makes the result again.
        variable_list keep{q, k, v, out.variable_data(), lse};
        keep_schedule(keep, s);
        ctx->save_for_backward(keep);
        Tensor watch = at::empty({0}, at::TensorOptions().dtype(at::kByte).device(at::kCPU));
        torch::autograd::impl::set_version_counter(watch, torch::autograd::impl::version_counter(out));
        ctx->saved_data["watch"] = watch;
        ctx->saved_data["version"] = (int64_t)watch._version();
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["lists"] = M.has_value() && N.has_value() && K.has_value();
        return {out};
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        TORCH_CHECK(ctx->saved_data["lists"].toBool(), "blockFusedAttention: the backward pass needs MList, NList and KList");
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &kept = saved[3], &lse = saved[4];
        const Tensor grad = grads[0].to(q.scalar_type()).contiguous();
        c10::hip::HIPGuardMasqueradingAsCUDA guard(grad.device());
        Schedule s = kept_schedule(saved, 5, grad);
        const ba_plan_info &info = s.info;
        const int64_t H = leading(grad);
        check_kept(grad, "gradient", grad, H, info.Dm1); check_kept(kept, "result", grad, H, info.Dm1);
        check_kept(q, "q", grad, H, info.Dm1); check_kept(k, "k", grad, H, info.Dm2); check_kept(v, "v", grad, H, info.Dm2);
        check_kept(lse, "row sums", grad, H, ba_attention_rows(&info, info.Dm1));
        for (const Tensor *t : {&q, &k, &v, &kept})
            TORCH_CHECK(t->scalar_type() == grad.scalar_type(), "backward: a saved operand came back as ", t->toString());
        const double scale = ctx->saved_data["scale"].toDouble();
        const bool changed = (int64_t)ctx->saved_data["watch"].toTensor()._version() != ctx->saved_data["version"].toInt();
        const Tensor out = changed ? attention_launch(q, k, v, s, scale, nullptr) : kept;
        Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v), delta = at::empty_like(lse);
        check_status(ba_varlen_attention_backward(s.plan.data_ptr(), &info, info.nseg, dtype_code(q, "attention backward"),
                                                  q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), grad.data_ptr(),
                                                  lse.data_ptr<float>(), delta.data_ptr<float>(), dq.data_ptr(),
                                                  dk.data_ptr(), dv.data_ptr(), H, info.Dm1, info.Dm2, info.Dout,
                                                  (float)scale, current_stream(q)),
                     "ba_varlen_attention_backward");
        return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor sparseBlockedAttention_op(const Tensor &q, const Tensor &k, const Tensor &v, const OptTensor &mat1Accum,
                                 const OptTensor &mat2Accum, const OptTensor &outAccum, const OptTensor &MList,
                                 const OptTensor &NList, const OptTensor &KList, double scale) {
    check_data(q, "q"); check_data(k, "k"); check_data(v, "v");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
        return SparseBlockedAttention::apply(q, k, v, mat1Accum, mat2Accum, outAccum, MList, NList, KList, scale)[0];
    Schedule s = attention_schedule(q, k, v, mat1Accum, mat2Accum, outAccum, MList, NList, KList);
    return attention_launch(q, k, v, s, scale, nullptr);
}

// ------------------------------------------------------------ paged key-value cache
// Operands are read by their strides; only the last dimension has to be contiguous.
void check_rows(const Tensor &t, const char *name, const Tensor &like) {
    TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
    TORCH_CHECK(t.device() == like.device(), name, " must be on the same device as the cache");
    TORCH_CHECK(t.dim() >= 1 && (t.stride(-1) == 1 || t.size(-1) <= 1), name, ": the last dimension must be contiguous");
}

// [heads, rows * dim] or [heads, rows, dim], as head and row strides in elements.
struct Rows {
    int64_t heads, rows, head_stride, row_stride;
};
Rows rows_of(const Tensor &t, const char *name, int64_t dim) {
    TORCH_CHECK(t.dim() == 2 || t.dim() == 3, name, " must be [heads, rows * dim] or [heads, rows, dim], got ", t.sizes());
    if (t.dim() == 3) {
        TORCH_CHECK(t.size(2) == dim, name, ": the cache holds rows of ", dim, " elements, got ", t.sizes());
        return {t.size(0), t.size(1), t.stride(0), t.stride(1)};
    }
    TORCH_CHECK(t.size(1) % dim == 0, name, ": the cache holds rows of ", dim, " elements, got ", t.sizes());
    return {t.size(0), t.size(1) / dim, t.stride(0), dim};
}

void check_no_grad(std::initializer_list<const Tensor *> tensors, const OptTensor &k_scale, const OptTensor &v_scale, const char *op) {
    std::vector<const Tensor *> all(tensors);
    for (const OptTensor *s : {&k_scale, &v_scale})
        if (s->has_value()) all.push_back(&**s);
    for (const Tensor *t : all)
        TORCH_CHECK(!(at::GradMode::is_enabled() && t->requires_grad()), op, " has no backward pass: detach its operands or use torch.no_grad()");
}

// A kernel has written behind PyTorch's back: what watches version counters is told.
void written(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// moved: what the cache holds is only moved, so nobody needs its scales.
ba_paged_cache cache_of(const Tensor &k, const Tensor &v, const OptTensor &k_scale, const OptTensor &v_scale, bool moved = false) {
    check_rows(k, "kCache", k); check_rows(v, "vCache", k);
    TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes(), "kCache and vCache must both be [pages, heads, page, dim], got ", k.sizes(), " and ", v.sizes());
    TORCH_CHECK(k.scalar_type() == v.scalar_type(), "kCache and vCache must have the same dtype");
    ba_paged_cache c{};
    const bool f8 = k.scalar_type() == at::kFloat8_e4m3fn;
    TORCH_CHECK(f8 || k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16,
                "a paged cache holds fp16, bf16 or float8_e4m3fn, got ", k.scalar_type());
    TORCH_CHECK(moved || (k_scale.has_value() == f8 && v_scale.has_value() == f8),
                f8 ? "a float8_e4m3fn cache needs kScale and vScale" : "kScale and vScale belong to a float8_e4m3fn cache");
    TORCH_CHECK(k.size(1) >= 1 && k.size(2) >= 1 && k.size(3) >= 1 && k.size(3) <= 256,
                "a paged cache has at least one head, one token a page and 1 to 256 dimensions, got ", k.sizes());
    if (f8 && !moved)
        for (const OptTensor *s : {&k_scale, &v_scale}) {
            check_data(**s, "kScale and vScale");
            TORCH_CHECK((*s)->scalar_type() == at::kFloat && (*s)->dim() == 1 && (*s)->numel() == k.size(1) && (*s)->device() == k.device(),
                        "kScale and vScale are fp32, one entry per head of the cache (", k.size(1), "), on its device");
        }
    c.k = k.data_ptr(); c.v = v.data_ptr();
    c.k_scale = f8 && !moved ? k_scale->data_ptr<float>() : nullptr; c.v_scale = f8 && !moved ? v_scale->data_ptr<float>() : nullptr;
    c.pages = k.size(0); c.heads = k.size(1); c.page = k.size(2); c.dim = k.size(3);
    c.k_page_stride = k.stride(0); c.k_head_stride = k.stride(1); c.k_token_stride = k.stride(2);
    c.v_page_stride = v.stride(0); c.v_head_stride = v.stride(1); c.v_token_stride = v.stride(2);
    c.dtype = f8 ? BA_F8_E4M3 : k.scalar_type() == at::kHalf ? BA_F16 : BA_BF16;
    return c;
}

void check_cache_operand(const Tensor &t, const char *name, const ba_paged_cache &c) {
    TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name, " must be fp16 or bf16, got ", t.scalar_type());
    TORCH_CHECK(c.dtype == BA_F8_E4M3 || c.dtype == (t.scalar_type() == at::kHalf ? BA_F16 : BA_BF16), name, " must have the cache's dtype");
}

void check_table(const Tensor &table, const Tensor &like) {
    check_rows(table, "table", like);
    TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2, "table must be int32 [requests, pages of a request]");
}

std::vector<Tensor> pagedResize_op(const Tensor &table, const Tensor &free_pages, const Tensor &state, const Tensor &lens,
                                   const Tensor &new_lens, int64_t page, int64_t tokens) {
    check_table(table, table);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(table.device());
    const int64_t R = table.size(0);
    TORCH_CHECK(page >= 1, "a page holds at least one token");
    TORCH_CHECK(tokens >= 0, "tokens must not be negative");
    check_data(free_pages, "free");
    TORCH_CHECK(free_pages.scalar_type() == at::kInt && free_pages.dim() == 1 && free_pages.device() == table.device(),
                "free must be 1-D int32 on the table's device");
    check_meta(state, "state", table, 2); check_meta(lens, "lens", table, R); check_meta(new_lens, "newLens", table, R);
    const auto opts = lens.options();
    Tensor slots = at::empty({tokens}, opts), accum = at::empty({R + 1}, opts), lens_out = at::empty({R}, opts), state_out = at::empty({2}, opts);
    const size_t bytes = ba_paged_resize_workspace(R);
    Tensor work;
    if (bytes) work = at::empty({(int64_t)bytes}, opts.dtype(at::kByte));
    check_status(ba_paged_resize(table.data_ptr<int32_t>(), table.stride(0), table.size(1), free_pages.data_ptr<int32_t>(), free_pages.numel(),
                                 state.data_ptr<int64_t>(), lens.data_ptr<int64_t>(), new_lens.data_ptr<int64_t>(), R, page,
                                 slots.data_ptr<int64_t>(), tokens, accum.data_ptr<int64_t>(), lens_out.data_ptr<int64_t>(),
                                 state_out.data_ptr<int64_t>(), bytes ? work.data_ptr() : nullptr, bytes, current_stream(table)),
                 "ba_paged_resize");
    written(table); written(free_pages);
    return {slots, accum, lens_out, state_out};
}

void pagedAppend_op(const Tensor &k, const Tensor &v, const Tensor &k_cache, const Tensor &v_cache, const Tensor &slots,
                    const OptTensor &k_scale, const OptTensor &v_scale) {
    const ba_paged_cache c = cache_of(k_cache, v_cache, k_scale, v_scale);
    check_rows(k, "k", k_cache); check_rows(v, "v", k_cache);
    check_no_grad({&k, &v, &k_cache, &v_cache}, k_scale, v_scale, "pagedAppend");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(k_cache.device());
    check_cache_operand(k, "k", c);
    TORCH_CHECK(k.scalar_type() == v.scalar_type(), "k and v must have the same dtype");
    const Rows kr = rows_of(k, "k", c.dim), vr = rows_of(v, "v", c.dim);
    TORCH_CHECK(kr.heads == c.heads && vr.heads == c.heads, "k and v must have the cache's ", c.heads, " heads, got ", kr.heads, " and ", vr.heads);
    TORCH_CHECK(kr.rows == vr.rows, "k and v disagree on the number of tokens");
    check_meta(slots, "slots", k_cache, kr.rows);
    check_status(ba_paged_append(&c, dtype_code(k, "pagedAppend"), k.data_ptr(), kr.head_stride, kr.row_stride, v.data_ptr(),
                                 vr.head_stride, vr.row_stride, slots.data_ptr<int64_t>(), kr.rows, current_stream(k_cache)),
                 "ba_paged_append");
    written(k_cache); written(v_cache);
}

// The counters of ba_paged_attention, zeros that every call leaves as zeros: kept for each of PyTorch's own streams, on
// which calls follow each other (and which live as long as the process).  A call that is being captured may be replayed on
// any stream, and a stream from elsewhere may end and its handle come back while its work still runs: those get
// counters of their own.
Tensor paged_counters(const Tensor &like) {
    const auto opts = at::TensorOptions().dtype(at::kInt).device(like.device());
    const c10::hip::HIPStream stream = c10::hip::getCurrentHIPStream(like.device().index());
    hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
    const int64_t id = stream.unwrap().id();
    const bool foreign = id != 0 && (id & 1) == 0;           // such ids are the stream's address
    if (foreign || hipStreamIsCapturing(stream.stream(), &capturing) != hipSuccess || capturing != hipStreamCaptureStatusNone)
        return at::zeros({BA_PAGED_COUNTERS}, opts);
    static std::mutex mu;
    static auto *kept = new std::map<std::pair<int, int64_t>, Tensor>;       // never taken down: the GPU may be gone by then
    std::lock_guard<std::mutex> lock(mu);
    Tensor &t = (*kept)[{(int)like.device().index(), id}];
    if (!t.defined()) {
        c10::InferenceMode normal_tensors(false);
        t = at::zeros({BA_PAGED_COUNTERS}, opts);
    }
    return t;
}

Tensor pagedAttention_op(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &table, const Tensor &lens,
                         double scale, int64_t window, const OptTensor &k_scale, const OptTensor &v_scale) {
    const ba_paged_cache c = cache_of(k_cache, v_cache, k_scale, v_scale);
    check_rows(q, "q", k_cache);
    check_table(table, k_cache);
    check_no_grad({&q, &k_cache, &v_cache}, k_scale, v_scale, "pagedAttention");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(k_cache.device());
    check_cache_operand(q, "q", c);
    TORCH_CHECK(window >= 0, "window must not be negative (0: all tokens)");
    const Rows qr = rows_of(q, "q", c.dim);
    TORCH_CHECK(qr.heads >= 1 && qr.heads % c.heads == 0, "q must have a multiple of the cache's ", c.heads, " heads, got ", qr.heads);
    TORCH_CHECK(table.size(0) == qr.rows, "q has ", qr.rows, " rows, table ", table.size(0));
    check_meta(lens, "lens", k_cache, qr.rows);
    // q's order of dimensions; but where rows of q overlap that may put the last dimension, which the kernel writes in one
    // piece, outside another
    Tensor out = at::empty_like(q);
    if (out.size(-1) > 1 && out.stride(-1) != 1) out = at::empty(q.sizes(), q.options());
    const Rows outr = rows_of(out, "out", c.dim);
    const size_t bytes = ba_paged_attention_workspace(&c, qr.heads, qr.rows, table.size(1));
    Tensor work;
    if (bytes) work = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    const Tensor counters = paged_counters(q);
    check_status(ba_paged_attention(&c, dtype_code(q, "pagedAttention"), q.data_ptr(), qr.head_stride, qr.row_stride, qr.heads, qr.rows,
                                    table.data_ptr<int32_t>(), table.stride(0), table.size(1), lens.data_ptr<int64_t>(), window, (float)scale,
                                    out.data_ptr(), outr.head_stride, outr.row_stride, counters.data_ptr<int32_t>(), bytes ? work.data_ptr() : nullptr, bytes,
                                    current_stream(q)),
                 "ba_paged_attention");
    return out;
}

std::vector<Tensor> pagedTree_op(const Tensor &parents, const Tensor &accum, int64_t nodes) {
    check_data(accum, "accum");
    TORCH_CHECK(accum.dim() == 1 && accum.numel() >= 1, "accum has one entry more than requests");
    check_meta(accum, "accum", accum, accum.numel());
    TORCH_CHECK(parents.dim() == 1, "parents must be 1-D");
    check_meta(parents, "parents", accum, parents.numel());
    TORCH_CHECK(nodes >= 1 && nodes <= BA_PAGED_TREE_NODES, "nodes must be 1 to ", BA_PAGED_TREE_NODES, ", got ", nodes);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(accum.device());
    const int64_t T = parents.numel();
    Tensor mask = at::empty({T, (nodes + 63) / 64}, accum.options()), depth = at::empty({T}, accum.options());
    check_status(ba_paged_tree(parents.data_ptr<int64_t>(), accum.data_ptr<int64_t>(), accum.numel() - 1, T, nodes, mask.data_ptr<int64_t>(),
                               depth.data_ptr<int64_t>(), current_stream(accum)),
                 "ba_paged_tree");
    return {mask, depth};
}

Tensor pagedTreeAttention_op(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &table, const Tensor &lens,
                             const Tensor &accum, const OptTensor &mask, double scale, int64_t window, const OptTensor &k_scale,
                             const OptTensor &v_scale) {
    const ba_paged_cache c = cache_of(k_cache, v_cache, k_scale, v_scale);
    check_rows(q, "q", k_cache);
    check_table(table, k_cache);
    check_no_grad({&q, &k_cache, &v_cache}, k_scale, v_scale, "pagedTreeAttention");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(k_cache.device());
    check_cache_operand(q, "q", c);
    TORCH_CHECK(window >= 0, "window must not be negative (0: all tokens)");
    const Rows qr = rows_of(q, "q", c.dim);
    TORCH_CHECK(qr.heads >= 1 && qr.heads % c.heads == 0, "q must have a multiple of the cache's ", c.heads, " heads, got ", qr.heads);
    const int64_t R = table.size(0);
    check_meta(lens, "lens", k_cache, R); check_meta(accum, "accum", k_cache, R + 1);
    if (mask.has_value()) {
        check_rows(*mask, "mask", k_cache);
        TORCH_CHECK(mask->scalar_type() == at::kLong && mask->dim() == 2 && mask->size(0) == qr.rows && mask->size(1) >= 1,
                    "mask must be int64 [", qr.rows, ", words], a row for each of q, got ", mask->sizes());
    }
    Tensor out = at::empty_like(q);
    if (out.size(-1) > 1 && out.stride(-1) != 1) out = at::empty(q.sizes(), q.options());        // (as in pagedAttention)
    const Rows outr = rows_of(out, "out", c.dim);
    const size_t bytes = ba_paged_tree_attention_workspace(&c, qr.heads, qr.rows, R, table.size(1));
    Tensor work;
    if (bytes) work = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    const Tensor counters = paged_counters(q);
    check_status(ba_paged_tree_attention(&c, dtype_code(q, "pagedTreeAttention"), q.data_ptr(), qr.head_stride, qr.row_stride, qr.heads, qr.rows,
                                         table.data_ptr<int32_t>(), table.stride(0), table.size(1), lens.data_ptr<int64_t>(),
                                         accum.data_ptr<int64_t>(), R, mask.has_value() ? mask->data_ptr<int64_t>() : nullptr,
                                         mask.has_value() ? mask->stride(0) : 0, mask.has_value() ? mask->size(1) : 0, window, (float)scale,
                                         out.data_ptr(), outr.head_stride, outr.row_stride, counters.data_ptr<int32_t>(),
                                         bytes ? work.data_ptr() : nullptr, bytes, current_stream(q)),
                 "ba_paged_tree_attention");
    return out;
}

Tensor pagedKeep_op(const Tensor &k_cache, const Tensor &v_cache, const Tensor &table, const Tensor &lens, const Tensor &path) {
    const ba_paged_cache c = cache_of(k_cache, v_cache, {}, {}, true);
    check_table(table, k_cache);
    check_no_grad({&k_cache, &v_cache}, {}, {}, "pagedKeep");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(k_cache.device());
    const int64_t R = table.size(0);
    check_meta(lens, "lens", k_cache, R);
    check_rows(path, "path", k_cache);
    TORCH_CHECK(path.scalar_type() == at::kLong && path.dim() == 2 && path.size(0) == R, "path must be int64 [", R, ", nodes], got ", path.sizes());
    Tensor out = at::empty({R}, lens.options());
    check_status(ba_paged_keep(&c, table.data_ptr<int32_t>(), table.stride(0), table.size(1), lens.data_ptr<int64_t>(), path.data_ptr<int64_t>(),
                               path.stride(0), R, path.size(1), out.data_ptr<int64_t>(), current_stream(k_cache)),
                 "ba_paged_keep");
    written(k_cache); written(v_cache);
    return out;
}

std::vector<Tensor> pagedFork_op(const Tensor &table, const Tensor &free_pages, const Tensor &state, const Tensor &shares, const Tensor &lens,
                                 const Tensor &origin, int64_t page) {
    check_table(table, table);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(table.device());
    const int64_t R = table.size(0);
    TORCH_CHECK(page >= 1, "a page holds at least one token");
    TORCH_CHECK(R <= BA_PAGED_FORK_ROWS, "pagedFork takes up to ", BA_PAGED_FORK_ROWS, " rows, got ", R);
    check_data(free_pages, "free"); check_data(shares, "shares");
    for (const Tensor *t : {&free_pages, &shares})
        TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1 && t->device() == table.device(), "free and shares must be 1-D int32 on the table's device");
    check_meta(state, "state", table, 2); check_meta(lens, "lens", table, R); check_meta(origin, "origin", table, R);
    Tensor table_out = at::empty({R, table.size(1)}, table.options()), lens_out = at::empty({R}, lens.options()), state_out = at::empty({2}, lens.options());
    Tensor shares_out = at::empty({shares.numel()}, shares.options()), source = at::empty({R}, table.options()), target = at::empty({R}, table.options());
    const size_t bytes = ba_paged_fork_workspace(R, shares.numel());
    Tensor work = at::empty({(int64_t)bytes}, table.options().dtype(at::kByte));
    check_status(ba_paged_fork(table.data_ptr<int32_t>(), table.stride(0), table.size(1), free_pages.data_ptr<int32_t>(), free_pages.numel(),
                               state.data_ptr<int64_t>(), shares.data_ptr<int32_t>(), shares.numel(), lens.data_ptr<int64_t>(),
                               origin.data_ptr<int64_t>(), R, page, table_out.data_ptr<int32_t>(), table_out.stride(0), lens_out.data_ptr<int64_t>(),
                               state_out.data_ptr<int64_t>(), shares_out.data_ptr<int32_t>(), source.data_ptr<int32_t>(), target.data_ptr<int32_t>(),
                               work.data_ptr(), bytes, current_stream(table)),
                 "ba_paged_fork");
    written(free_pages);
    return {table_out, lens_out, state_out, shares_out, source, target};
}

void pagedCopy_op(const Tensor &k_cache, const Tensor &v_cache, const Tensor &source, const Tensor &target) {
    const ba_paged_cache c = cache_of(k_cache, v_cache, {}, {}, true);
    check_no_grad({&k_cache, &v_cache}, {}, {}, "pagedCopy");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(k_cache.device());
    check_data(source, "source"); check_data(target, "target");
    for (const Tensor *t : {&source, &target})
        TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1 && t->numel() == source.numel() && t->device() == k_cache.device(),
                    "source and target must be 1-D int32 of one length on the cache's device");
    check_status(ba_paged_copy(&c, source.data_ptr<int32_t>(), target.data_ptr<int32_t>(), source.numel(), current_stream(k_cache)), "ba_paged_copy");
    written(k_cache); written(v_cache);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("sparseBlockedGEMM", &sparseBlockedGEMM_op, "sparseBlockedGEMM forward");
    m.def("sparseBlockedSoftmax", &sparseBlockedSoftmax_op, "sparseBlockedSoftmax forward");
    m.def("sparseBlockedSoftmaxScaled", &sparseBlockedSoftmaxScaled_op, "sparseBlockedSoftmax with a fused scale");
    m.def("sparseBlockedGEMMSoftmax", &sparseBlockedGEMMSoftmax_op, "fused sparseBlockedGEMM + softmax forward");
    m.def("sparseBlockedAttention", &sparseBlockedAttention_op, "softmax(scale q k^T) v per segment, one pass");
    m.def("pagedResize", &pagedResize_op, "page tables and slots from the requests' lengths before and after");
    m.def("pagedAppend", &pagedAppend_op, "keys and values of new tokens into a paged cache, in place");
    m.def("pagedAttention", &pagedAttention_op, "one query per request over a paged cache");
    m.def("pagedTree", &pagedTree_op, "what the nodes of trees of drafted tokens see, and how deep they lie");
    m.def("pagedTreeAttention", &pagedTreeAttention_op, "several queries per request over a paged cache, of a tree of drafted tokens");
    m.def("pagedKeep", &pagedKeep_op, "an accepted path's keys and values to consecutive places, in place");
    m.def("pagedFork", &pagedFork_op, "rows of a page table that go on from other rows");
    m.def("pagedCopy", &pagedCopy_op, "pages of a cache to other pages, in place");
    m.def("set_schedule_cache", &set_schedule_cache, "number of schedules kept for repeated metadata (0 = off)");
    m.def("schedule_cache_stats", &schedule_cache_stats, "[hits, misses, entries, capacity]");
}
