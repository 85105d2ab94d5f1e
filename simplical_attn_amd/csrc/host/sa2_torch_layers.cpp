// Host path of the operators of ordinary attention layers (rotary positions, causal attention over prompts, rows of a
// cache, drafted trees): checks, outputs, workspaces, the calls of the C ABI and the autograd formulas.
#include <c10/core/DeviceGuard.h>
#include <c10/core/InferenceMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <vector>

#include "sa2_torch.h"

namespace sa2_host {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

decltype(&sa2_rotary) rotary_fn = nullptr;
decltype(&sa2_cache_append) append_fn = nullptr;
decltype(&sa2_causal_forward) causal_fwd_fn = nullptr;
decltype(&sa2_causal_bwd_workspace_bytes) causal_ws_fn = nullptr;
decltype(&sa2_causal_backward) causal_bwd_fn = nullptr;
decltype(&sa2_window_forward) window_fwd_fn = nullptr;
decltype(&sa2_window_bwd_workspace_bytes) window_ws_fn = nullptr;
decltype(&sa2_window_backward) window_bwd_fn = nullptr;
decltype(&sa2_tree_workspace_bytes) tree_ws_fn = nullptr;
decltype(&sa2_tree_attention) tree_fn = nullptr;
decltype(&sa2_window_tree_workspace_bytes) window_tree_ws_fn = nullptr;
decltype(&sa2_window_tree_attention) window_tree_fn = nullptr;
decltype(&sa2_key_weights_workspace_bytes) key_weights_ws_fn = nullptr;
decltype(&sa2_key_weights) key_weights_fn = nullptr;
decltype(&sa2_cache_evict) evict_fn = nullptr;

// ---- checks ----------------------------------------------------------------------------------------------------------
// The first tensor of a call: [batch, rows, heads, head_dim], or packed [rows, heads, head_dim]
void check_first(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.dim() == 4 || t.dim() == 3, name, ": expected [batch, seq_len, heads, head_dim] or packed [rows, heads, head_dim], got ", t.sizes());
    TORCH_CHECK_TYPE(dtype_code(t) >= 0, name, ": unsupported dtype ", t.scalar_type(), " (float32, bfloat16, float16)");
}
// One that goes with it: same leading sizes, head_dim, dtype and device
void check_beside(const Tensor& t, const char* name, const Tensor& q, const char* first) {
    TORCH_CHECK_VALUE(t.dim() == q.dim() && t.size(-1) == q.size(-1) && t.size(0) == q.size(0) && (q.dim() == 3 || t.size(1) == q.size(1)), name, ": ",
                      t.sizes(), " does not go with ", first, " ", q.sizes());
    TORCH_CHECK_VALUE(t.scalar_type() == q.scalar_type() && t.device() == q.device(), name, " must match ", first, " in dtype and device");
}
void check_heads(const Tensor& q, const Tensor& k) {
    TORCH_CHECK_VALUE(k.size(-2) >= 1 && q.size(-2) % k.size(-2) == 0, "the ", q.size(-2), " query heads are not a multiple of the ", k.size(-2), " heads of keys and values");
}
void check_ints(const Maybe& t, const char* name, const Tensor& q, int64_t dim) {
    if (!t) return;
    TORCH_CHECK_VALUE(t->scalar_type() == at::kInt && t->dim() == dim, name, " must be an int32 tensor of ", dim, " dimension(s), got ", t->scalar_type(), " ", t->sizes());
    TORCH_CHECK_VALUE(t->device() == q.device(), name, " must be on the device of the other tensors");
}
void check_cu(const Maybe& cu, const Tensor& q) {
    check_ints(cu, "cu_seqlens", q, 1);
    TORCH_CHECK_VALUE(!cu || (q.dim() == 3 && cu->numel() >= 2), "cu_seqlens needs packed [rows, heads, head_dim] tensors and at least two entries");
}
// While the operators work.  They are no dispatcher operators: a dispatch mode of the user (FLOP counting, selective checkpointing) sees
// nothing of them, neither a call nor what is allocated inside.  Modes that record or fake operators would miss the kernels: refused.
struct Unseen {
    explicit Unseen(const char* op) {
        if (!c10::impl::dispatch_mode_enabled()) return;
        using Key = c10::impl::TorchDispatchModeKey;
        for (const Key key : {Key::FAKE, Key::PROXY, Key::FUNCTIONAL})
            TORCH_CHECK(!c10::impl::TorchDispatchModeTLS::get_mode(key), op, " cannot run under fake tensors, make_fx or functionalization: no dispatcher operator stands for it");
        guard.emplace(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot}));
    }
    std::optional<c10::impl::ExcludeDispatchKeyGuard> guard;
};
void check_place(const char* op, std::initializer_list<Tensor> ts) {
    for (const Tensor& t : ts) {
        TORCH_CHECK(t.is_cuda(), op, " runs on the GPU only; got a ", t.device(), " tensor");
        TORCH_CHECK(!t._fw_grad(0).defined() && (t.key_set() & at::kTensorSubclassLike).empty(), op, " takes plain tensors: no forward-mode derivatives, torch.func transforms or tensor subclasses");
    }
    TORCH_CHECK(!torch::jit::tracer::isTracing(), op, " cannot be recorded by torch.jit.trace");
}

// ---- tensors as the C ABI takes them -----------------------------------------------------------------------------------
// Unit stride along head_dim and positive strides on every axis longer than 1; anything else is copied
bool strided(const Tensor& t) {
    bool ok = t.stride(-1) == 1 || t.size(-1) == 1;
    for (int64_t a = 0; a + 1 < t.dim(); ++a) ok = ok && (t.stride(a) > 0 || t.size(a) == 1);
    return ok;
}
Tensor rows(const Tensor& t) { return strided(t) ? t : t.contiguous(); }
void put_strides(int64_t* s, const Tensor& t) {
    const bool batched = t.dim() == 4;
    s[0] = batched ? t.stride(0) : 0;
    s[1] = t.stride(batched ? 1 : 0);
    s[2] = t.stride(batched ? 2 : 1);
}
struct Sizes {
    int B, N, H, D;
};
Sizes sizes(const Tensor& t) {
    const bool batched = t.dim() == 4;
    TORCH_CHECK_VALUE(t.numel() <= (int64_t)1 << 40 && t.size(0) < ((int64_t)1 << 31) && t.size(1) < ((int64_t)1 << 31) && t.size(-2) < ((int64_t)1 << 31), "sizes beyond 2^31: ", t.sizes());
    return {batched ? (int)t.size(0) : 1, (int)t.size(batched ? 1 : 0), (int)t.size(-2), (int)t.size(-1)};
}
Tensor like(const Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous)); }
void* stream(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
const int32_t* ints(const Tensor& t) { return t.defined() ? t.const_data_ptr<int32_t>() : nullptr; }
Tensor dense(const Maybe& t) { return t ? t->contiguous() : Tensor(); }

// ---- rotary ----------------------------------------------------------------------------------------------------------
struct Angles {
    Tensor frequencies, positions, cu;         // the last two may be undefined
    double amplitude;
    bool interleaved, inverse;
};

std::pair<Tensor, Tensor> run_rotary(const Tensor& q_, const Tensor& k_, const Angles& a) {
    const Unseen unseen("rotary_embedding");
    const Tensor q = rows(q_), k = k_.defined() ? rows(k_) : Tensor();
    const c10::DeviceGuard guard(q.device());
    Tensor q2 = like(q), k2 = k.defined() ? like(k) : Tensor();
    const Sizes z = sizes(q);
    const int hk = k.defined() ? sizes(k).H : 0;
    if (z.B == 0 || z.N == 0 || z.D == 0 || (z.H == 0 && hk == 0)) return {q2, k2};
    if (z.H == 0) return {q2, run_rotary(k, Tensor(), a).first};
    int64_t s[12] = {};
    put_strides(s, q);
    put_strides(s + 6, q2);
    if (hk) {
        put_strides(s + 3, k);
        put_strides(s + 9, k2);
    }
    check(rotary_fn(q.const_data_ptr(), hk ? k.const_data_ptr() : nullptr, q2.data_ptr(), hk ? k2.data_ptr() : nullptr, a.frequencies.const_data_ptr<double>(),
                    a.positions.defined() ? a.positions.const_data_ptr() : nullptr, a.positions.defined() ? (int)a.positions.element_size() : 0, ints(a.cu),
                    a.cu.defined() ? (int)a.cu.numel() - 1 : 0, z.B, z.N, z.H, hk, z.D, (int)(2 * a.frequencies.numel()), s, (float)a.amplitude, a.interleaved, a.inverse,
                    dtype_code(q), stream(q)));
    return {q2, k2};
}

std::pair<Tensor, Tensor> turn(const Tensor& q, const Tensor& k, const Angles& a);

// (its backward is the same operator, so it has derivatives of every order)
struct RotaryFormula : torch::autograd::Function<RotaryFormula> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Maybe& k, Angles a) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({a.frequencies, a.positions, a.cu});
        ctx->saved_data["amplitude"] = a.amplitude;
        ctx->saved_data["interleaved"] = a.interleaved;
        ctx->saved_data["inverse"] = a.inverse;
        auto [q2, k2] = run_rotary(q, k ? *k : Tensor(), a);
        return k2.defined() ? variable_list{q2, k2} : variable_list{q2};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Angles a{s[0], s[1], s[2], ctx->saved_data["amplitude"].toDouble(), ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool()};
        Tensor dq = ctx->needs_input_grad(0) ? grads[0] : Tensor(), dk = grads.size() > 1 && ctx->needs_input_grad(1) ? grads[1] : Tensor();
        if (dq.defined()) std::tie(dq, dk) = turn(dq, dk, a);
        else if (dk.defined()) dk = turn(dk, Tensor(), a).first;
        return {dq, dk, Tensor()};
    }
};

// `k` may be undefined
std::pair<Tensor, Tensor> turn(const Tensor& q, const Tensor& k, const Angles& a) {
    if (at::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()))) {
        auto r = RotaryFormula::apply(q, k.defined() ? Maybe(k) : Maybe(), a);
        return {r[0], k.defined() ? r[1] : Tensor()};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return run_rotary(q, k, a);
}

std::pair<Tensor, Maybe> rotary(const Tensor& q, const Maybe& k, const Tensor& frequencies, const Maybe& positions, const Maybe& cu, bool interleaved, double amplitude) {
    check_first(q, "q");
    if (k) check_beside(*k, "k", q, "q");
    TORCH_CHECK_VALUE(q.size(-1) <= 256, "head_dim ", q.size(-1), " is above 256");
    TORCH_CHECK_VALUE(frequencies.dim() == 1 && frequencies.scalar_type() == at::kDouble && frequencies.device() == q.device(), "frequencies must be a float64 vector on q's device");
    TORCH_CHECK_VALUE(frequencies.numel() >= 1 && 2 * frequencies.numel() <= q.size(-1), "frequencies turn ", 2 * frequencies.numel(), " columns, head_dim is ", q.size(-1));
    TORCH_CHECK_VALUE(!frequencies.requires_grad(), "rotary_embedding has no gradient for frequencies");
    check_cu(cu, q);
    if (positions) {
        TORCH_CHECK_VALUE(!cu, "give positions or cu_seqlens, not both");
        TORCH_CHECK_VALUE(positions->scalar_type() == at::kInt || positions->scalar_type() == at::kLong, "positions must be int32 or int64");
        TORCH_CHECK_VALUE(positions->sizes() == q.sizes().slice(0, q.dim() - 2) && positions->device() == q.device(), "positions ", positions->sizes(), " must have q's leading sizes and device");
    }
    check_place("rotary_embedding", {q});
    if (k) check_place("rotary_embedding", {*k});
    const Angles a{frequencies.contiguous(), dense(positions), dense(cu), amplitude, interleaved, false};
    py::gil_scoped_release nogil;
    auto [q2, k2] = turn(q, k ? *k : Tensor(), a);
    return {q2, k ? Maybe(k2) : Maybe()};
}

// ---- cache -----------------------------------------------------------------------------------------------------------
// A cache's two tensors and what finds rows in them; `beside` has the rows' heads and head_dim
struct CacheView {
    Tensor k, v, lengths, table;
    int page_size, pages, width;
};
CacheView check_cache(const Tensor& k_cache, const Tensor& v_cache, const Tensor& lengths, const Maybe& table, const Tensor& k, int64_t sequences) {
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(k_cache, "k_cache"), {v_cache, "v_cache"}}) {
        TORCH_CHECK_VALUE(t.dim() == 4 && t.size(2) == k.size(-2) && t.size(3) == k.size(-1) && t.sizes() == k_cache.sizes(), name,
                          ": expected [pages, page_size, ", k.size(-2), ", ", k.size(-1), "], got ", t.sizes());
        TORCH_CHECK_VALUE(t.scalar_type() == k.scalar_type() && t.device() == k.device(), name, " must match k in dtype and device");
        TORCH_CHECK_VALUE(strided(t), name, " needs unit stride along head_dim and positive strides: it is used in place");
        TORCH_CHECK_VALUE(t.size(0) >= 1 && t.size(1) >= 1 && t.size(0) < ((int64_t)1 << 31) && t.size(1) < ((int64_t)1 << 31), name, ": a cache needs at least one page of one row, got ", t.sizes());
    }
    check_ints(lengths, "lengths", k, 1);
    TORCH_CHECK_VALUE(lengths.numel() == sequences, "lengths has ", lengths.numel(), " entries for ", sequences, " sequences");
    check_ints(table, "page_table", k, 2);
    TORCH_CHECK_VALUE(!table || (table->size(0) == sequences && table->size(1) >= 1), "page_table ", table ? table->sizes() : at::IntArrayRef(), " must be [", sequences, ", pages of a sequence]");
    if (!table) TORCH_CHECK_VALUE(k_cache.size(0) == sequences, "without a page_table the cache is [sequences, capacity, heads, head_dim]: got ", k_cache.size(0), " pieces for ", sequences, " sequences");
    return {k_cache, v_cache, lengths.contiguous(), dense(table), (int)k_cache.size(1), (int)k_cache.size(0), table ? (int)table->size(1) : 1};
}

// Whether the memory from a tensor's first element to its last meets the other's
bool meet(const Tensor& a, const Tensor& b) {
    auto end = [](const Tensor& t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        return (const char*)t.const_data_ptr() + (last + 1) * t.element_size();
    };
    return (const char*)a.const_data_ptr() < end(b) && (const char*)b.const_data_ptr() < end(a);
}

// Bytes from one element to another are sums of these: `stride` times any number from lo to hi
struct Steps {
    int64_t stride, lo, hi;
};
// Whether the steps from `i` on (longest first) can add up to `bytes`; a search of too many turns, of axes that reach over one another, counts as yes
bool reaches(const std::vector<Steps>& steps, size_t i, int64_t bytes, int& turns) {
    if (i == steps.size()) return bytes == 0;
    int64_t least = 0, most = 0;               // of the others
    for (size_t j = i + 1; j < steps.size(); ++j) {
        least += steps[j].stride * steps[j].lo;
        most += steps[j].stride * steps[j].hi;
    }
    const Steps& s = steps[i];
    const auto down = [&](int64_t x) { return x / s.stride - (x % s.stride < 0); };
    for (int64_t n = std::max(s.lo, -down(most - bytes)); n <= std::min(s.hi, down(bytes - least)); ++n)
        if (--turns < 0 || reaches(steps, i + 1, bytes - n * s.stride, turns)) return true;
    return false;
}
// Whether two tensors with positive strides have a byte in common.  Halves of one buffer, whose elements lie between each other, have none.
bool share(const Tensor& a, const Tensor& b) {
    if (a.numel() == 0 || b.numel() == 0 || !meet(a, b)) return false;
    const int64_t size = a.element_size();
    std::vector<Steps> steps{{1, 1 - size, size - 1}};
    const auto add = [&](int64_t stride, int64_t lo, int64_t hi) {
        for (Steps& s : steps)
            if (s.stride == stride) {
                s.lo += lo;
                s.hi += hi;
                return;
            }
        steps.push_back({stride, lo, hi});
    };
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1) add(a.stride(i) * size, 0, a.size(i) - 1);
    for (int64_t i = 0; i < b.dim(); ++i)
        if (b.size(i) > 1) add(b.stride(i) * size, 1 - b.size(i), 0);
    std::sort(steps.begin(), steps.end(), [](const Steps& x, const Steps& y) { return x.stride > y.stride; });
    int turns = 4096;
    return reaches(steps, 0, (const char*)b.const_data_ptr() - (const char*)a.const_data_ptr(), turns);
}
// Whether two elements of one tensor (with positive strides) have memory in common
bool folded(const Tensor& t) {
    std::vector<Steps> steps;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) steps.push_back({t.stride(i), 1 - t.size(i), t.size(i) - 1});
    std::sort(steps.begin(), steps.end(), [](const Steps& x, const Steps& y) { return x.stride > y.stride; });
    int turns = 4096;
    int64_t inner = 0;                         // what the shorter steps reach
    for (size_t i = steps.size(); i-- > 0;) {
        const Steps& s = steps[i];
        for (int64_t n = 1; n <= std::min(s.hi, inner / s.stride); ++n)
            if (--turns < 0 || reaches(steps, i + 1, n * s.stride, turns)) return true;
        inner += s.hi * s.stride;
    }
    return false;
}

void check_added(const Tensor& t) {
    TORCH_CHECK_VALUE(strided(t), "weights need unit stride along the places and positive strides: they are added to in place");
    TORCH_CHECK_VALUE(t.numel() == 0 || !folded(t), "weights of different places share memory: they are added to in place");
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), "weights are added to in place and have no gradient: call it under torch.no_grad() or on detached tensors");
    TORCH_CHECK(c10::InferenceMode::is_enabled() || !t.is_inference(), "weights are changed in place, which inference tensors allow in inference mode only");
}
// The weights that the rows of a cache have gathered, of `heads` heads each: changed in place where `written`
void check_weights(const Tensor& t, const CacheView& c, int64_t heads, bool written) {
    const int64_t capacity = (int64_t)c.page_size * c.width;
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.dim() == 3 && t.size(0) == c.lengths.numel() && t.size(1) == heads && t.size(2) >= capacity, "weights must be float32 [",
                      c.lengths.numel(), ", ", heads, ", ", capacity, " or more], got ", t.scalar_type(), " ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == c.k.device(), "weights must be on the device of the other tensors");
    TORCH_CHECK_VALUE(strided(t), "weights need unit stride along the places and positive strides");
    if (written) check_added(t);
}

void append(const Tensor& k_, const Tensor& v_, const Tensor& k_cache, const Tensor& v_cache, const Tensor& lengths, const Maybe& table, const Maybe& chosen, const Maybe& cu) {
    check_first(k_, "k");
    check_beside(v_, "v", k_, "k");
    TORCH_CHECK_VALUE(k_.size(-2) == v_.size(-2), "k and v differ in heads: ", k_.sizes(), ", ", v_.sizes());
    TORCH_CHECK_VALUE(k_.size(-1) >= 1 && k_.size(-1) <= 256 && k_.size(-2) >= 1, "heads and head_dim must be at least 1, head_dim at most 256: ", k_.sizes());
    check_cu(cu, k_);
    TORCH_CHECK_VALUE(k_.dim() == 4 || cu, "packed rows need cu_seqlens");
    const int64_t sequences = cu ? cu->numel() - 1 : k_.size(0);
    check_ints(chosen, "rows", k_, 2);
    if (chosen) TORCH_CHECK_VALUE(!cu && chosen->size(0) == sequences, "rows must be [batch, any] and go with [batch, seq_len, heads, head_dim] tensors");
    const CacheView c = check_cache(k_cache, v_cache, lengths, table, k_, sequences);
    TORCH_CHECK(!(at::GradMode::is_enabled() && (k_.requires_grad() || v_.requires_grad() || k_cache.requires_grad() || v_cache.requires_grad())),
                "cache_append has no gradient: call it under torch.no_grad() or on detached tensors");
    TORCH_CHECK(c10::InferenceMode::is_enabled() || !(k_cache.is_inference() || v_cache.is_inference()), "cache_append changes the cache in place, which inference tensors allow in inference mode only");
    check_place("cache_append", {k_, v_, k_cache, v_cache});
    py::gil_scoped_release nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    const Unseen unseen("cache_append");
    Tensor k = rows(k_), v = rows(v_);
    const Tensor pick = dense(chosen), ends = dense(cu);
    const c10::DeviceGuard guard(k.device());
    const Sizes z = sizes(k);
    if (z.B == 0 || z.N == 0 || (pick.defined() && pick.numel() == 0)) return;
    // rows that are a view of the cache (moved within it) are read before any is written
    if (meet(k, c.k) || meet(k, c.v)) k = k.clone(at::MemoryFormat::Contiguous);
    if (meet(v, c.k) || meet(v, c.v)) v = v.clone(at::MemoryFormat::Contiguous);
    int64_t s[12];
    put_strides(s, k);
    put_strides(s + 3, v);
    put_strides(s + 6, c.k);
    put_strides(s + 9, c.v);
    check(append_fn(k.const_data_ptr(), v.const_data_ptr(), c.k.data_ptr(), c.v.data_ptr(), ints(c.lengths), ints(c.table), ints(pick), pick.defined() ? (int)pick.size(1) : 0, ints(ends),
                    ends.defined() ? (int)ends.numel() - 1 : 0, z.B, z.N, z.H, z.D, c.page_size, c.pages, c.width, s, dtype_code(k), stream(k)));
    torch::autograd::impl::bump_version(c.k);
    torch::autograd::impl::bump_version(c.v);
}

// ---- causal attention --------------------------------------------------------------------------------------------------
struct Prompt {
    Tensor cu;                                 // may be undefined
    double scale;
    unsigned flags;
    int window, sinks;                         // window 0: none
};
Tensor workspace(const Tensor& q, size_t bytes) { return at::empty({(int64_t)bytes}, q.options().dtype(at::kByte).requires_grad(false)); }

// `low`: receives what rounding the output left, for a backward (16-bit types)
std::pair<Tensor, Tensor> run_causal_forward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Prompt& a, Tensor* low = nullptr) {
    const Unseen unseen("causal_attention");
    const Tensor q = rows(q_), k = rows(k_), v = rows(v_);
    const c10::DeviceGuard guard(q.device());
    const Sizes z = sizes(q);
    const auto fp32 = q.options().dtype(at::kFloat).requires_grad(false);
    Tensor out = like(q), lse = q.dim() == 4 ? at::empty({z.B, z.H, z.N}, fp32) : at::empty({z.H, z.N}, fp32);
    if (low && dtype_code(q) != SA2_F32) *low = like(q);
    if (out.numel() == 0) return {out, lse};
    int64_t s[12];
    put_strides(s, q);
    put_strides(s + 3, k);
    put_strides(s + 6, v);
    put_strides(s + 9, out);
    void* const left = low && low->defined() ? low->data_ptr() : nullptr;
    const int sequences = a.cu.defined() ? (int)a.cu.numel() - 1 : 0, hk = (int)k.size(-2);
    if (a.window)
        check(window_fwd_fn(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), out.data_ptr(), left, (float*)lse.data_ptr(), ints(a.cu), sequences, z.B, z.N, z.H, hk, z.D, s,
                            a.window, a.sinks, (float)a.scale, dtype_code(q), a.flags, stream(q)));
    else
        check(causal_fwd_fn(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), out.data_ptr(), left, (float*)lse.data_ptr(), ints(a.cu), sequences, z.B, z.N, z.H, hk, z.D, s,
                            (float)a.scale, dtype_code(q), a.flags, stream(q)));
    return {out, lse};
}

// `needs`: bit t set = gradient t of (q, k, v) is wanted; the others stay undefined
std::array<Tensor, 3> run_causal_backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& out_, const Tensor& low_, const Tensor& lse, const Tensor& dout_, unsigned needs,
                                           const Prompt& a) {
    const Unseen unseen("causal_attention");
    const Tensor q = rows(q_), k = rows(k_), v = rows(v_), dout = rows(dout_);
    const bool alike = !low_.defined() || low_.strides() == out_.strides();       // (the ABI has the strides of one for both)
    const Tensor out = alike ? rows(out_) : out_.contiguous(), low = !low_.defined() ? low_ : alike ? rows(low_) : low_.contiguous();
    const c10::DeviceGuard guard(q.device());
    const Sizes z = sizes(q);
    const int hk = (int)k.size(-2);
    std::array<Tensor, 3> g;
    const Tensor* const of[3] = {&q, &k, &v};
    for (int i = 0; i < 3; ++i)
        if (needs >> i & 1) g[i] = like(*of[i]);
    if (q.numel() == 0) {
        for (Tensor& t : g)
            if (t.defined()) t.zero_();        // (keys that no query head reads)
        return g;
    }
    const int sequences = a.cu.defined() ? (int)a.cu.numel() - 1 : 0;
    const size_t bytes = a.window ? window_ws_fn(sequences, z.B, z.N, z.H, hk, z.D, a.window, a.sinks, dtype_code(q), a.flags) : causal_ws_fn(z.B, z.N, z.H, hk, z.D, dtype_code(q), a.flags);
    const Tensor ws = workspace(q, std::max<size_t>(bytes, 256));
    int64_t s[24];
    const Tensor* const t[8] = {&q, &k, &v, &out, &dout, g[0].defined() ? &g[0] : &q, g[1].defined() ? &g[1] : &k, g[2].defined() ? &g[2] : &v};
    for (int i = 0; i < 8; ++i) put_strides(s + 3 * i, *t[i]);
    auto ptr = [&](int i) { return g[i].defined() ? g[i].data_ptr() : nullptr; };
    const void* const left = low.defined() ? low.const_data_ptr() : nullptr;
    if (a.window)
        check(window_bwd_fn(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), out.const_data_ptr(), left, dout.const_data_ptr(), (const float*)lse.const_data_ptr(), ptr(0), ptr(1), ptr(2),
                            ws.data_ptr(), (size_t)ws.numel(), ints(a.cu), sequences, z.B, z.N, z.H, hk, z.D, s, a.window, a.sinks, (float)a.scale, dtype_code(q), a.flags, stream(q)));
    else
        check(causal_bwd_fn(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), out.const_data_ptr(), left, dout.const_data_ptr(), (const float*)lse.const_data_ptr(), ptr(0), ptr(1), ptr(2),
                            ws.data_ptr(), (size_t)ws.numel(), ints(a.cu), sequences, z.B, z.N, z.H, hk, z.D, s, (float)a.scale, dtype_code(q), a.flags, stream(q)));
    return g;
}

struct CausalFormula : torch::autograd::Function<CausalFormula> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, Prompt a) {
        at::AutoDispatchBelowADInplaceOrView below;
        Tensor low;
        auto [out, lse] = run_causal_forward(q, k, v, a, &low);
        ctx->save_for_backward({q, k, v, out, lse, a.cu, low});
        ctx->saved_data["scale"] = a.scale;
        ctx->saved_data["flags"] = (int64_t)a.flags;
        ctx->saved_data["window"] = (int64_t)a.window;
        ctx->saved_data["sinks"] = (int64_t)a.sinks;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "causal_attention has first derivatives only: its backward cannot run with create_graph=True");
        at::AutoDispatchBelowADInplaceOrView below;
        const auto s = ctx->get_saved_variables();
        const Prompt a{s[5], ctx->saved_data["scale"].toDouble(), (unsigned)ctx->saved_data["flags"].toInt(), (int)ctx->saved_data["window"].toInt(), (int)ctx->saved_data["sinks"].toInt()};
        unsigned needs = 0;
        for (int i = 0; i < 3; ++i) needs |= (ctx->needs_input_grad(i) ? 1u : 0u) << i;
        auto g = run_causal_backward(s[0], s[1], s[2], s[3], s[6], s[4], grads[0], needs, a);
        return {g[0], g[1], g[2], Tensor()};
    }
};

// (window, first keys) as the C ABI takes them; (0, 0): none
std::pair<int, int> check_window(const std::optional<int64_t>& window, int64_t sinks) {
    TORCH_CHECK_VALUE(!window || *window >= 1, "window must be at least 1, got ", window ? *window : 0);
    TORCH_CHECK_VALUE(sinks >= 0, "sinks must not be negative, got ", sinks);
    TORCH_CHECK_VALUE(window || sinks == 0, "sinks go with a window");
    const int64_t most = 0x7fffffff;
    return {window ? (int)std::min(*window, most) : 0, (int)std::min(sinks, most)};
}

Prompt check_causal(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& cu, const std::optional<double>& scale, unsigned flags, const std::optional<int64_t>& window, int64_t sinks) {
    check_first(q, "q");
    check_beside(k, "k", q, "q");
    check_beside(v, "v", q, "q");
    TORCH_CHECK_VALUE(k.size(-2) == v.size(-2), "k and v differ in heads: ", k.sizes(), ", ", v.sizes());
    check_heads(q, k);
    TORCH_CHECK_VALUE(q.size(-1) >= 1 && q.size(-1) <= 256, "head_dim must be 1 to 256, got ", q.size(-1));
    check_cu(cu, q);
    TORCH_CHECK_VALUE(q.dim() == 4 || cu, "packed rows need cu_seqlens");
    const auto [reach, first] = check_window(window, sinks);
    check_place("causal_attention", {q, k, v});
    return {dense(cu), scale ? *scale : 1.0 / std::sqrt((double)q.size(-1)), flags, reach, first};
}

Tensor causal(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& cu, std::optional<double> scale, unsigned flags, std::optional<int64_t> window, int64_t sinks) {
    const Prompt a = check_causal(q, k, v, cu, scale, flags, window, sinks);
    py::gil_scoped_release nogil;
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) return CausalFormula::apply(q, k, v, a);
    at::AutoDispatchBelowADInplaceOrView below;
    return run_causal_forward(q, k, v, a).first;
}

std::tuple<Tensor, Tensor, Maybe> causal_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& cu, std::optional<double> scale, unsigned flags, bool keep_low,
                                                std::optional<int64_t> window, int64_t sinks) {
    const Prompt a = check_causal(q, k, v, cu, scale, flags, window, sinks);
    py::gil_scoped_release nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor low;
    auto [out, lse] = run_causal_forward(q, k, v, a, keep_low ? &low : nullptr);
    return {out, lse, low.defined() ? Maybe(low) : Maybe()};
}

std::tuple<Maybe, Maybe, Maybe> causal_backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse, const Tensor& dout, const Maybe& cu,
                                                std::optional<double> scale, unsigned needs, unsigned flags, const Maybe& low, std::optional<int64_t> window, int64_t sinks) {
    TORCH_CHECK_VALUE(!low || dtype_code(q) != SA2_F32, "out_low goes with 16-bit tensors");
    if (low) TORCH_CHECK_VALUE(low->sizes() == q.sizes() && low->scalar_type() == q.scalar_type() && low->device() == q.device(), "out_low must match q in shape, dtype and device");
    const Prompt a = check_causal(q, k, v, cu, scale, flags, window, sinks);
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(out, "out"), {dout, "dout"}})
        TORCH_CHECK_VALUE(t.sizes() == q.sizes() && t.scalar_type() == q.scalar_type() && t.device() == q.device(), name, " must match q in shape, dtype and device");
    const bool batched = q.dim() == 4;
    TORCH_CHECK_VALUE(lse.scalar_type() == at::kFloat && lse.device() == q.device() && lse.is_contiguous() && lse.dim() == q.dim() - 1 && lse.size(-1) == q.size(-3) && lse.size(-2) == q.size(-2) &&
                          (!batched || lse.size(0) == q.size(0)), "lse must be the contiguous float32 tensor that the forward returned, got ", lse.scalar_type(), " ", lse.sizes());
    check_place("causal_attention", {out, lse, dout});
    if (low) check_place("causal_attention", {*low});
    py::gil_scoped_release nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    auto g = run_causal_backward(q, k, v, out, low ? *low : Tensor(), lse, dout, needs, a);
    auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
    return {maybe(g[0]), maybe(g[1]), maybe(g[2])};
}

// ---- drafted trees -----------------------------------------------------------------------------------------------------
Tensor tree(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Maybe& parents, const Tensor& k_cache, const Tensor& v_cache, const Tensor& lengths, const Maybe& table,
            std::optional<double> scale, unsigned flags, std::optional<int64_t> window, int64_t sinks, const Maybe& weights) {
    TORCH_CHECK_VALUE(q_.dim() == 4, "q: expected [batch, nodes, heads, head_dim], got ", q_.sizes());
    check_first(q_, "q");
    check_beside(k_, "k", q_, "q");
    check_beside(v_, "v", q_, "q");
    TORCH_CHECK_VALUE(k_.size(-2) == v_.size(-2), "k and v differ in heads: ", k_.sizes(), ", ", v_.sizes());
    check_heads(q_, k_);
    TORCH_CHECK_VALUE(q_.size(-1) >= 1 && q_.size(-1) <= 256, "head_dim must be 1 to 256, got ", q_.size(-1));
    TORCH_CHECK_VALUE(q_.size(1) >= 1 && q_.size(1) <= SA2_TREE_NODES, "a drafted tree has 1 to ", SA2_TREE_NODES, " nodes, got ", q_.size(1));
    check_ints(parents, "parents", q_, 2);
    TORCH_CHECK_VALUE(!parents || (parents->size(0) == q_.size(0) && parents->size(1) == q_.size(1)), "parents must be [batch, nodes]");
    const CacheView c = check_cache(k_cache, v_cache, lengths, table, k_, q_.size(0));
    TORCH_CHECK(!(at::GradMode::is_enabled() && (q_.requires_grad() || k_.requires_grad() || v_.requires_grad() || k_cache.requires_grad() || v_cache.requires_grad())),
                "tree_attention has no gradient: call it under torch.no_grad() or on detached tensors");
    const auto [reach, first] = check_window(window, sinks);
    if (weights) {
        TORCH_CHECK_VALUE(q_.size(1) == 1, "weights are gathered from single tokens: a tree has ", q_.size(1), " nodes");
        check_weights(*weights, c, k_.size(2), true);
        check_place("tree_attention", {*weights});
    }
    check_place("tree_attention", {q_, k_, v_, k_cache, v_cache});
    py::gil_scoped_release nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    const Unseen unseen("tree_attention");
    const Tensor q = rows(q_), k = rows(k_), v = rows(v_), up = dense(parents);
    const c10::DeviceGuard guard(q.device());
    Tensor out = like(q);
    if (out.numel() == 0) return out;
    const Sizes z = sizes(q);
    const int hk = (int)k.size(2);
    const bool banded = reach > 0 || weights;
    const size_t bytes = banded ? window_tree_ws_fn(z.B, z.N, z.H, hk, z.D, c.page_size, c.width, reach, first, weights.has_value(), dtype_code(q), flags)
                                : tree_ws_fn(z.B, z.N, z.H, hk, z.D, c.page_size, c.width, dtype_code(q), flags);
    const Tensor ws = bytes ? workspace(q, bytes) : Tensor();
    int64_t s[20] = {};
    const Tensor* const t[6] = {&q, &k, &v, &c.k, &c.v, &out};
    for (int i = 0; i < 6; ++i) put_strides(s + 3 * i, *t[i]);
    void* const space = bytes ? ws.data_ptr() : nullptr;
    const float factor = (float)(scale ? *scale : 1.0 / std::sqrt((double)z.D));
    if (banded) {
        if (weights) {
            s[18] = weights->stride(0);
            s[19] = weights->stride(1);
        }
        check(window_tree_fn(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), c.k.const_data_ptr(), c.v.const_data_ptr(), out.data_ptr(), weights ? (float*)weights->data_ptr() : nullptr, ints(up),
                             ints(c.lengths), ints(c.table), space, bytes, z.B, z.N, z.H, hk, z.D, c.page_size, c.pages, c.width, s, reach, first, factor, dtype_code(q), flags, stream(q)));
        if (weights) torch::autograd::impl::bump_version(*weights);
    } else {
        check(tree_fn(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), c.k.const_data_ptr(), c.v.const_data_ptr(), out.data_ptr(), ints(up), ints(c.lengths), ints(c.table), space, bytes,
                      z.B, z.N, z.H, hk, z.D, c.page_size, c.pages, c.width, s, factor, dtype_code(q), flags, stream(q)));
    }
    return out;
}

// ---- gathered weights ---------------------------------------------------------------------------------------------------
Maybe key_weights(const Tensor& q_, const Tensor& k_, const Tensor& lse, const Maybe& cu, std::optional<double> scale, std::optional<int64_t> window, int64_t sinks, const Maybe& weights,
                  const Maybe& lengths, unsigned flags) {
    check_first(q_, "q");
    check_beside(k_, "k", q_, "q");
    check_heads(q_, k_);
    TORCH_CHECK_VALUE(q_.size(-1) >= 1 && q_.size(-1) <= 256, "head_dim must be 1 to 256, got ", q_.size(-1));
    check_cu(cu, q_);
    TORCH_CHECK_VALUE(q_.dim() == 4 || cu, "packed rows need cu_seqlens");
    const bool batched = q_.dim() == 4;
    TORCH_CHECK_VALUE(lse.scalar_type() == at::kFloat && lse.device() == q_.device() && lse.is_contiguous() && lse.dim() == q_.dim() - 1 && lse.size(-1) == q_.size(-3) && lse.size(-2) == q_.size(-2) &&
                          (!batched || lse.size(0) == q_.size(0)), "lse must be the contiguous float32 tensor that the forward returned, got ", lse.scalar_type(), " ", lse.sizes());
    const auto [reach, first] = check_window(window, sinks);
    const int64_t sequences = cu ? cu->numel() - 1 : q_.size(0), hk64 = k_.size(-2);
    TORCH_CHECK_VALUE(weights.has_value() == lengths.has_value(), "weights and lengths go together");
    if (weights) {
        check_ints(lengths, "lengths", q_, 1);
        TORCH_CHECK_VALUE(lengths->numel() == sequences, "lengths has ", lengths->numel(), " entries for ", sequences, " sequences");
        TORCH_CHECK_VALUE(weights->scalar_type() == at::kFloat && weights->dim() == 3 && weights->size(0) == sequences && weights->size(1) == hk64 && weights->size(2) >= 1 && weights->device() == q_.device(),
                          "weights must be float32 [", sequences, ", ", hk64, ", places] on the device of the other tensors, got ", weights->scalar_type(), " ", weights->sizes());
        check_added(*weights);
        check_place("key_weights", {*weights});
    }
    TORCH_CHECK(!(at::GradMode::is_enabled() && (q_.requires_grad() || k_.requires_grad() || lse.requires_grad())), "key_weights has no gradient: call it under torch.no_grad() or on detached tensors");
    check_place("key_weights", {q_, k_, lse});
    py::gil_scoped_release nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    const Unseen unseen("key_weights");
    const Tensor q = rows(q_), k = rows(k_), ends = dense(cu), held = dense(lengths);
    const c10::DeviceGuard guard(q.device());
    const Sizes z = sizes(q);
    const int hk = (int)hk64;
    const auto fp32 = q.options().dtype(at::kFloat).requires_grad(false);
    const Tensor out = weights ? *weights : batched ? at::empty({z.B, hk, z.N}, fp32) : at::empty({hk, z.N}, fp32);
    const Maybe result = weights ? Maybe() : Maybe(out);
    if (z.B == 0 || z.N == 0 || hk == 0 || z.H == 0) {
        if (!weights) out.zero_();                 // (keys that no query head reads)
        return result;
    }
    const size_t bytes = key_weights_ws_fn(ends.defined() ? (int)ends.numel() - 1 : 0, z.B, z.N, z.H, hk, z.D, reach, first, dtype_code(q), flags);
    const Tensor ws = bytes ? workspace(q, bytes) : Tensor();
    int64_t s[8];
    put_strides(s, q);
    put_strides(s + 3, k);
    s[6] = out.dim() == 3 ? out.stride(0) : 0;
    s[7] = out.stride(-2);
    check(key_weights_fn(q.const_data_ptr(), k.const_data_ptr(), (const float*)lse.const_data_ptr(), (float*)out.data_ptr(), ints(held), weights ? weights->size(2) : 0, bytes ? ws.data_ptr() : nullptr, bytes,
                         ints(ends), ends.defined() ? (int)ends.numel() - 1 : 0, z.B, z.N, z.H, hk, z.D, s, reach, first, (float)(scale ? *scale : 1.0 / std::sqrt((double)z.D)), dtype_code(q), flags,
                         stream(q)));
    if (weights) torch::autograd::impl::bump_version(*weights);
    return result;
}

std::pair<Tensor, Tensor> evict(const Tensor& k_cache, const Tensor& v_cache, const Tensor& weights, const Tensor& lengths, int64_t keep, int64_t first, int64_t recent, const Maybe& table) {
    TORCH_CHECK_VALUE(k_cache.dim() == 4 && k_cache.size(3) >= 1 && k_cache.size(3) <= 256 && k_cache.size(2) >= 1, "k_cache: expected [pages, page_size, heads, head_dim], head_dim 1 to 256, got ", k_cache.sizes());
    TORCH_CHECK_TYPE(dtype_code(k_cache) >= 0, "k_cache: unsupported dtype ", k_cache.scalar_type(), " (float32, bfloat16, float16)");
    TORCH_CHECK_VALUE(lengths.dim() == 1, "lengths must be an int32 tensor of 1 dimension, got ", lengths.sizes());
    const CacheView c = check_cache(k_cache, v_cache, lengths, table, k_cache, lengths.numel());
    TORCH_CHECK_VALUE((int64_t)c.page_size * c.width <= 0x7fffffff - 64, "a cache of 2^31 - 64 rows per sequence or more");
    TORCH_CHECK_VALUE(weights.dim() == 3, "weights must be float32 [batch, heads, places], got ", weights.sizes());
    check_weights(weights, c, weights.size(1) == 1 ? 1 : k_cache.size(2), false);
    TORCH_CHECK_VALUE(keep >= 1 && first >= 0 && recent >= 0 && keep < ((int64_t)1 << 31) && first <= keep && recent <= keep - first, "keep must be at least 1, first and recent at least 0 and together at most keep, got ", keep, ", ", first, ", ", recent);
    TORCH_CHECK(!(at::GradMode::is_enabled() && (k_cache.requires_grad() || v_cache.requires_grad() || weights.requires_grad())), "cache_evict has no gradient: call it under torch.no_grad() or on detached tensors");
    TORCH_CHECK(c10::InferenceMode::is_enabled() || !(k_cache.is_inference() || v_cache.is_inference()), "cache_evict changes the cache in place, which inference tensors allow in inference mode only");
    TORCH_CHECK_VALUE(k_cache.numel() == 0 || !(folded(k_cache) || folded(v_cache)), "rows of a cache share memory with one another: they move in place");
    TORCH_CHECK_VALUE(!share(k_cache, v_cache), "k_cache and v_cache have rows in the same memory, which would move twice");
    check_place("cache_evict", {k_cache, v_cache, weights});
    py::gil_scoped_release nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    const Unseen unseen("cache_evict");
    const c10::DeviceGuard guard(k_cache.device());
    const auto options = weights.options().requires_grad(false);
    const Tensor kept = at::empty({weights.size(0), weights.size(1), keep}, options.dtype(at::kInt)), left = at::empty(weights.sizes(), options.memory_format(at::MemoryFormat::Contiguous));
    if (weights.size(0) == 0) return {kept, left};
    int64_t s[8];
    put_strides(s, c.k);
    put_strides(s + 3, c.v);
    s[6] = weights.stride(0);
    s[7] = weights.stride(1);
    check(evict_fn(c.k.data_ptr(), c.v.data_ptr(), (const float*)weights.const_data_ptr(), (float*)left.data_ptr(), kept.data_ptr<int32_t>(), ints(c.lengths), ints(c.table), (int)weights.size(0),
                   (int)c.k.size(2), (int)weights.size(1), (int)c.k.size(3), c.page_size, c.pages, c.width, weights.size(2), (int)keep, (int)first, (int)recent, s, dtype_code(c.k), stream(c.k)));
    torch::autograd::impl::bump_version(c.k);
    torch::autograd::impl::bump_version(c.v);
    return {kept, left};
}

}  // namespace

void define_layers(py::module_& m) {
    m.def("bind_layers", [](uintptr_t rotary, uintptr_t append, uintptr_t causal_fwd, uintptr_t causal_ws, uintptr_t causal_bwd, uintptr_t tree_ws, uintptr_t tree, uintptr_t window_fwd, uintptr_t window_ws, uintptr_t window_bwd,
                             uintptr_t window_tree_ws, uintptr_t window_tree, uintptr_t key_weights_ws, uintptr_t key_weights, uintptr_t evict) {
        rotary_fn = (decltype(rotary_fn))rotary;
        append_fn = (decltype(append_fn))append;
        causal_fwd_fn = (decltype(causal_fwd_fn))causal_fwd;
        causal_ws_fn = (decltype(causal_ws_fn))causal_ws;
        causal_bwd_fn = (decltype(causal_bwd_fn))causal_bwd;
        tree_ws_fn = (decltype(tree_ws_fn))tree_ws;
        tree_fn = (decltype(tree_fn))tree;
        window_fwd_fn = (decltype(window_fwd_fn))window_fwd;
        window_ws_fn = (decltype(window_ws_fn))window_ws;
        window_bwd_fn = (decltype(window_bwd_fn))window_bwd;
        window_tree_ws_fn = (decltype(window_tree_ws_fn))window_tree_ws;
        window_tree_fn = (decltype(window_tree_fn))window_tree;
        key_weights_ws_fn = (decltype(key_weights_ws_fn))key_weights_ws;
        key_weights_fn = (decltype(key_weights_fn))key_weights;
        evict_fn = (decltype(evict_fn))evict;
    });
    m.def("rotary", &rotary);
    m.def("cache_append", &append);
    m.def("causal", &causal);
    m.def("causal_forward", &causal_forward);
    m.def("causal_backward", &causal_backward);
    m.def("tree", &tree);
    m.def("key_weights", &key_weights);
    m.def("cache_evict", &evict);
}

}  // namespace sa2_host
