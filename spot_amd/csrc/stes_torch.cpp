// The sequence operators (stes_gated_scan_*, stes_distill*) for torch: checks of the tensors, workspaces, streams and autograd nodes.
// spot_amd/recurrence.py and spot_amd/distill.py are its callers and hold the documentation.
//
// Why this side is compiled: the smallest calls take the GPU 4 us, and a call from Python through ctypes took the host 10; a backward pass
// runs on autograd's device thread, where Python code finds another core's caches: clips of 16 x 64 x 768 forward and backward took 52 us
// where the two threads shared a cache and 121 where they did not.
#include <algorithm>
#include <memory>
#include <mutex>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <unordered_map>
#include <vector>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/StreamGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/stes.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct Refused : std::runtime_error {                 // spot_amd.lib.StesError in Python
    int rc;
    Refused(const std::string& text, int rc_ = 0) : std::runtime_error(text), rc(rc_) {}
};

template <typename... Args>
[[noreturn]] void refuse(const Args&... args) { throw Refused(c10::str(args...)); }

void check(int rc, const char* entry) {
    if (rc) throw Refused(c10::str(entry, " failed (", rc, "): ", stes_last_error()), rc);
}

auto current(c10::Device dev) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()); }
void* stream_of(c10::Device dev) { return current(dev).stream(); }
// The device's default stream and torch's own streams last as long as the process.  A stream from outside, whose number is its handle, may be
// destroyed and its handle given out again (and one handle stands for a default stream of each thread): nothing is kept for it.
bool lasts(c10::Device dev) {
    const auto s = current(dev);
    return !s.stream() || s.id() != reinterpret_cast<c10::StreamId>(s.stream());
}
bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

// Makes `dev` the current device for a call on its tensors, and allocations skip the layers that record gradients.
struct Call {
    c10::DeviceGuard device;
    at::AutoDispatchBelowADInplaceOrView below;
    explicit Call(c10::Device dev) : device(dev) {}
};

Tensor fresh(at::IntArrayRef sizes, const Tensor& like, at::ScalarType type) { return at::empty(sizes, like.options().dtype(type)); }
Tensor fresh(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options()); }

// torch only notes some values down: a negative view's memory holds the opposite, a zero tensor has no memory.
bool noted(const Tensor& t) { return t.is_neg() || t._is_zerotensor(); }
Tensor plain(const Tensor& t) { return !t.defined() || !noted(t) ? t : t._is_zerotensor() ? t.clone() : t.resolve_neg(); }

template <typename T = void> T* at_(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

bool element(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
int f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }

// A caller's tensor that a kernel has changed in place, as torch's own in-place functions say it: a graph that saved it refuses
// its backward pass.
void written(const Tensor& t) {
    if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// A trace would record the allocation of a result and not the kernel that writes it.
void untraced(const char* op) {
    using c10::impl::TorchDispatchModeKey;
    typedef c10::impl::TorchDispatchModeTLS Modes;
    bool traced = at::tracer::impl::is_dispatch_enabled() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
    if (Modes::any_modes_set()) traced = traced || Modes::get_mode(TorchDispatchModeKey::PROXY) || Modes::get_mode(TorchDispatchModeKey::FAKE) || Modes::get_mode(TorchDispatchModeKey::FUNCTIONAL);
    if (traced) refuse(op, "cannot be traced (torch.jit.trace, make_fx): call it outside of what is recorded");
}
// (forward-mode tangents would be lost without a word)
template <typename... Tensors>
void no_tangents(const char* op, const Tensors&... t) {
    if ((... || (t.defined() && t._fw_grad(0).defined()))) refuse(op, "no forward-mode derivatives");
}
bool asks_for_gradients(const Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

// A tensor saved for the backward pass.  Hooks (torch.autograd.graph.saved_tensors_hooks) may give another one back: of the same sizes, type and
// device, or it is refused, but of any strides.
struct Saved {
    SavedVariable variable;
    std::vector<int64_t> sizes;
    at::ScalarType type = at::kFloat;
    c10::Device device = c10::kCPU;

    void operator=(const Tensor& t) {
        variable = SavedVariable(t, false);
        sizes = t.sizes().vec(), type = t.scalar_type(), device = t.device();
    }
    Tensor unpack() const {
        Tensor t = variable.unpack();
        if (t.defined() && (t.sizes() != at::IntArrayRef(sizes) || t.scalar_type() != type || t.device() != device))
            refuse("a saved ", type, " ", at::IntArrayRef(sizes), " on ", device, " came back as ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
        return plain(t);
    }
    Tensor whole() const { const Tensor t = unpack(); return t.defined() ? t.contiguous() : t; }
    void reset() { variable.reset_data(); }
};

// ---------------------------------------------------------------- leaves
// The node that accumulates a leaf's gradient keeps the stream on which it was made for as long as some autograd graph holds it, whoever made
// that graph; a captured backward pass makes that stream wait for the capture's, which ends the process where an eager graph made the
// node (the default stream cannot be part of a capture).  A captured call refuses such leaves, and notes those that it finds in order: a later
// capture on another stream may meet them while this one's outputs live.
struct Leaves {
    std::mutex lock;
    std::unordered_map<Node*, std::weak_ptr<Node>> captured;
    size_t sweep = 64;
};
Leaves& leaves() {
    static Leaves* all = new Leaves;                  // (never destroyed: autograd's threads outlive main)
    return *all;
}

// The inputs' edges into the graph, held while they are looked at: leaves' nodes live as long as something holds them.
torch::autograd::edge_list guarded(torch::autograd::edge_list edges, c10::Device dev) {
    if (!capturing()) return edges;
    const c10::Stream here = current(dev).unwrap();
    Leaves& l = leaves();
    std::lock_guard<std::mutex> g(l.lock);
    for (const auto& e : edges) {
        std::shared_ptr<Node> n = e.function;
        for (int i = 0; i < 4 && n && n->num_outputs() == 1; ++i) n = n->next_edge(0).function;      // (through the views and copies that a call makes of a leaf)
        if (!n || n->num_outputs() != 0) continue;
        const std::optional<c10::Stream> made = n->stream();
        bool inside = !made || *made == here;
        if (!inside && made->id() != 0) {
            const c10::StreamGuard there(*made);
            inside = capturing();                     // (another stream of a capture)
        }
        const auto seen = l.captured.find(n.get());
        if (!inside && (seen == l.captured.end() || seen->second.lock() != n))
            refuse("an autograd graph from outside this capture still holds one of its leaves: drop its outputs first");
        l.captured[n.get()] = n;
    }
    if (l.captured.size() > l.sweep) {
        for (auto i = l.captured.begin(); i != l.captured.end();) i = i->second.expired() ? l.captured.erase(i) : std::next(i);
        l.sweep = 64 + 2 * l.captured.size();
    }
    return edges;
}

// Gradients that cannot be differentiated again: they depend on what `node` depends on and on the gradients that came in, through a node
// that says so where somebody tries.
variable_list once(variable_list&& grads, const Node& node, const variable_list& came, const char* what) {
    if (!at::GradMode::is_enabled()) return std::move(grads);
    for (Tensor& g : grads)
        if (g.defined()) {
            torch::autograd::edge_list edges = torch::autograd::collect_next_edges(came);
            edges.insert(edges.end(), node.next_edges().begin(), node.next_edges().end());
            std::shared_ptr<Node> end(new torch::autograd::Error(c10::str(what, " is differentiable once"), std::move(edges)), torch::autograd::deleteNode);
            torch::autograd::set_history(g, end);
        }
    return std::move(grads);
}

// ---------------------------------------------------------------- kept workspaces
// The two workspaces that the scan's calls on one stream take in turn: a call finds its own zero and leaves the one of the call before zero,
// so none needs a launch that clears.  A call's launch happens under the lock: what is clean follows the stream's order.
struct Kept {
    std::mutex lock;
    Tensor pair[2];
    int turn = 0;
    int64_t dirty[2] = {0, 0};
    Tensor zeros;                           // of the distillation's calls, which leave it zero
};
constexpr int64_t KEPT_BYTES = 16 << 20;    // larger workspaces are not kept: clearing them is a small part of such calls (2 % of the data)
struct Streams {
    std::mutex lock;
    std::vector<std::pair<std::pair<int, void*>, std::shared_ptr<Kept>>> all;
    size_t most = 64;                       // the oldest one's memory then goes back, in its stream's order
};
Streams& streams() {
    static Streams* s = new Streams;        // (never destroyed: the allocator may be gone by then)
    return *s;
}

// The lock of a stream's workspaces.  Its holder allocates, and an allocation that Python watches (torch's memory history, dispatch modes) needs the
// interpreter: a Python thread that waits for the lock lets go of it.
std::unique_lock<std::mutex> hold(std::mutex& lock) {
    std::unique_lock<std::mutex> held(lock, std::try_to_lock);
    if (!held.owns_lock()) {
        std::optional<pybind11::gil_scoped_release> others;
        if (PyGILState_Check()) others.emplace();
        held.lock();
    }
    return held;
}

std::shared_ptr<Kept> kept(int device, void* stream) {
    Streams& s = streams();
    std::shared_ptr<Kept> oldest;           // (freed after the lock)
    std::lock_guard<std::mutex> g(s.lock);
    for (const auto& k : s.all)
        if (k.first == std::make_pair(device, stream)) return k.second;
    if (s.all.size() >= s.most) {
        oldest = s.all.front().second;
        s.all.erase(s.all.begin());
    }
    s.all.emplace_back(std::make_pair(device, stream), std::make_shared<Kept>());
    return s.all.back().second;
}

// One call of the library with the workspace that it needs.  A captured call gets one of its own, cleared in the graph: a graph may
// be replayed on any stream, next to others.
void scan_call(int (*entry)(const stes_gated_scan_args*, void*), const char* name, stes_gated_scan_args& a, c10::Device dev) {
    void* s = stream_of(dev);
    const int64_t n = a.T <= STES_SCAN_BLOCK ? 0 : stes_gated_scan_ws_bytes(a.B, a.T, a.H);
    if (!n) return check(entry(&a, s), name);
    const auto bytes = at::TensorOptions().device(dev).dtype(at::kByte);
    a.ws_bytes = n;
    if (n > KEPT_BYTES || capturing() || !lasts(dev)) {
        const Tensor ws = at::empty({n}, bytes);
        a.ws = ws.data_ptr();
        return check(entry(&a, s), name);
    }
    const auto k = kept(dev.index(), s);
    const auto held = hold(k->lock);
    if (!k->pair[0].defined() || k->pair[0].numel() < n) {
        k->pair[0] = Tensor();
        Tensor one = at::zeros({n}, bytes), two = at::zeros({n}, bytes);
        k->pair[0] = one, k->pair[1] = two;
        k->turn = 0, k->dirty[0] = k->dirty[1] = 0;
    }
    const int i = k->turn, j = 1 - i;
    a.ws = k->pair[i].data_ptr();
    a.ws_zero = 1;
    if (k->dirty[j]) a.scrub = k->pair[j].data_ptr(), a.scrub_bytes = k->dirty[j];
    const int rc = entry(&a, s);
    if (rc) k->pair[0] = Tensor();
    check(rc, name);
    k->dirty[i] = n, k->dirty[j] = 0, k->turn = j;
}

// ---------------------------------------------------------------- gated scan
constexpr const char* SCAN = "gated_scan: ";

// (frame stride, sequence stride) of a [B, T, width] tensor; the frame stride of a single frame is immaterial.
std::pair<int64_t, int64_t> strides(const Tensor& t, int64_t width) { return {t.size(1) > 1 ? t.stride(1) : width, t.stride(0)}; }

// Whether the frames of a [B, T, width] tensor are contiguous and do not overlap.
bool frames(const Tensor& t) { return t.is_contiguous() || ((t.size(2) <= 1 || t.stride(2) == 1) && (t.size(1) <= 1 || t.stride(1) >= t.size(2))); }

// Stride between the rows of a float32 [B, H] tensor whose rows are contiguous and apart.
int64_t row_stride(const Tensor& t, int64_t B, int64_t H, const char* name) {
    if (t.scalar_type() != at::kFloat || t.dim() != 2 || t.size(0) != B || t.size(1) != H)
        refuse(SCAN, name, " must be float32 [", B, ", ", H, "], got ", t.scalar_type(), " ", t.sizes());
    if ((H > 1 && t.stride(1) != 1) || (B > 1 && t.stride(0) < H)) refuse(SCAN, "rows of ", name, " must be contiguous and not overlap");
    return B > 1 ? t.stride(0) : std::max<int64_t>(H, 1);
}

struct Scanned { Tensor h, last, states; };

Scanned scan_forward(const Tensor& pre, const Tensor& h0, const Tensor& lengths, bool reverse, const Tensor& out, const Tensor& state_out, bool keep_states) {
    const int64_t B = pre.size(0), T = pre.size(1), W = pre.size(2), H = W / 2;
    Scanned r;
    r.h = out.defined() ? out : fresh({B, T, H}, pre);
    r.last = state_out.defined() ? state_out : fresh({B, H}, pre, at::kFloat);
    if (keep_states) r.states = fresh({B, (T + STES_SCAN_BLOCK - 1) / STES_SCAN_BLOCK, H}, pre, at::kFloat);
    if (!B || !H) return r;
    stes_gated_scan_args a{};
    a.pre = pre.data_ptr();
    std::tie(a.ld_pre, a.bs_pre) = strides(pre, W);
    a.h0 = at_<float>(h0);
    a.bs_h0 = !h0.defined() || h0.dim() == 1 ? 0 : row_stride(h0, B, H, "h0");
    a.lengths = at_<int32_t>(lengths);
    a.h = r.h.data_ptr();
    std::tie(a.ld_h, a.bs_h) = strides(r.h, H);
    a.h_last = at_<float>(r.last);
    a.bs_hl = row_stride(r.last, B, H, "state_out");
    a.states = at_<float>(r.states);
    a.B = B, a.T = T, a.H = H, a.f32 = f32(pre), a.reverse = reverse;
    scan_call(stes_gated_scan_fwd, "stes_gated_scan_fwd", a, pre.device());
    return r;
}

struct GatedScanBackward : public Node {
    Saved pre, lengths, states;
    bool reverse = false;
    int h0_dim = 0;                         // of an initial state that asks for a gradient

    std::string name() const override { return "GatedScanBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> g(mutex_);
        pre.reset();
        lengths.reset();
        states.reset();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> g(mutex_);
        Tensor p = pre.unpack(), dpre, dh0, total;
        untraced(SCAN);
        no_tangents(SCAN, grads[0], grads[1]);
        if (grads[0].defined() || grads[1].defined()) {
            const Call call(p.device());
            const Tensor n = lengths.whole(), st = states.whole();
            if (!frames(p)) p = p.contiguous();
            const int64_t B = p.size(0), T = p.size(1), W = p.size(2), H = W / 2;
            dpre = fresh({B, T, W}, p);
            if (h0_dim) dh0 = fresh({B, H}, p, at::kFloat);
            if (h0_dim == 1) total = fresh({H}, p, at::kFloat);
            if (H && (B || total.defined())) {
                Tensor dh = plain(grads[0]), dlast = plain(grads[1]);
                stes_gated_scan_args a{};
                if (dh.defined()) {
                    // (a gradient that was expanded or transposed)
                    if (!frames(dh)) dh = dh.contiguous();
                    std::tie(a.ld_dh, a.bs_dh) = strides(dh, H);
                }
                if (dlast.defined()) dlast = dlast.contiguous();
                a.pre = p.data_ptr();
                std::tie(a.ld_pre, a.bs_pre) = strides(p, W);
                a.lengths = at_<int32_t>(n);
                a.states = at_<float>(st);
                a.dh = at_(dh);
                a.dh_last = at_<float>(dlast);
                a.bs_dhl = H;
                a.dpre = dpre.data_ptr();
                a.ld_dpre = W, a.bs_dpre = T * W;
                a.dh0 = at_<float>(dh0);
                a.dh0_sum = at_<float>(total);
                a.B = B, a.T = T, a.H = H, a.f32 = f32(p), a.reverse = reverse;
                scan_call(stes_gated_scan_bwd, "stes_gated_scan_bwd", a, p.device());
            }
        }
        return once({dpre, h0_dim == 1 ? total : dh0}, *this, grads, "gated_scan");
    }
};

// Whether the rows of a [B, T, width] tensor with a contiguous last dimension are apart: frames within sequences or the reverse.
bool apart(const Tensor& t, int64_t width) {
    std::pair<int64_t, int64_t> in{0, 1}, out{0, 1};
    if (t.size(0) > 1) in = {t.stride(0), t.size(0)};
    if (t.size(1) > 1) out = {t.stride(1), t.size(1)};
    if (out < in) std::swap(in, out);
    if (in.second > 1 && in.first < width) return false;
    return out.second == 1 || out.first >= in.first * (in.second - 1) + width;
}

std::tuple<Tensor, Tensor> gated_scan(const Tensor& pre_, const Maybe& h0_, const Maybe& lengths_, bool reverse, const Maybe& out_, const Maybe& state_out_) {
    untraced(SCAN);
    const Tensor pre = plain(pre_), lengths = plain(lengths_.value_or(Tensor())), out = out_.value_or(Tensor()), state_out = state_out_.value_or(Tensor());
    Tensor h0 = plain(h0_.value_or(Tensor()));
    if (!pre.is_cuda() || pre.dim() != 3 || !element(pre)) refuse(SCAN, "pre must be a bfloat16 or float32 tensor [B, T, 2H] on the GPU");
    const int64_t B = pre.size(0), T = pre.size(1), W = pre.size(2), H = W / 2;
    const c10::Device dev = pre.device();
    if (W % 2) refuse(SCAN, "the last dimension of pre holds gates and candidates and is even, got ", W);
    if (std::max({B, T, W}) > INT32_MAX) refuse(SCAN, "sizes beyond 32 bits: ", pre.sizes());
    if (!frames(pre)) refuse(SCAN, "frames of pre must be contiguous and not overlap");
    if (h0.defined()) {
        const bool rows = h0.dim() == 2 && h0.size(0) == B && h0.size(1) == H;
        if (h0.device() != dev || h0.scalar_type() != at::kFloat || !(rows || (h0.dim() == 1 && h0.size(0) == H)))
            refuse(SCAN, "h0 must be float32 [", B, ", ", H, "] or [", H, "] on ", dev, ", got ", h0.scalar_type(), " ", h0.sizes(), " on ", h0.device());
        if (!h0.is_contiguous() && ((H > 1 && h0.stride(-1) != 1) || (rows && B > 1 && h0.stride(0) < H))) {
            if (state_out.defined() && state_out.data_ptr() == h0.data_ptr()) refuse(SCAN, "a state in place needs contiguous rows that do not overlap");
            h0 = h0.contiguous();
        }
    }
    if (lengths.defined() && (lengths.device() != dev || lengths.scalar_type() != at::kInt || lengths.dim() != 1 || lengths.size(0) != B || !lengths.is_contiguous()))
        refuse(SCAN, "lengths must be contiguous int32 [", B, "] on ", dev, ", got ", lengths.scalar_type(), " ", lengths.sizes(), " on ", lengths.device());
    no_tangents(SCAN, pre, h0, out, state_out);
    const bool grad = asks_for_gradients(pre) || (h0.defined() && asks_for_gradients(h0));
    if (grad && (out.defined() || state_out.defined())) refuse(SCAN, "out and state_out are for calls without gradients");
    if (out.defined()) {
        if (out.device() != dev || out.scalar_type() != pre.scalar_type() || out.dim() != 3 || out.size(0) != B || out.size(1) != T || out.size(2) != H || asks_for_gradients(out) || noted(out))
            refuse(SCAN, "out must be ", pre.scalar_type(), " [", B, ", ", T, ", ", H, "] on ", dev, ", without gradients, with memory of its values");
        if ((H > 1 && out.stride(2) != 1) || !apart(out, H)) refuse(SCAN, "frames of out must be contiguous and not overlap");
    }
    if (state_out.defined()) {
        if (state_out.device() != dev || asks_for_gradients(state_out) || noted(state_out)) refuse(SCAN, "state_out must be on ", dev, ", without gradients, with memory of its values");
        const int64_t stride = row_stride(state_out, B, H, "state_out");
        if (h0.defined() && state_out.data_ptr() == h0.data_ptr() && B > 1 && (h0.dim() == 1 || h0.stride(0) != stride))
            refuse(SCAN, "a state in place is h0 itself, one row per sequence");
    }
    if (!grad) {
        Scanned r;
        {
            const Call call(dev);
            r = scan_forward(pre, h0, lengths, reverse, out, state_out, false);
        }
        written(out);
        written(state_out);
        return {r.h, r.last};
    }
    Scanned r;
    std::shared_ptr<GatedScanBackward> node(new GatedScanBackward, torch::autograd::deleteNode);
    {
        const Call call(dev);
        node->set_next_edges(guarded(torch::autograd::collect_next_edges(pre, h0), dev));
        r = scan_forward(pre, h0, lengths, reverse, out, state_out, true);
    }
    node->pre = pre;
    if (lengths.defined()) node->lengths = lengths;
    node->states = r.states;
    node->reverse = reverse;
    node->h0_dim = h0.defined() && h0.requires_grad() ? h0.dim() : 0;
    torch::autograd::set_history(r.h, node);
    torch::autograd::set_history(r.last, node);
    return {r.h, r.last};
}

// ---------------------------------------------------------------- distillation
constexpr const char* KL = "topk_distill: ";

// [..., n] -> [M, n] without a copy where the strides allow one row stride, else a contiguous copy.
Tensor flat(Tensor t, int64_t n) {
    if (t.dim() != 2) t = t.reshape({-1, n});
    if (!t.is_contiguous() && ((n > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < n))) t = t.contiguous();
    return t;
}
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct Rows {
    Tensor logits, idx, val, weight;        // [M, ...] with contiguous rows
    double temperature, denom;
};

stes_distill_args distill_args(const Rows& r) {
    stes_distill_args a{};
    a.logits = r.logits.data_ptr(), a.ld = ld(r.logits), a.f32 = f32(r.logits);
    a.idx = r.idx.data_ptr(), a.ld_idx = ld(r.idx), a.idx_i64 = r.idx.scalar_type() == at::kLong;
    a.val = r.val.data_ptr(), a.ld_val = ld(r.val), a.val_f32 = f32(r.val);
    a.weight = at_<float>(r.weight);
    a.M = r.logits.size(0), a.V = r.logits.size(1), a.k = r.idx.size(1);
    a.temperature = r.temperature, a.denom = r.denom, a.grad_scale = 1.f;
    return a;
}

void into(stes_distill_args& a, const Tensor& d) { a.dlogits = d.data_ptr(), a.ld_d = ld(d), a.d_f32 = f32(d); }

// loss, and whatever else `a` asks for
Tensor distill_call(stes_distill_args& a, const Tensor& logits) {
    const Tensor loss = fresh({}, logits, at::kFloat);
    void* s = stream_of(logits.device());
    a.loss = static_cast<float*>(loss.data_ptr());
    std::shared_ptr<Kept> k;
    if (a.M > 1 && !capturing() && lasts(logits.device())) {          // (a graph may be replayed on any stream, next to others)
        k = kept(logits.device().index(), s);
        const auto held = hold(k->lock);
        if (!k->zeros.defined()) k->zeros = at::zeros({STES_DISTILL_WORDS}, logits.options().dtype(at::kLong));
        a.zeros = static_cast<uint64_t*>(k->zeros.data_ptr());
    }
    const int64_t n = stes_distill_ws_floats(a.M, a.V, a.k, a.zeros != nullptr);
    Tensor ws;                              // (of this call's own)
    if (n) ws = fresh({n}, logits, at::kFloat);
    a.ws = at_<float>(ws), a.ws_floats = n;
    check(stes_distill(&a, s), "stes_distill");
    return loss;
}

Rows distill_check(const Tensor& logits_, const Tensor& idx_, const Tensor& val_, double temperature, const Maybe& weight_, std::optional<double> denom) {
    untraced(KL);
    const Tensor logits = plain(logits_), idx = plain(idx_), val = plain(val_), weight = plain(weight_.value_or(Tensor()));
    if (!logits.is_cuda() || !element(logits) || logits.dim() < 1) refuse(KL, "logits must be a bfloat16 or float32 tensor [..., classes] on the GPU");
    const c10::Device dev = logits.device();
    const int64_t V = logits.size(-1);
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    if (V < 1) refuse(KL, "no classes");
    if (idx.device() != dev || (idx.scalar_type() != at::kLong && idx.scalar_type() != at::kInt) || idx.dim() != logits.dim() || idx.sizes().slice(0, idx.dim() - 1) != lead)
        refuse(KL, "idx must be int64 or int32 ", lead, " + [k] on ", dev, ", got ", idx.scalar_type(), " ", idx.sizes(), " on ", idx.device());
    const int64_t k = idx.size(-1);
    if (k < 1 || k > STES_DISTILL_MAX_K) refuse(KL, "1 to ", STES_DISTILL_MAX_K, " teacher classes a row, got ", k);
    if (val.device() != dev || !element(val) || val.sizes() != idx.sizes()) refuse(KL, "val must be float32 or bfloat16 ", idx.sizes(), " on ", dev);
    if (weight.defined() && (weight.device() != dev || weight.scalar_type() != at::kFloat || weight.sizes() != lead)) refuse(KL, "weight must be float32 ", lead, " on ", dev);
    if (asks_for_gradients(val) || (weight.defined() && asks_for_gradients(weight))) refuse(KL, "the teacher's logits and the weights are constants: detach them");
    no_tangents(KL, logits, val, weight);
    if (!(temperature >= 1e-6 && temperature <= 1e6)) refuse(KL, "the temperature lies between 1e-6 and 1e6, got ", temperature);
    Rows r{flat(logits, V), flat(idx, k), flat(val, k), Tensor(), temperature, 0.0};
    if (std::max(r.logits.size(0), V) > INT32_MAX) refuse(KL, "sizes beyond 32 bits: ", logits.sizes());
    r.denom = denom ? *denom : std::max<double>(1.0, r.logits.size(0));
    if (!(r.denom > 0.0 && r.denom < INFINITY)) refuse(KL, "the denominator is positive, got ", r.denom);
    if (weight.defined()) r.weight = weight.reshape({-1}).contiguous();
    return r;
}

struct DistillBackward : public Node {
    Saved logits, idx, val, weight, stats;
    double temperature = 1.0, denom = 1.0;

    std::string name() const override { return "DistillBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> g(mutex_);
        for (Saved* v : {&logits, &idx, &val, &weight, &stats}) v->reset();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> g(mutex_);
        Rows r{logits.unpack(), Tensor(), Tensor(), Tensor(), temperature, denom};
        Tensor d;
        untraced(KL);
        no_tangents(KL, grads[0]);
        if (grads[0].defined()) {
            const Call call(r.logits.device());
            const Tensor i = idx.unpack(), v = val.unpack(), st = stats.whole();
            r.logits = flat(r.logits, r.logits.size(1)), r.idx = flat(i, i.size(1)), r.val = flat(v, v.size(1)), r.weight = weight.whole();
            d = fresh(r.logits.sizes(), r.logits);
            if (r.logits.size(0)) {
                stes_distill_args a = distill_args(r);
                const Tensor up = plain(grads[0]);
                a.upstream = at_<float>(up);
                a.stats = at_<float>(st);
                into(a, d);
                check(stes_distill_bwd(&a, stream_of(r.logits.device())), "stes_distill_bwd");
            }
        }
        return once({d}, *this, grads, "topk_distill_loss");
    }
};

Tensor topk_distill_loss(const Tensor& logits, const Tensor& idx, const Tensor& val, double temperature, const Maybe& weight, std::optional<double> denom) {
    const Rows r = distill_check(logits, idx, val, temperature, weight, denom);
    stes_distill_args a = distill_args(r);
    if (!asks_for_gradients(r.logits)) {
        const Call call(r.logits.device());
        return distill_call(a, r.logits);
    }
    std::shared_ptr<DistillBackward> node(new DistillBackward, torch::autograd::deleteNode);
    Tensor loss, stats;
    {
        const Call call(r.logits.device());
        node->set_next_edges(guarded(torch::autograd::collect_next_edges(r.logits), r.logits.device()));
        stats = fresh({r.logits.size(0), 2}, r.logits, at::kFloat);
        a.stats = at_<float>(stats);
        loss = distill_call(a, r.logits);
    }
    node->logits = r.logits;
    node->idx = r.idx;
    node->val = r.val;
    if (r.weight.defined()) node->weight = r.weight;
    node->stats = stats;
    node->temperature = r.temperature, node->denom = r.denom;
    torch::autograd::set_history(loss, node);
    return loss;
}

std::tuple<Tensor, Tensor> topk_distill_grad(const Tensor& logits, const Tensor& idx, const Tensor& val, double temperature, const Maybe& weight,
                                             std::optional<double> denom, double grad_scale, const Maybe& out_, bool accumulate) {
    const Rows r = distill_check(logits, idx, val, temperature, weight, denom);
    Tensor out = out_.value_or(Tensor()), d;
    no_tangents(KL, out);
    const Call call(r.logits.device());
    if (!out.defined()) {
        if (accumulate) refuse(KL, "accumulate adds to out");
        out = fresh(logits.sizes(), logits);
    } else if (out.device() != logits.device() || !element(out) || out.sizes() != logits.sizes() || asks_for_gradients(out) || noted(out))
        refuse(KL, "out must be float32 or bfloat16 ", logits.sizes(), " on ", logits.device(), ", without gradients, with memory of its values");
    const int64_t V = out.size(-1);
    d = out.dim() == 2 ? out : out.reshape({-1, V});
    if (d.data_ptr() != out.data_ptr()) refuse(KL, "rows of out must be one stride apart");
    if (!d.is_contiguous() && ((V > 1 && d.stride(1) != 1) || (d.size(0) > 1 && d.stride(0) < V))) refuse(KL, "rows of out must be contiguous and not overlap");
    stes_distill_args a = distill_args(r);
    a.grad_scale = grad_scale;
    a.accumulate = accumulate;
    into(a, d);
    const Tensor loss = distill_call(a, r.logits);
    if (out_) written(out);
    return {loss, out};
}

PyObject* stes_error = nullptr;             // spot_amd.lib.StesError

}  // namespace

PYBIND11_MODULE(_stes_torch, m) {
    namespace py = pybind11;
    py::register_local_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refused& e) {
            py::object error = py::reinterpret_borrow<py::object>(stes_error ? stes_error : PyExc_RuntimeError)(e.what());
            if (e.rc) error.attr("rc") = e.rc;
            PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(error.ptr())), error.ptr());
        }
    });
    m.def("set_error", [](py::object type) { stes_error = type.release().ptr(); });
    m.def("keep_streams", [](size_t most) { std::lock_guard<std::mutex> g(streams().lock); std::swap(streams().most, most); return most; }, "How many streams' workspaces are kept; returns what it was");
    m.def("kept_streams", []() { std::lock_guard<std::mutex> g(streams().lock); return streams().all.size(); });
    m.def("gated_scan", &gated_scan);
    m.def("topk_distill_loss", &topk_distill_loss);
    m.def("topk_distill_grad", &topk_distill_grad);
}
