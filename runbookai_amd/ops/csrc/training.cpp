// Bindings of the training kernels: packed attention with gradients,
// cross-entropy, gradient norm and clipping.  Arguments are checked here, every
// launch runs on the tensors' own device and its current stream, and scratch
// memory comes from torch's allocator for each call, so that two streams or two
// captured graphs never share any.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "grad_norm.h"
#include "packed_attn.h"

extern "C" {
int launch_packed_tiles(const PackedArgs*, void*);
int launch_packed_attn_fwd(const PackedArgs*, void*);
int launch_packed_attn_dq(const PackedArgs*, void*);
int launch_packed_attn_dkv(const PackedArgs*, void*);
int launch_xent_fwd(int, const void*, long, const void*, long, int, int, void*, void*, void*,
                    void*, void*);
int xent_parts(int, int);
int launch_xent_reduce(const void*, const void*, int, int, void*, void*, void*);
int launch_xent_bwd(int, const void*, long, const void*, long, int, int, const void*,
                    const void*, long, const void*, void*, long, void*);
int launch_grad_sums(const GradTable*, int, void*, void*);
int launch_grad_norm(const void*, int, void*, void*);
int launch_grad_clip(const GradTable*, int, const void*, int, double, double, void*, void*);
}

namespace {

using torch::Tensor;

void* stream_of(const Tensor& t) {
    return (void*)at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

void launched(int code, const char* what) {
    TORCH_CHECK(code == 0, what, ": the launch failed with HIP error ", code);
}

// The kernels take a tensor's memory.  What it has beside that (a tangent, its
// place in a trace that is recorded) would be lost without a word, and one that
// only stands for memory (a fake one, a wrapper, freed storage) would lead them to
// address 0.
void plain(const Tensor& t, const char* name) {
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(),
                                "the training ops cannot be recorded by torch.jit.trace");
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), name,
                                " has a forward-mode derivative, which the training ops do not "
                                "have on the GPU");
    TORCH_CHECK_VALUE(t.layout() == torch::kStrided &&
                          !t.key_set().has(c10::DispatchKey::Python) && t.has_storage() &&
                          (t.numel() == 0 || t.const_data_ptr()),
                      name, " must be a plain tensor with memory of its own");
}

// Memory for a kernel to write.  Where a dispatch mode is on it may be none, though
// all inputs are real.
Tensor blank(at::IntArrayRef sizes, const torch::TensorOptions& options) {
    const Tensor t = torch::empty(sizes, options);
    plain(t, "a result");
    return t;
}

// What a backward pass returns: without a gradient of its own, and with an
// error where somebody asks for one (create_graph).
std::vector<Tensor> once(std::vector<Tensor> grads, const char* what) {
    if (!torch::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    const auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string(what) + " has no second derivative", (int)grads.size());
    return (*error)(std::move(grads));
}

// Scratch memory of several parts in one allocation: each part's offset, and
// the size of all.
struct Parts {
    size_t size = 0;
    size_t add(size_t bytes) {
        const size_t at = size;
        size += (bytes + 255) / 256 * 256;
        return at;
    }
    Tensor make(const Tensor& like) const {
        return blank({(long)size}, like.options().dtype(torch::kUInt8));
    }
};

template <typename T>
T* part(const Tensor& t, size_t at) {
    return reinterpret_cast<T*>(static_cast<char*>(t.data_ptr()) + at);
}

// ------------------------------------------------------------ packed attention

// What the kernels take: head rows that are dense, at 16-byte boundaries, and
// close enough for 32-bit offsets within a tile.
bool fits(const Tensor& t) {
    return t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
           t.stride(0) < (1L << 23) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

Tensor rows16(const Tensor& t) {
    return fits(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

void check_rows(const Tensor& t, const char* name, const Tensor& like) {
    plain(t, name);
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on ", like.device());
    TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bfloat16");
    TORCH_CHECK(t.dim() == 3, name, " must have 3 dimensions: tokens, heads, head dim");
    TORCH_CHECK(fits(t), name, " has too many or too wide heads");
}

unsigned short* bf16(const Tensor& t) { return (unsigned short*)t.data_ptr(); }

// The arguments that both passes have
PackedArgs packed_args(const Tensor& q, const Tensor& k, const Tensor& v, double scale) {
    check_rows(q, "q", q);
    check_rows(k, "k", q);
    check_rows(v, "v", q);
    const long T = q.size(0), Hq = q.size(1), D = q.size(2), Hk = k.size(1);
    TORCH_CHECK(D == 64 || D == 128, "head dim must be 64 or 128, not ", D);
    TORCH_CHECK(k.size(0) == T && v.size(0) == T && k.size(2) == D && v.size(2) == D &&
                    v.size(1) == Hk,
                "q, k and v must have the same tokens and head dim, k and v the same heads");
    TORCH_CHECK(Hk > 0 && Hq > 0 && Hq % Hk == 0,
                "query heads must be a multiple of key/value heads");
    TORCH_CHECK(T < (1L << 30), "at most 2^30 tokens");
    PackedArgs a = {};
    a.q = bf16(q); a.qt = q.stride(0); a.qh = q.stride(1);
    a.k = bf16(k); a.kt = k.stride(0); a.kh = k.stride(1);
    a.v = bf16(v); a.vt = v.stride(0); a.vh = v.stride(1);
    a.T = (int)T; a.Hq = (int)Hq; a.Hk = (int)Hk; a.D = (int)D;
    a.scale = (float)scale;
    return a;
}

// How many tiles there may be, and whether the forward kernel searches the starts
// for them: that makes it 2 us longer, where the table is a launch of its own of 6 us
// for 63 sequences (11 for 164, 54 for 1022, of 385 rows each).
void plan_tiles(PackedArgs& a, long B) {
    const long most = a.T / PACKED_ROWS + B + 2;
    // a launch's threads are counted in 32 bits; tiles are rounded up to the XCDs that
    // share a kv head
    const long share = 8 % a.Hk ? 1 : 8 / a.Hk;
    TORCH_CHECK((2 * most + share - 1) / share * share * a.Hq * 256 < (1L << 32),
                "too many rows, sequences and heads for one call");
    a.B = (int)B;
    a.max_tiles = (int)most;
    a.search = B <= PACKED_FEW;
}

// In how many parts the kernel for dk and dv may take a workgroup's queries.  It
// splits only what is longer than the card's share, so nothing where all rows
// together are not; workgroups of parts that are not there cost a little, and each
// part's sums are a copy of dk and dv in fp32.  dq and dk/dv with 1, 2 and 4 parts at
// most (us), by workgroups:
//   32/8 heads of 128 (256 run at once)      8/4 heads of 64 (768)
//     88  1024             143 102  84         88  1024            51  41  39
//    152  2048             290 203 197        280  4096           175 139 118
//    280  4096             655 585 587        536  8192           400 347 343
//    304  4 x 1024         201 180 181        792  12288          669 638 639
//    560  4096 to 596      775 731 739       1528  24000         2014 2001 2015
//    592  8 x 1024         328 327 327       2350  36 x 64..1536  188 189 193
void plan_parts(PackedArgs& a, bool keys) {
    const long slots = packed_slots(a.D);
    const long all = (long)a.max_tiles * a.Hk * (PACKED_ROWS / packed_keys(a.D));
    const long steps = ((a.T - 1) / packed_keys(a.D) + 1) * (long)(a.Hq / a.Hk);
    a.parts = !keys || steps <= packed_worth(a.D) || all > 3 * slots ? 1 : all > slots ? 2 : 4;
    a.counters = a.parts > 1 ? (int)all : 0;
}

// What the forward pass keeps for the backward one, and the table of tiles.
struct Kept {
    Parts parts;
    size_t tiles, rest = 0, lse = 0;
    Kept(const PackedArgs& a, bool save)
        : tiles(parts.add(save || !a.search ? 32 * (size_t)a.max_tiles + 16 : 0)) {
        if (!save) return;
        rest = parts.add(2 * (size_t)a.T * a.Hq * a.D);
        lse = parts.add(4 * (size_t)a.T * a.Hq);
    }
};

// -> out and, with `save`, what the backward pass needs
std::vector<Tensor> packed_attn_fwd(const Tensor& q, const Tensor& k, const Tensor& v,
                                    const Tensor& starts, double scale, bool save) {
    PackedArgs a = packed_args(q, k, v, scale);
    plain(starts, "seq_starts");
    TORCH_CHECK(starts.device() == q.device() && starts.scalar_type() == torch::kInt32 &&
                    starts.is_contiguous() && starts.dim() == 1 && starts.numel() >= 1,
                "seq_starts must be a dense int32 vector on the device of q");
    const c10::cuda::CUDAGuard guard(q.device());
    const Tensor out = blank({a.T, a.Hq, a.D}, q.options());
    plan_tiles(a, starts.numel() - 1);
    const Kept at(a, save);
    Tensor kept;
    if (at.parts.size) {
        kept = at.parts.make(q);
        a.tiles = part<void>(kept, at.tiles);
    }
    a.starts = starts.data_ptr<int>();
    a.out = bf16(out);
    if (save) {
        a.out_lo = part<unsigned short>(kept, at.rest);
        a.lse = part<float>(kept, at.lse);
    }
    if (a.T > 0) {
        void* st = stream_of(q);
        if (!a.search) launched(launch_packed_tiles(&a, st), "packed_attention");
        launched(launch_packed_attn_fwd(&a, st), "packed_attention");
    }
    return {out, kept};
}

// -> dq, dk, dv (the last two undefined without `keys`)
std::vector<Tensor> packed_attn_bwd(const Tensor& dout, const Tensor& q, const Tensor& k,
                                    const Tensor& v, const Tensor& out, const Tensor& kept,
                                    long B, double scale, bool keys) {
    PackedArgs a = packed_args(q, k, v, scale);
    check_rows(dout, "the gradient", q);
    TORCH_CHECK(dout.sizes() == q.sizes(), "the gradient must have the shape of q");
    const c10::cuda::CUDAGuard guard(q.device());
    const auto opt = q.options();
    const Tensor dq = blank({a.T, a.Hq, a.D}, opt);
    Tensor dk, dv;
    if (keys) {
        dk = blank({a.T, a.Hk, a.D}, opt);
        dv = blank({a.T, a.Hk, a.D}, opt);
    }
    if (a.T > 0) {
        plan_tiles(a, B);
        Parts parts;
        const size_t delta = parts.add(4 * (size_t)a.Hq * a.T);
        plan_parts(a, keys);
        const size_t counts = parts.add(a.parts > 1 ? 4 * (size_t)a.counters : 0);
        const size_t sums = parts.add(a.parts > 1 ? 8 * (size_t)a.parts * a.Hk * a.T * a.D : 0);
        const Tensor scratch = parts.make(q);
        const Kept at(a, true);
        a.tiles = part<void>(kept, at.tiles);
        a.out = bf16(out);
        a.out_lo = part<unsigned short>(kept, at.rest);
        a.lse = part<float>(kept, at.lse);
        a.dout = bf16(dout); a.ot = dout.stride(0); a.oh = dout.stride(1);
        a.delta = part<float>(scratch, delta);
        a.counts = part<int>(scratch, counts);
        a.sums = part<float>(scratch, sums);
        a.dq = bf16(dq);
        void* st = stream_of(q);
        launched(launch_packed_attn_dq(&a, st), "packed_attention's gradient");
        if (keys) {
            a.dk = bf16(dk);
            a.dv = bf16(dv);
            launched(launch_packed_attn_dkv(&a, st), "packed_attention's gradient");
        }
    }
    return {dq, dk, dv};
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q0,
                          const Tensor& k0, const Tensor& v0, const Tensor& starts,
                          double scale) {
        const Tensor q = rows16(q0), k = rows16(k0), v = rows16(v0);
        const auto got = packed_attn_fwd(q, k, v, starts, scale, true);
        ctx->save_for_backward({q, k, v, got[0], got[1]});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["sequences"] = starts.numel() - 1;
        return got[0];
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list g) {
        const auto s = ctx->get_saved_variables();
        auto d = packed_attn_bwd(rows16(g[0]), s[0], s[1], s[2], s[3], s[4],
                                 ctx->saved_data["sequences"].toInt(),
                                 ctx->saved_data["scale"].toDouble(),
                                 ctx->needs_input_grad(1) || ctx->needs_input_grad(2));
        d = once(std::move(d), "packed_attention");
        return {d[0], d[1], d[2], Tensor(), Tensor()};
    }
};

// The starts as the kernels take them.  No other value's low 32 bits.
Tensor starts32(const Tensor& starts, const Tensor& q) {
    Tensor s = starts;
    if (s.scalar_type() != torch::kInt32) s = s.clamp(-1, (1L << 31) - 1).to(torch::kInt32);
    if (s.device() != q.device()) s = s.to(q.device());
    return s.contiguous();
}

Tensor packed_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts0,
                        std::optional<double> scale0) {
    TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.dim() == 3,
                      "q, k and v must be [tokens, heads, head dim]");
    TORCH_CHECK_VALUE(k.sizes() == v.sizes() && q.size(0) == k.size(0) && q.size(2) == k.size(2),
                      "shapes do not fit: q ", q.sizes(), ", k ", k.sizes(), ", v ", v.sizes());
    TORCH_CHECK_VALUE(q.size(1) > 0 && k.size(1) > 0 && q.size(1) % k.size(1) == 0, q.size(1),
                      " query heads are no multiple of ", k.size(1), " key/value heads");
    TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type() &&
                          q.device() == k.device() && q.device() == v.device(),
                      "q, k and v must have one type and device");
    const auto kind = starts0.scalar_type();
    TORCH_CHECK_VALUE(starts0.dim() == 1 && starts0.numel() >= 1 &&
                          (kind == torch::kInt32 || kind == torch::kInt64),
                      "seq_starts must be a vector of whole numbers, one more than sequences");
    TORCH_CHECK_VALUE(q.scalar_type() == torch::kBFloat16,
                      "on the GPU q, k and v must be bfloat16, not ", q.scalar_type());
    TORCH_CHECK_VALUE(q.size(2) == 64 || q.size(2) == 128,
                      "on the GPU the head dim must be 64 or 128, not ", q.size(2));
    plain(q, "q");
    plain(k, "k");
    plain(v, "v");
    plain(starts0, "seq_starts");
    const double scale = scale0 ? *scale0 : 1.0 / std::sqrt((double)q.size(2));
    // times log2(e) it is still an fp32 number; a 0 would make NaN of shut places' -inf
    TORCH_CHECK_VALUE(scale >= 0x1p-126 && scale < 0x1p127,
                      "scale must be positive and a normal fp32 number, not ", scale);
    const Tensor starts = starts32(starts0, q);
    if (torch::GradMode::is_enabled() &&
        (q.requires_grad() || k.requires_grad() || v.requires_grad()))
        return PackedAttention::apply(q, k, v, starts, scale);
    return packed_attn_fwd(rows16(q), rows16(k), rows16(v), starts, scale, false)[0];
}

// --------------------------------------------------------------- cross-entropy

int kind_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case torch::kFloat32: return 0;
        case torch::kBFloat16: return 1;
        case torch::kFloat16: return 2;
        default: TORCH_CHECK_VALUE(false, name, " must be float32, bfloat16 or float16");
    }
}

void check_logits(const Tensor& x, const Tensor& targets) {
    plain(x, "logits");
    plain(targets, "targets");
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(1) >= 1 &&
                    (x.size(1) == 1 || x.stride(1) == 1),
                "logits must be [rows, vocabulary] on the GPU with dense rows");
    TORCH_CHECK(x.size(0) < (1L << 31) && x.size(1) < (1L << 30), "logits are too large");
    TORCH_CHECK(targets.device() == x.device() && targets.scalar_type() == torch::kInt64 &&
                    targets.is_contiguous() && targets.dim() == 1 &&
                    targets.numel() == x.size(0),
                "targets must be a dense int64 vector with one label a row, beside the logits");
}

// What the loss leaves: of every row its maximum and 1 / sum, the factor before
// a row's gradient, and what is needed on the way to a sum of rows.
struct Losses {
    Parts parts;
    size_t stats, factor, rows = 0, sums = 0, counts = 0;
    Losses(long N, long workgroups, bool mode, bool save)
        : stats(parts.add(save ? 8 * N : 0)), factor(parts.add(mode ? 4 : 0)) {
        if (!mode) return;
        rows = parts.add(4 * N);
        sums = parts.add(8 * workgroups);
        counts = parts.add(4 * workgroups);
    }
};

// mode 0: the loss of each row, 1: their mean, 2: their sum -> it and what the
// backward pass needs
std::vector<Tensor> xent_fwd(const Tensor& x, const Tensor& targets, int64_t ignore,
                             int64_t mode, bool save) {
    check_logits(x, targets);
    const int kind = kind_of(x, "logits");
    const int N = (int)x.size(0), V = (int)x.size(1);
    const c10::cuda::CUDAGuard guard(x.device());
    const auto opt = x.options().dtype(torch::kFloat32);
    const Tensor result = mode ? blank({}, opt) : blank({N}, opt);
    const int parts = N > 0 ? xent_parts(N, V) : 0;
    const Losses at(N, parts, mode != 0, save);
    Tensor kept;
    if (at.parts.size) kept = at.parts.make(x);
    double* sums = mode ? part<double>(kept, at.sums) : nullptr;
    int* counts = mode ? part<int>(kept, at.counts) : nullptr;
    void* st = stream_of(x);
    if (N > 0)
        launched(launch_xent_fwd(kind, x.data_ptr(), x.stride(0), targets.data_ptr(), ignore, N,
                                 V, mode ? part<void>(kept, at.rows) : result.data_ptr(),
                                 save ? part<void>(kept, at.stats) : nullptr, sums, counts, st),
                 "cross_entropy");
    if (mode)
        launched(launch_xent_reduce(sums, counts, parts, mode == 1, result.data_ptr(),
                                    part<void>(kept, at.factor), st), "cross_entropy");
    return {result, kept};
}

Tensor xent_bwd(const Tensor& gout, const Tensor& x, const Tensor& targets, int64_t ignore,
                int64_t mode, const Tensor& kept) {
    check_logits(x, targets);
    const int kind = kind_of(x, "logits");
    const int N = (int)x.size(0), V = (int)x.size(1);
    plain(gout, "the gradient");
    TORCH_CHECK(gout.device() == x.device() && gout.scalar_type() == torch::kFloat32 &&
                    (gout.dim() == 0 || (gout.dim() == 1 && gout.numel() == N)),
                "the gradient must be float32, one value or one a row");
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor dx = blank({N, V}, x.options());
    const Losses at(N, N > 0 ? xent_parts(N, V) : 0, mode != 0, true);
    if (N > 0)
        launched(launch_xent_bwd(kind, x.data_ptr(), x.stride(0), targets.data_ptr(), ignore, N,
                                 V, part<void>(kept, at.stats), gout.data_ptr(),
                                 gout.dim() ? gout.stride(0) : 0,
                                 mode ? part<void>(kept, at.factor) : nullptr, dx.data_ptr(), V,
                                 stream_of(x)),
                 "cross_entropy's gradient");
    return dx;
}

struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x,
                          const Tensor& targets, int64_t ignore, int64_t mode) {
        const auto got = xent_fwd(x, targets, ignore, mode, true);
        ctx->save_for_backward({x, targets, got[1]});
        ctx->saved_data["ignore"] = ignore;
        ctx->saved_data["mode"] = mode;
        return got[0];
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list g) {
        const auto s = ctx->get_saved_variables();
        const auto d = once({xent_bwd(g[0], s[0], s[1], ctx->saved_data["ignore"].toInt(),
                                      ctx->saved_data["mode"].toInt(), s[2])},
                            "cross_entropy");
        return {d[0], Tensor(), Tensor(), Tensor()};
    }
};

Tensor cross_entropy(const Tensor& x0, const Tensor& targets0, int64_t ignore, int64_t mode) {
    TORCH_CHECK_VALUE(x0.dim() == 2 && x0.size(1) >= 1 && targets0.dim() == 1 &&
                          targets0.size(0) == x0.size(0),
                      "logits must be [rows, vocabulary] with one label a row: logits ",
                      x0.sizes(), ", targets ", targets0.sizes());
    const auto type = targets0.scalar_type();
    TORCH_CHECK_VALUE(type == torch::kInt32 || type == torch::kInt64,
                      "targets must be whole numbers, not ", type);
    TORCH_CHECK_VALUE(targets0.device() == x0.device(),
                      "logits and targets must be on one device");
    kind_of(x0, "on the GPU logits");
    plain(x0, "logits");
    plain(targets0, "targets");
    const Tensor targets = targets0.to(torch::kInt64).contiguous();
    const Tensor x = x0.stride(1) == 1 ? x0 : x0.contiguous();
    if (torch::GradMode::is_enabled() && x.requires_grad())
        return CrossEntropy::apply(x, targets, ignore, mode);
    return xent_fwd(x, targets, ignore, mode, false)[0];
}

// --------------------------------------------------------------- gradient norm

struct Grads {
    std::vector<Tensor> at;     // dense memory, one for each gradient
    std::vector<long> copied;   // those that are copies, to be written back
    std::vector<GradTable> tables;
    std::vector<int> blocks;
    int partial = 0;
};

// Whether no two elements share memory, as in every slice of a dense tensor:
// each stride reaches over all that the smaller ones cover.
bool apart(const Tensor& t) {
    std::vector<std::pair<long, long>> dims;
    for (int64_t a = 0; a < t.dim(); ++a)
        if (t.size(a) > 1) dims.emplace_back(t.stride(a), t.size(a));
    std::sort(dims.begin(), dims.end());
    long reach = 0;
    for (const auto& d : dims) {
        if (d.first <= reach) return false;
        reach += (d.second - 1) * d.first;
    }
    return true;
}

Grads collect(const std::vector<Tensor>& grads, bool write) {
    Grads g;
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor& t = grads[i];
        TORCH_CHECK_VALUE(t.layout() == torch::kStrided && t.is_cuda() &&
                              t.device() == grads[0].device(),
                          "gradients must be dense and on one device");
        kind_of(t, "gradients");
        plain(t, "a gradient");
        if (t.numel() == 0) continue;
        Tensor d = t;
        if (!t.is_non_overlapping_and_dense()) {
            TORCH_CHECK_VALUE(!write || apart(t),
                              "a gradient must not share memory between its elements");
            d = t.clone(at::MemoryFormat::Contiguous);
            plain(d, "a gradient's copy");
            g.copied.push_back((long)i);
        }
        if (write) {
            long last = 0;
            for (int64_t a = 0; a < t.dim(); ++a) last += (t.size(a) - 1) * t.stride(a);
            const auto p = reinterpret_cast<uintptr_t>(t.data_ptr());
            spans.emplace_back(p, p + (last + 1) * t.element_size());
        }
        g.at.push_back(d);
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        TORCH_CHECK_VALUE(spans[i].first >= spans[i - 1].second,
                          "two of the gradients share or interleave their memory");
    for (const Tensor& d : g.at) {
        const long size = d.element_size();
        const auto p = reinterpret_cast<uintptr_t>(d.data_ptr());
        const long chunks = ((long)(p & 15) / size + d.numel() + GRAD_CHUNK - 1) / GRAD_CHUNK;
        TORCH_CHECK(p % size == 0 && chunks < (1L << 30), "a gradient is too large");
        if (g.tables.empty() || g.tables.back().n == GRAD_TENSORS ||
            g.tables.back().first[g.tables.back().n] + chunks >= (1L << 30)) {
            g.tables.emplace_back();
            g.tables.back().n = 0;
            g.tables.back().first[0] = 0;
        }
        GradTable& t = g.tables.back();
        t.ptr[t.n] = d.data_ptr();
        t.size[t.n] = d.numel();
        t.kind[t.n] = (unsigned char)kind_of(d, "gradients");
        t.first[t.n + 1] = t.first[t.n] + (int)chunks;
        ++t.n;
    }
    for (const GradTable& t : g.tables) {
        g.blocks.push_back(std::min(t.first[t.n], 1024));
        g.partial += g.blocks.back();
    }
    return g;
}

Tensor sums_of(const Grads& g, const Tensor& like, void* st) {
    Tensor sums = blank({g.partial}, like.options().dtype(torch::kFloat64));
    int at = 0;
    for (size_t i = 0; i < g.tables.size(); ++i) {
        launched(launch_grad_sums(&g.tables[i], g.blocks[i], sums.data_ptr<double>() + at, st),
                 "the gradient norm");
        at += g.blocks[i];
    }
    return sums;
}

std::vector<Tensor> grads_of(const std::vector<Tensor>& parameters) {
    std::vector<Tensor> grads;
    for (const Tensor& p : parameters)
        if (p.grad().defined()) grads.push_back(p.grad());
    TORCH_CHECK_VALUE(!grads.empty(), "no parameter has a gradient");
    return grads;
}

Tensor grad_norm(const std::vector<Tensor>& parameters) {
    const std::vector<Tensor> grads = grads_of(parameters);
    const at::NoGradGuard no_grad;
    const Grads g = collect(grads, false);
    const c10::cuda::CUDAGuard guard(grads[0].device());
    void* st = stream_of(grads[0]);
    Tensor norm = blank({}, grads[0].options().dtype(torch::kFloat32));
    const Tensor sums = sums_of(g, norm, st);
    launched(launch_grad_norm(sums.data_ptr(), g.partial, norm.data_ptr(), st),
             "the gradient norm");
    return norm;
}

Tensor grad_clip(const std::vector<Tensor>& parameters, double limit, double eps) {
    const std::vector<Tensor> grads = grads_of(parameters);
    const at::NoGradGuard no_grad;
    const Grads g = collect(grads, true);
    const c10::cuda::CUDAGuard guard(grads[0].device());
    void* st = stream_of(grads[0]);
    Tensor norm = blank({}, grads[0].options().dtype(torch::kFloat32));
    const Tensor sums = sums_of(g, norm, st);
    if (g.tables.empty())
        launched(launch_grad_norm(sums.data_ptr(), 0, norm.data_ptr(), st), "the gradient norm");
    for (size_t i = 0; i < g.tables.size(); ++i)
        launched(launch_grad_clip(&g.tables[i], g.blocks[i], sums.data_ptr(), g.partial, limit,
                                  eps, i ? nullptr : norm.data_ptr(), st),
                 "clipping gradients");
    size_t k = 0;
    for (size_t i = 0, c = 0; i < grads.size(); ++i) {
        if (grads[i].numel() == 0) continue;
        if (c < g.copied.size() && g.copied[c] == (long)i) {
            grads[i].copy_(g.at[k]);
            ++c;
        } else if (!grads[i].is_inference()) {
            grads[i].unsafeGetTensorImpl()->bump_version();
        }
        ++k;
    }
    return norm;
}

}  // namespace

void bind_training(pybind11::module_& m) {
    m.def("packed_attention", &packed_attention,
          "causal attention of packed sequences, with gradients");
    m.def("cross_entropy", &cross_entropy, "cross-entropy of rows with labels, with gradient");
    m.def("grad_norm", &grad_norm, "norm of all gradients together");
    m.def("grad_clip", &grad_clip, "norm of all gradients together, and clipping by it");
}
