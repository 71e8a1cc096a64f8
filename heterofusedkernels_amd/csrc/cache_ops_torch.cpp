// The cache and attention ops of the pcie_through namespace: cache_write, cache_read, prompt_attention and
// prefix_attention over the C-ABI of libhfk_hip.so. Like the ops of pcie_through_ops.cpp they run on the current stream
// of the device that owns the cache, write into tensors the caller gives and wait for nothing. The attention ops
// take their workspace from torch's allocator, so that concurrent calls and captured graphs each have their own.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <initializer_list>
#include <optional>

#include "hfk.h"

namespace pciethrough {

namespace {

using OptTensor = std::optional<at::Tensor>;

hfk_stream_t stream_of_current_device() {
    return static_cast<hfk_stream_t>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream());
}

void check_call(int rc, const char* entry) {
    TORCH_CHECK(rc == 0, entry, " failed: ", hfk_status_string(rc), " (", rc, ")");
}

uint32_t row_type(const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, what, " must be bfloat16 or float16, got ",
                c10::toString(t.scalar_type()));
    return t.scalar_type() == at::kBFloat16 ? HFK_BF16 : HFK_FP16;
}

void check_on(const at::Tensor& t, const at::Tensor& cache, const char* what) {
    TORCH_CHECK(t.device() == cache.device(), what, " must be on the cache's device ", cache.device(), ", got ", t.device());
}

void check_written(const at::Tensor& t, const char* what) {
    TORCH_CHECK(at::has_internal_overlap(t) != at::MemOverlap::Yes, what, " is written and must not overlap itself");
}

// An argument and the bytes from its first value to its last one; none where it is not given or empty.
struct Named {
    const at::Tensor* tensor = nullptr;
    const char* name;
    uintptr_t first = 0, end = 0;
    Named(const at::Tensor& t, const char* name) : tensor(&t), name(name) {
        if (t.numel() == 0) return;
        const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
        int64_t last = 0;
        for (size_t i = 0; i < sizes.size(); ++i) last += (sizes[i] - 1) * strides[i];
        first = reinterpret_cast<uintptr_t>(t.const_data_ptr());
        end = first + static_cast<uintptr_t>(last + 1) * t.element_size();
    }
    Named(const OptTensor& t, const char* name) : name(name) {
        if (t.has_value()) *this = Named(*t, name);
    }
};

// What is written lies apart from everything else that is written and from everything that is read: rows are read and written
// by different workgroups in no order. Views whose overlap cannot be told at a glance are the caller's. (Most pairs are apart by their
// addresses, which costs a call of one token 0.1 us; at::get_overlap_status for each of them 0.3.)
void check_apart(std::initializer_list<Named> written, std::initializer_list<Named> read) {
    const auto check = [](const Named& a, const Named& b) {
        if (a.first >= b.end || b.first >= a.end) return;
        const at::MemOverlapStatus s = at::get_overlap_status(*a.tensor, *b.tensor);
        TORCH_CHECK(a.first != b.first && s != at::MemOverlapStatus::Partial && s != at::MemOverlapStatus::Full, a.name, " and ", b.name,
                    " must not overlap");
    };
    for (const Named* w = written.begin(); w != written.end(); ++w) {
        for (const Named* other = w + 1; other != written.end(); ++other) check(*w, *other);
        for (const Named& r : read) check(*w, r);
    }
}

// Results in place of the queries: every value where its query's was, or nowhere near.
void check_in_place(const at::Tensor& out, const at::Tensor& q) {
    bool sound = at::get_overlap_status(out, q) != at::MemOverlapStatus::Partial;
    if (q.numel() != 0 && out.const_data_ptr() == q.const_data_ptr())
        for (int64_t i = 0; i < q.dim(); ++i) sound &= q.size(i) == 1 || q.stride(i) == out.stride(i);
    TORCH_CHECK(sound, "out and q, unless they are one tensor, must not overlap");
}

void check_no_gradient(const at::Tensor& t, const char* what) {
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what,
                " requires a gradient, which this op does not compute: detach it or call the op under torch.no_grad()");
    TORCH_CHECK(!t._fw_grad(0).defined(), what, " carries a tangent, which this op does not pass on: give its primal alone");
}
void check_no_gradient(const OptTensor& t, const char* what) {
    if (t.has_value()) check_no_gradient(*t, what);
}

void check_index(const at::Tensor& t, const at::Tensor& cache, int64_t dims, const char* what) {
    check_on(t, cache, what);
    TORCH_CHECK(t.scalar_type() == at::kLong, what, " must be int64");
    TORCH_CHECK(t.dim() == dims, what, " must have ", dims, " dimension(s), got ", t.dim());
    TORCH_CHECK(t.is_contiguous(), what, " must be contiguous");
}

// [blocks, T, heads, dim] and, for e4m3 values, [blocks, T, heads] scales.
hfk_cache_plane plane_of(const at::Tensor& cache, const OptTensor& scales, const char* what) {
    TORCH_CHECK(cache.is_cuda(), what, " must be a device tensor");
    TORCH_CHECK(cache.dim() == 4, what, " must be [blocks, blockSize, heads, headDim], got ", cache.dim(), " dims");
    TORCH_CHECK(cache.numel() == 0 || cache.stride(3) == 1, what, ": values of a head must be contiguous");
    hfk_cache_plane p{};
    if (cache.scalar_type() == at::kFloat8_e4m3fn) {
        p.type = HFK_FP8_E4M3;
        TORCH_CHECK(scales.has_value(), what, " holds float8_e4m3fn values: its scales are needed");
        TORCH_CHECK(scales->scalar_type() == at::kFloat, what, ": scales must be float32");
        check_on(*scales, cache, "scales");
        TORCH_CHECK(scales->dim() == 3 && scales->size(0) == cache.size(0) && scales->size(1) == cache.size(1) &&
                        scales->size(2) == cache.size(2),
                    what, ": scales must be [blocks, blockSize, heads]");
        p.scales = scales->data_ptr<float>();
        p.scale_block_stride = scales->stride(0);
        p.scale_token_stride = scales->stride(1);
        p.scale_head_stride = scales->stride(2);
    } else {
        TORCH_CHECK(cache.scalar_type() == at::kBFloat16 || cache.scalar_type() == at::kHalf, what,
                    " must be bfloat16, float16 or float8_e4m3fn, got ", c10::toString(cache.scalar_type()));
        TORCH_CHECK(!scales.has_value(), what, ": only a float8_e4m3fn cache has scales");
        p.type = row_type(cache, what);
    }
    for (int i = 1; i < 4; ++i) {
        TORCH_CHECK(cache.size(i) > 0 && cache.size(i) <= 0xffffffffLL, what, ": dimension ", i, " is empty or too large");
    }
    p.values = cache.data_ptr();
    p.block_stride = cache.stride(0);
    p.token_stride = cache.stride(1);
    p.head_stride = cache.stride(2);
    p.blocks = static_cast<uint64_t>(cache.size(0));
    p.block_tokens = static_cast<uint32_t>(cache.size(1));
    p.heads = static_cast<uint32_t>(cache.size(2));
    p.head_dim = static_cast<uint32_t>(cache.size(3));
    return p;
}

// [n, heads, dim]
hfk_token_rows rows_of(const at::Tensor& t, const at::Tensor& cache, int64_t n, int64_t heads, const char* what) {
    check_on(t, cache, what);
    TORCH_CHECK(t.dim() == 3 && t.size(0) == n && t.size(1) == heads && t.size(2) == cache.size(3), what, " must be [", n, ", ",
                heads, ", ", cache.size(3), "], got ", t.sizes());
    TORCH_CHECK(t.numel() == 0 || t.stride(2) == 1, what, ": values of a head must be contiguous");
    hfk_token_rows r{};
    r.data = t.data_ptr();
    r.token_stride = t.stride(0);
    r.head_stride = t.stride(1);
    r.type = row_type(t, what);
    return r;
}

// The two sides of cache_write and cache_read, checked and unpacked.
struct Tokens {
    hfk_cache_plane plane[2];
    hfk_token_rows rows[2];
    int64_t n;
    bool both;
};

Tokens tokens_of(const at::Tensor& k, const at::Tensor& kCache, const at::Tensor& slots, const OptTensor& v, const OptTensor& vCache,
                 const OptTensor& kScales, const OptTensor& vScales) {
    Tokens t{};
    TORCH_CHECK(v.has_value() == vCache.has_value(), "v and vCache go together");
    TORCH_CHECK(vCache.has_value() || !vScales.has_value(), "vScales without vCache");
    t.plane[0] = plane_of(kCache, kScales, "kCache");
    check_index(slots, kCache, 1, "slots");
    t.n = slots.size(0);
    t.rows[0] = rows_of(k, kCache, t.n, kCache.size(2), "k");
    t.both = v.has_value();
    if (t.both) {
        check_on(*vCache, kCache, "vCache");
        TORCH_CHECK(vCache->scalar_type() == kCache.scalar_type(), "kCache and vCache must have one type, got ",
                    c10::toString(kCache.scalar_type()), " and ", c10::toString(vCache->scalar_type()));
        t.plane[1] = plane_of(*vCache, vScales, "vCache");      // so that both have scales or neither has
        t.rows[1] = rows_of(*v, *vCache, t.n, vCache->size(2), "v");
    }
    check_no_gradient(k, "k");
    check_no_gradient(v, "v");
    check_no_gradient(kCache, "kCache");
    check_no_gradient(vCache, "vCache");
    check_no_gradient(kScales, "kScales");
    check_no_gradient(vScales, "vScales");
    return t;
}

}  // namespace

// Tokens into the cache; see hfk_cache_write.
void cache_write(const at::Tensor& k, const at::Tensor& kCache, const at::Tensor& slots, const OptTensor& v, const OptTensor& vCache,
                 const OptTensor& kScales, const OptTensor& vScales) {
    const Tokens t = tokens_of(k, kCache, slots, v, vCache, kScales, vScales);
    check_written(kCache, "kCache");
    if (kScales.has_value()) check_written(*kScales, "kScales");
    if (t.both) check_written(*vCache, "vCache");
    if (vScales.has_value()) check_written(*vScales, "vScales");
    check_apart({{kCache, "kCache"}, {vCache, "vCache"}, {kScales, "kScales"}, {vScales, "vScales"}},
                {{k, "k"}, {v, "v"}, {slots, "slots"}});
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(kCache));
    check_call(hfk_cache_write(&t.plane[0], &t.rows[0], t.both ? &t.plane[1] : nullptr, t.both ? &t.rows[1] : nullptr,
                               slots.data_ptr<int64_t>(), static_cast<uint64_t>(t.n), stream_of_current_device()),
               "hfk_cache_write");
}

// Tokens out of the cache; see hfk_cache_read.
void cache_read(const at::Tensor& kCache, const at::Tensor& k, const at::Tensor& slots, const OptTensor& vCache, const OptTensor& v,
                const OptTensor& kScales, const OptTensor& vScales) {
    const Tokens t = tokens_of(k, kCache, slots, v, vCache, kScales, vScales);
    check_written(k, "k");
    if (t.both) check_written(*v, "v");
    check_apart({{k, "k"}, {v, "v"}},
                {{kCache, "kCache"}, {vCache, "vCache"}, {kScales, "kScales"}, {vScales, "vScales"}, {slots, "slots"}});
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(kCache));
    check_call(hfk_cache_read(&t.plane[0], &t.rows[0], t.both ? &t.plane[1] : nullptr, t.both ? &t.rows[1] : nullptr,
                              slots.data_ptr<int64_t>(), static_cast<uint64_t>(t.n), stream_of_current_device()),
               "hfk_cache_read");
}

namespace {

hfk_attention attention_of(const at::Tensor& q, const at::Tensor& kCache, const at::Tensor& vCache, const at::Tensor& out,
                           double scale, const OptTensor& kScales, const OptTensor& vScales, const OptTensor& lse) {
    hfk_attention a{};
    a.k = plane_of(kCache, kScales, "kCache");
    a.v = plane_of(vCache, vScales, "vCache");
    check_on(vCache, kCache, "vCache");
    TORCH_CHECK(vCache.sizes() == kCache.sizes() && vCache.scalar_type() == kCache.scalar_type(),
                "kCache and vCache must have one shape and one type");
    TORCH_CHECK(q.dim() == 3, "q must be [tokens, heads, headDim], got ", q.dim(), " dims");
    a.q = rows_of(q, kCache, q.size(0), q.size(1), "q");
    a.out = rows_of(out, kCache, q.size(0), q.size(1), "out");
    check_written(out, "out");
    check_in_place(out, q);
    check_apart({{lse, "lse"}}, {{q, "q"}});
    check_apart({{out, "out"}, {lse, "lse"}}, {{kCache, "kCache"}, {vCache, "vCache"}, {kScales, "kScales"}, {vScales, "vScales"}});
    check_no_gradient(q, "q");
    check_no_gradient(kCache, "kCache");
    check_no_gradient(vCache, "vCache");
    check_no_gradient(kScales, "kScales");
    check_no_gradient(vScales, "vScales");
    check_no_gradient(out, "out");
    check_no_gradient(lse, "lse");
    TORCH_CHECK(q.size(1) > 0 && q.size(1) <= 0xffffffffLL && q.size(1) % kCache.size(2) == 0, "q has ", q.size(1),
                " heads, which is no multiple of the cache's ", kCache.size(2));
    TORCH_CHECK(out.scalar_type() == q.scalar_type(), "out must have q's type");
    TORCH_CHECK(a.k.type == HFK_FP8_E4M3 || a.k.type == a.q.type, "the cache must hold q's type or float8_e4m3fn");
    TORCH_CHECK(kCache.size(3) % 16 == 0 && kCache.size(3) <= 256, "headDim must be a multiple of 16 up to 256, got ", kCache.size(3));
    a.n_rows = static_cast<uint64_t>(q.size(0));
    a.q_heads = static_cast<uint32_t>(q.size(1));
    a.scale = static_cast<float>(scale);
    TORCH_CHECK(a.scale >= 0x1p-100f && a.scale <= 0x1p100f, "scale must be positive and finite, from 2^-100 to 2^100, got ", scale);
    if (lse.has_value()) {
        check_on(*lse, kCache, "lse");
        TORCH_CHECK(lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->dim() == 2 && lse->size(0) == q.size(0) &&
                        lse->size(1) == q.size(1),
                    "lse must be a contiguous float32 tensor [", q.size(0), ", ", q.size(1), "]");
        a.lse = lse->data_ptr<float>();
    }
    return a;
}

// From torch's allocator, on the current stream: the memory is free for others once the stream has passed the call.
at::Tensor workspace_of(const at::Tensor& q, uint64_t bytes) {
    return bytes == 0 ? at::Tensor() : at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
}

}  // namespace

// Packed prompts over the paged cache; see hfk_prompt_attention.
void prompt_attention(const at::Tensor& q, const at::Tensor& kCache, const at::Tensor& vCache, const at::Tensor& blockTable,
                      const at::Tensor& queryStarts, const at::Tensor& kvLens, const at::Tensor& out, double scale, bool causal,
                      const OptTensor& kScales, const OptTensor& vScales, const OptTensor& lse) {
    const hfk_attention a = attention_of(q, kCache, vCache, out, scale, kScales, vScales, lse);
    check_index(blockTable, kCache, 2, "blockTable");
    check_index(queryStarts, kCache, 1, "queryStarts");
    check_index(kvLens, kCache, 1, "kvLens");
    const int64_t n = kvLens.size(0);
    TORCH_CHECK(blockTable.size(0) == n && queryStarts.size(0) == n + 1, "blockTable must have one row and queryStarts one entry more per kvLens' ",
                n, " sequences, got ", blockTable.size(0), " and ", queryStarts.size(0));
    check_apart({{out, "out"}, {lse, "lse"}}, {{blockTable, "blockTable"}, {queryStarts, "queryStarts"}, {kvLens, "kvLens"}});
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(kCache));
    const uint64_t width = static_cast<uint64_t>(blockTable.size(1));
    uint64_t bytes = 0;
    check_call(hfk_prompt_attention_workspace(&a, static_cast<uint64_t>(n), width, &bytes), "hfk_prompt_attention_workspace");
    const at::Tensor workspace = workspace_of(q, bytes);
    check_call(hfk_prompt_attention(&a, blockTable.data_ptr<int64_t>(), static_cast<uint64_t>(n), width, queryStarts.data_ptr<int64_t>(),
                                    kvLens.data_ptr<int64_t>(), causal ? 1 : 0, bytes != 0 ? workspace.data_ptr() : nullptr, bytes,
                                    stream_of_current_device()),
               "hfk_prompt_attention");
}

// One token per sequence under a common prefix; see hfk_prefix_attention.
void prefix_attention(const at::Tensor& q, const at::Tensor& kCache, const at::Tensor& vCache, const at::Tensor& prefixBlocks,
                      const at::Tensor& prefixLen, const at::Tensor& blockTable, const at::Tensor& kvLens, const at::Tensor& out,
                      double scale, const OptTensor& kScales, const OptTensor& vScales, const OptTensor& lse) {
    const hfk_attention a = attention_of(q, kCache, vCache, out, scale, kScales, vScales, lse);
    check_index(prefixBlocks, kCache, 1, "prefixBlocks");
    check_index(prefixLen, kCache, 1, "prefixLen");
    check_index(blockTable, kCache, 2, "blockTable");
    check_index(kvLens, kCache, 1, "kvLens");
    TORCH_CHECK(prefixLen.size(0) == 1, "prefixLen must hold one length");
    TORCH_CHECK(blockTable.size(0) == q.size(0) && kvLens.size(0) == q.size(0), "blockTable and kvLens must have one row per row of q");
    check_apart({{out, "out"}, {lse, "lse"}},
                {{prefixBlocks, "prefixBlocks"}, {prefixLen, "prefixLen"}, {blockTable, "blockTable"}, {kvLens, "kvLens"}});
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(kCache));
    const uint64_t prefix = static_cast<uint64_t>(prefixBlocks.size(0)), width = static_cast<uint64_t>(blockTable.size(1));
    uint64_t bytes = 0;
    check_call(hfk_prefix_attention_workspace(&a, prefix, width, &bytes), "hfk_prefix_attention_workspace");
    const at::Tensor workspace = workspace_of(q, bytes);
    check_call(hfk_prefix_attention(&a, prefixBlocks.data_ptr<int64_t>(), prefix, prefixLen.data_ptr<int64_t>(),
                                    blockTable.data_ptr<int64_t>(), width, kvLens.data_ptr<int64_t>(),
                                    bytes != 0 ? workspace.data_ptr() : nullptr, bytes, stream_of_current_device()),
               "hfk_prefix_attention");
}

}  // namespace pciethrough

TORCH_LIBRARY_FRAGMENT(pcie_through, m) {
    m.def(
        "cache_write(Tensor k, Tensor(a!) kCache, Tensor slots, Tensor? v=None, Tensor(b!)? vCache=None, Tensor(c!)? "
        "kScales=None, Tensor(d!)? vScales=None) -> ()");
    m.def(
        "cache_read(Tensor kCache, Tensor(a!) k, Tensor slots, Tensor? vCache=None, Tensor(b!)? v=None, Tensor? "
        "kScales=None, Tensor? vScales=None) -> ()");
    m.def(
        "prompt_attention(Tensor q, Tensor kCache, Tensor vCache, Tensor blockTable, Tensor queryStarts, Tensor kvLens, "
        "Tensor(a!) out, float scale, bool causal=True, Tensor? kScales=None, Tensor? vScales=None, Tensor(b!)? lse=None) -> ()");
    m.def(
        "prefix_attention(Tensor q, Tensor kCache, Tensor vCache, Tensor prefixBlocks, Tensor prefixLen, Tensor blockTable, "
        "Tensor kvLens, Tensor(a!) out, float scale, Tensor? kScales=None, Tensor? vScales=None, Tensor(b!)? lse=None) -> ()");
}

TORCH_LIBRARY_IMPL(pcie_through, CUDA, m) {
    m.impl("cache_write", TORCH_FN(pciethrough::cache_write));
    m.impl("cache_read", TORCH_FN(pciethrough::cache_read));
    m.impl("prompt_attention", TORCH_FN(pciethrough::prompt_attention));
    m.impl("prefix_attention", TORCH_FN(pciethrough::prefix_attention));
}
