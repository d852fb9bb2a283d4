// Attention: arguments, the choice of kernels, workspaces (kernels: wst_attention.h, wst_attention_t.hip).
#include <cmath>

#include "wst_attention.h"

namespace {

using namespace wst_tok;

// dslopes where no k_attn_dkv_join follows.
__global__ __launch_bounds__(1024) void k_attn_slopes(AttnArgs a) {
    __shared__ float s[16];
    add_slopes(a, blockIdx.x, s);
}

template <typename T>
struct Tag {
    using type = T;
};
template <typename F>
void with_type(int dtype, F f) {
    if (dtype == WST_F32) f(Tag<float>{});
    else if (dtype == WST_BF16) f(Tag<bf16>{});
    else f(Tag<f16>{});
}
template <typename F>
void with_width(int dim, F f) {
    if (dim <= 32) f(std::integral_constant<int, 32>{});
    else if (dim <= 64) f(std::integral_constant<int, 64>{});
    else if (dim <= 96) f(std::integral_constant<int, 96>{});
    else f(std::integral_constant<int, 128>{});
}

int check(const wst_attention_desc* d) {
    if (!d) return fail(WST_ERR_INVALID, "attention: descriptor is NULL");
    if (d->batch < 0 || d->q_len < 0 || d->k_len < 0) return fail(WST_ERR_INVALID, "attention: negative size");
    if (d->q_heads < 1 || d->k_heads < 1 || d->q_heads % d->k_heads)
        return fail(WST_ERR_INVALID, "attention: %d query heads do not share %d key heads evenly", d->q_heads, d->k_heads);
    if (d->dim < 1) return fail(WST_ERR_INVALID, "attention: bad head width %d", d->dim);
    if (d->dim > WST_MAX_HEAD_DIM) return fail(WST_ERR_UNSUPPORTED, "attention: heads wider than %d", WST_MAX_HEAD_DIM);
    if (d->dtype != WST_F32 && d->dtype != WST_BF16 && d->dtype != WST_F16) return fail(WST_ERR_INVALID, "attention: unknown type");
    if (!std::isfinite(d->scale)) return fail(WST_ERR_INVALID, "attention: scale must be finite");
    if (d->cap != 0.f && !(d->cap >= 1e-30f && d->cap <= 1e30f))
        return fail(WST_ERR_INVALID, "attention: cap must be 0 (none) or from 1e-30 to 1e30");
    // (what has no elements may have no address)
    if (d->batch && d->q_len && d->k_len && (!d->q_pos != !d->k_pos || !d->q_doc != !d->k_doc))
        return fail(WST_ERR_INVALID, "attention: positions and documents are given for queries and keys alike");
    if (d->q_pos && (d->axes < 1 || d->axes > WST_MAX_DISTANCE_AXES))
        return fail(WST_ERR_INVALID, "attention: 1 to %d axes", WST_MAX_DISTANCE_AXES);
    if (d->prefix && !d->causal) return fail(WST_ERR_INVALID, "attention: a prefix needs causal order");
    if (d->batch > 65535 || d->q_heads > 65535) return fail(WST_ERR_UNSUPPORTED, "attention: more than 65535 sequences or heads");
    // blocks of every kernel are counted in 31 bits; splits and parts are many only where rows are few
    if (static_cast<double>(d->batch) * d->q_heads * (static_cast<double>(d->q_len) / 4 + static_cast<double>(d->k_len) / 4 + 512) > 2147483647.0)
        return fail(WST_ERR_UNSUPPORTED, "attention: too many rows for one call");
    if (d->q_len > (1LL << 30) || d->k_len > (1LL << 30)) return fail(WST_ERR_UNSUPPORTED, "attention: more than 2^30 tokens");
    return WST_OK;
}

size_t rows_of(const wst_attention_desc& d) { return static_cast<size_t>(d.batch) * d.q_heads * d.q_len; }

// Rows that can be fetched 16 bytes at a time, with offsets of 32 bits inside a tile of 64.
bool lined_up(const wst_attention_desc& d, const void* p, const int64_t (&s)[3]) {
    const int64_t size = d.dtype == WST_F32 ? 4 : 2;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] * size % 16 == 0 && s[1] * size % 16 == 0 && s[2] * size % 16 == 0 &&
           s[1] >= 0 && s[1] <= (1LL << 31) / (64 * size);
}

bool can_tile(const wst_attention_desc& d) {
    return d.dim % 8 == 0 && d.dim <= 128 && d.scale != 0.f && lined_up(d, d.q, d.q_strides) && lined_up(d, d.k, d.k_strides) && lined_up(d, d.v, d.v_strides);
}

AttnPlan plan_of(const wst_attention_desc& d, bool tiles) {
    AttnPlan p{};
    p.tiles = tiles;
    const int64_t rows = static_cast<int64_t>(rows_of(d)), group = d.q_heads / d.k_heads;
    p.slots = static_cast<int>(d.q_len);
    p.parts = 1;
    if (p.tiles && rows) {
        const int64_t blocks = d.batch * d.q_heads * ((d.q_len + kBQ - 1) / kBQ);
        const int64_t row_tiles = (group * d.q_len + 31) / 32, cells = d.batch * d.k_heads * row_tiles;
        if (d.q_len <= 32 || (blocks < 128 && d.k_len >= 1024)) {
            // two blocks a CU, all at once (64 queries over 4096 keys, 2 x 64: 512 blocks 29 us, 1024 34)
            int64_t s = (512 + cells - 1) / cells, most = (d.k_len + 255) / 256;
            s = s < most ? s : most;
            p.splits = static_cast<int>(s < 1 ? 1 : s > 256 ? 256 : s);
            if (p.splits > 1) p.forward = static_cast<size_t>(p.splits) * rows * (d.dim + 2);
        }
        const int64_t items = group * ((d.q_len + 63) / 64), keys = d.batch * d.k_heads * ((d.k_len + kBQ - 1) / kBQ);
        // Blocks of dk and dv: two a CU, all at once; in order, where the first keys' walks are the longest, twice as many,
        // so that short ones come in beside long ones (8192 x 8 heads x 64: 266 us, 193 and 22 for the join; wider heads
        // have one block of eight waves a CU and are even as they are).
        const int64_t want = d.causal && d.dim <= 64 && d.dtype != WST_F32 ? 1024 : 512;
        int64_t parts = keys ? (want + keys - 1) / keys : 1;
        parts = parts < items / 2 ? parts : items / 2;
        parts = parts < 1 ? 1 : parts > 64 ? 64 : parts;
        // whole heads a part, or whole parts a head, where that takes less than twice as many (k_attn_dkv)
        int64_t even = parts;
        while (even % group && group % even) ++even;
        p.parts = static_cast<int>(even < 2 * parts ? even : parts);
        p.slots = static_cast<int>((d.q_len + kBQ - 1) / kBQ * 4);
        if (p.parts > 1) p.backward = static_cast<size_t>(p.parts) * d.batch * d.k_heads * d.k_len * 2 * d.dim;
    }
    p.backward += d.dtype == WST_F32 ? 2 * rows : rows;
    if (d.slopes) p.backward += static_cast<size_t>(d.q_heads) * d.batch * p.slots;
    return p;
}

// Whether every launch of a call has fewer than 2^32 threads along each axis: one that asks for more is cut to what is left
// of them, without an error.
bool launchable(const wst_attention_desc& d, const AttnPlan& p, bool backward) {
    auto fits = [](double blocks, int threads) { return blocks * threads < 4294967296.0; };
    const double q4 = std::ceil(d.q_len / 4.0), k4 = std::ceil(d.k_len / 4.0), seqs = d.batch;
    if (!p.tiles) return fits(q4, 256) && (!backward || fits(k4, 256));
    const double q_blocks = seqs * d.q_heads * std::ceil(d.q_len / static_cast<double>(kBQ));
    if (!backward && p.splits)
        return fits(p.splits * seqs * d.k_heads * std::ceil(static_cast<double>(d.q_heads / d.k_heads) * d.q_len / 32.0), 256);
    if (!fits(q_blocks, two_teams(d) ? 512 : 256)) return false;
    const double k_blocks = seqs * d.k_heads * std::ceil(d.k_len / static_cast<double>(kBQ));
    return !backward || (fits(q4, 256) && fits(k_blocks * p.parts, dkv_threads(d.dtype == WST_F32 ? 4 : 2, d.dim)) &&
                         (p.parts == 1 || fits(k4 + d.q_heads, 256)));
}

size_t bytes_of(const wst_attention_desc& d, int backward) {
    // either way of running: the gradient of the output, which decides with the rest, is not known here
    const AttnPlan p = plan_of(d, true), q = plan_of(d, false);
    const size_t b = p.backward > q.backward ? p.backward : q.backward;
    return sizeof(float) * (backward ? b : p.forward);
}

}  // namespace

extern "C" {

int wst_attention_workspace(const wst_attention_desc* d, int backward, size_t* bytes) {
    if (!bytes) return fail(WST_ERR_INVALID, "attention: bytes is NULL");
    if (const int e = check(d)) return e;
    *bytes = bytes_of(*d, backward);
    return WST_OK;
}

int wst_attention_forward(const wst_attention_desc* d, void* o, float* lse, void* workspace, size_t workspace_bytes,
                          void* stream) {
    if (const int e = check(d)) return e;
    if (rows_of(*d) == 0) return WST_OK;
    if (!d->q || !o || (d->k_len && (!d->k || !d->v))) return fail(WST_ERR_INVALID, "attention: a pointer is NULL");
    const size_t need = bytes_of(*d, 0);
    if (need && (!workspace || workspace_bytes < need)) return fail(WST_ERR_INVALID, "attention: workspace too small");
    AttnArgs a{};
    const AttnPlan p = plan_of(*d, can_tile(*d));
    if (!launchable(*d, p, false)) return fail(WST_ERR_UNSUPPORTED, "attention: too many rows for one launch");
    a.d = *d;
    a.o = o;
    a.lse = lse;
    a.splits = p.splits;
    a.part = static_cast<float*>(workspace);
    if (p.splits > 1) a.part_ml = a.part + static_cast<size_t>(p.splits) * rows_of(*d) * d->dim;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    with_type(d->dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        if (p.tiles) {
            with_width(d->dim, [&](auto w) { attend<T, decltype(w)::value>(a, p, st); });
        } else {
            k_attn_rows<T><<<dim3(static_cast<unsigned>((d->q_len + 3) / 4), d->q_heads, static_cast<unsigned>(d->batch)), dim3(256), 0, st>>>(a);
        }
    });
    return launched("attention");
}

int wst_attention_backward(const wst_attention_desc* d, const wst_attention_grads* g, void* workspace,
                           size_t workspace_bytes, void* stream) {
    if (const int e = check(d)) return e;
    if (!g) return fail(WST_ERR_INVALID, "attention: gradients' descriptor is NULL");
    if (rows_of(*d) == 0 || d->k_len == 0) return fail(WST_ERR_INVALID, "attention: no queries or keys, all gradients are zero");
    if (!d->q || !d->k || !d->v || !g->o || !g->d_o || !g->lse) return fail(WST_ERR_INVALID, "attention: a pointer is NULL");
    if (g->dslopes && !d->slopes) return fail(WST_ERR_INVALID, "attention: no slopes to have a gradient");
    if (!workspace || workspace_bytes < bytes_of(*d, 1)) return fail(WST_ERR_INVALID, "attention: workspace too small");
    AttnArgs a{};
    a.d = *d;
    a.g = *g;
    const AttnPlan p = plan_of(*d, can_tile(*d) && lined_up(*d, g->d_o, g->do_strides));
    if (!launchable(*d, p, true)) return fail(WST_ERR_UNSUPPORTED, "attention: too many rows for one launch");
    a.delta = static_cast<float*>(workspace);
    a.slots = p.slots;
    a.parts = p.parts;
    float* rest = a.delta + rows_of(*d);
    if (d->dtype == WST_F32) {
        a.unit = rest;
        rest += rows_of(*d);
    }
    if (d->slopes) {
        if (g->dslopes) a.slope_part = rest;
        rest += static_cast<size_t>(d->q_heads) * d->batch * p.slots;
    }
    a.part = rest;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    with_type(d->dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        if (p.tiles) {
            with_width(d->dim, [&](auto w) { attend_backward<T, decltype(w)::value>(a, p, st); });
            return;
        }
        launch_delta<T>(a, st);
        if (g->dq || g->dslopes || a.unit)
            k_attn_dq_rows<T><<<dim3(static_cast<unsigned>((d->q_len + 3) / 4), d->q_heads, static_cast<unsigned>(d->batch)), dim3(256), 0, st>>>(a);
        if (g->dk || g->dv)
            k_attn_dkv_rows<T><<<dim3(static_cast<unsigned>((d->k_len + 3) / 4), d->k_heads, static_cast<unsigned>(d->batch)), dim3(256), 0, st>>>(a);
    });
    const bool joined = p.tiles && p.parts > 1 && (g->dk || g->dv);
    if (g->dslopes && !joined) k_attn_slopes<<<dim3(d->q_heads), dim3(1024), 0, st>>>(a);
    return launched("attention backward");
}

}  // extern "C"
