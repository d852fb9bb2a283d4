// Attention on coefficient tokens, with scores capped by tanh, a bias that depends on distance, documents, order and a
// prefix (C ABI and formulas: include/wst_hip.h, "Token operators").
//
//   z = scale q.k;  z = cap tanh(z / cap);  s = z - slope * distance;  p = softmax(s over the keys seen);  o = p v
//   backward, with delta_i = sum_d do_id o_id:  dv = p^T do;  dp = do v^T;  ds = p (dp - delta);
//   dslope = -sum ds distance;  dz = ds (1 - (z / cap)^2) scale;  dq = dz k;  dk = dz^T q
#include <cmath>

#include "wst_tokens.h"

namespace {

using namespace wst_tok;

struct AttnArgs {
    wst_attention_desc d;
    wst_attention_grads g;
    void* o;
    float* lse;
    float* delta;        // (batch, heads, q_len)
    float* slope_part;   // (heads, batch, slots)
    int slots;
};

// What one batch entry's keys and queries may see.
struct Scope {
    int64_t length, shift, prefix;   // keys that exist; place(i) = i + shift; keys below prefix are seen out of order
    const int32_t *q_doc, *k_doc, *q_pos, *k_pos;
    bool causal;
    int axes;

    __device__ __forceinline__ Scope(const wst_attention_desc& d, int64_t b) {
        length = d.k_len;
        if (d.k_lengths) {
            const int64_t l = d.k_lengths[b];
            length = l < 0 ? 0 : l < length ? l : length;
        }
        shift = length - d.q_len;
        prefix = d.prefix ? d.prefix[b] : 0;
        causal = d.causal != 0;
        axes = d.axes;
        q_doc = d.q_doc ? d.q_doc + b * d.q_doc_stride : nullptr;
        k_doc = d.k_doc ? d.k_doc + b * d.k_doc_stride : nullptr;
        q_pos = d.q_pos ? d.q_pos + b * d.q_pos_stride : nullptr;
        k_pos = d.k_pos ? d.k_pos + b * d.k_pos_stride : nullptr;
    }
    __device__ __forceinline__ bool seen(int64_t i, int64_t j) const {
        if (j >= length) return false;
        if (causal && j > i + shift && j >= prefix) return false;
        if (q_doc) {
            const int32_t x = q_doc[i];
            return x >= 0 && x == k_doc[j];
        }
        return true;
    }
    __device__ __forceinline__ float distance(int64_t i, int64_t j) const {
        if (!q_pos) return static_cast<float>(i + shift > j ? i + shift - j : j - i - shift);
        float s = 0.f;
        for (int a = 0; a < axes; ++a) {
            const int64_t x = static_cast<int64_t>(q_pos[i * axes + a]) - k_pos[j * axes + a];
            s += static_cast<float>(x < 0 ? -x : x);
        }
        return s;
    }
};

constexpr int kD = WST_MAX_HEAD_DIM, kPer = kD / 64;   // values of a row a lane holds: d = lane + 64 c

template <typename T>
__device__ __forceinline__ const T* at(const void* p, const int64_t (&s)[3], int64_t b, int64_t t, int h) {
    return static_cast<const T*>(p) + b * s[0] + t * s[1] + h * s[2];
}

// dot of a row in LDS with a row in memory
template <typename T>
__device__ __forceinline__ float dot_row(const float* a, const T* b, int dim) {
    float s = 0.f;
    int d = 0;
    for (; d + 8 <= dim; d += 8) {
        float v[8];
        load<8>(b + d, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += a[d + e] * v[e];
    }
    for (; d < dim; ++d) s += a[d] * static_cast<float>(b[d]);
    return s;
}

// capped score before the bias, and the slope of the cap there
__device__ __forceinline__ float capped(float z, float cap, float& grad) {
    grad = 1.f;
    if (cap > 0.f) {
        const float t = tanhf(z / cap);
        grad = 1.f - t * t;
        z = cap * t;
    }
    return z;
}

// One query by one wave, a key a lane. q: the query's row in LDS (this wave's own).
template <typename T>
__device__ void row_forward(const AttnArgs& a, const Scope& sc, int64_t b, int h, int64_t i, float* q) {
    const wst_attention_desc& d = a.d;
    const int lane = threadIdx.x & 63, kvh = h / (d.q_heads / d.k_heads);
    const T* qr = at<T>(d.q, d.q_strides, b, i, h);
    for (int x = lane; x < d.dim; x += 64) q[x] = static_cast<float>(qr[x]);
    __builtin_amdgcn_wave_barrier();
    const float slope = d.slopes ? d.slopes[h] : 0.f;
    float m = -INFINITY, l = 0.f, acc[kPer] = {};
    for (int64_t j0 = 0; j0 < sc.length; j0 += 64) {
        const int64_t j = j0 + lane;
        const bool see = sc.seen(i, j);
        float s = -INFINITY, unused;
        if (see) {
            s = capped(dot_row(q, at<T>(d.k, d.k_strides, b, j, kvh), d.dim) * d.scale, d.cap, unused);
            if (d.slopes) s -= slope * sc.distance(i, j);
        }
        const uint64_t who = __ballot(see);
        if (!who) continue;
        const float mn = fmaxf(m, wave_max(s)), base = mn == -INFINITY ? 0.f : mn;
        const float p = see ? expf(s - base) : 0.f, f = expf(m - base);
        l = l * f + wave_sum(p);
        m = mn;
#pragma unroll
        for (int c = 0; c < kPer; ++c) acc[c] *= f;
        for (uint64_t w = who; w; w &= w - 1) {
            const int e = __builtin_ctzll(w);
            const float pe = __shfl(p, e);
            const T* v = at<T>(d.v, d.v_strides, b, j0 + e, kvh);
#pragma unroll
            for (int c = 0; c < kPer; ++c)
                if (lane + 64 * c < d.dim) acc[c] += pe * static_cast<float>(v[lane + 64 * c]);
        }
    }
    T* o = const_cast<T*>(at<T>(a.o, d.o_strides, b, i, h));
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < kPer; ++c)
        if (lane + 64 * c < d.dim) o[lane + 64 * c] = static_cast<T>(acc[c] * inv);
    if (lane == 0 && a.lse) a.lse[(b * d.q_heads + h) * d.q_len + i] = l == 0.f ? -INFINITY : m + logf(l);
}

// The gradient of one query, and its share of -sum ds distance. LDS: q and do of the row.
template <typename T>
__device__ float row_dq(const AttnArgs& a, const Scope& sc, int64_t b, int h, int64_t i, float* q, float* dout) {
    const wst_attention_desc& d = a.d;
    const int lane = threadIdx.x & 63, kvh = h / (d.q_heads / d.k_heads);
    const T *qr = at<T>(d.q, d.q_strides, b, i, h), *dr = at<T>(a.g.d_o, a.g.do_strides, b, i, h);
    for (int x = lane; x < d.dim; x += 64) {
        q[x] = static_cast<float>(qr[x]);
        dout[x] = static_cast<float>(dr[x]);
    }
    __builtin_amdgcn_wave_barrier();
    const float slope = d.slopes ? d.slopes[h] : 0.f;
    const int64_t row = (b * d.q_heads + h) * d.q_len + i;
    const float lse = a.g.lse[row], delta = a.delta[row];
    float acc[kPer] = {}, share = 0.f;
    if (lse != -INFINITY)
        for (int64_t j0 = 0; j0 < sc.length; j0 += 64) {
            const int64_t j = j0 + lane;
            const bool see = sc.seen(i, j);
            float dz = 0.f;
            if (see) {
                float grad;
                float s = capped(dot_row(q, at<T>(d.k, d.k_strides, b, j, kvh), d.dim) * d.scale, d.cap, grad);
                const float far = d.slopes ? sc.distance(i, j) : 0.f;
                s -= slope * far;
                const float ds = expf(s - lse) * (dot_row(dout, at<T>(d.v, d.v_strides, b, j, kvh), d.dim) - delta);
                share -= ds * far;
                dz = ds * grad * d.scale;
            }
            for (uint64_t w = __ballot(see); w; w &= w - 1) {
                const int e = __builtin_ctzll(w);
                const float x = __shfl(dz, e);
                const T* k = at<T>(d.k, d.k_strides, b, j0 + e, kvh);
#pragma unroll
                for (int c = 0; c < kPer; ++c)
                    if (lane + 64 * c < d.dim) acc[c] += x * static_cast<float>(k[lane + 64 * c]);
            }
        }
    if (a.g.dq) {
        T* o = const_cast<T*>(at<T>(a.g.dq, a.g.dq_strides, b, i, h));
#pragma unroll
        for (int c = 0; c < kPer; ++c)
            if (lane + 64 * c < d.dim) o[lane + 64 * c] = static_cast<T>(acc[c]);
    }
    return wave_sum(share);
}

// The gradients of one key and value, over all queries of the heads that share it. LDS: k and v of the row.
template <typename T>
__device__ void row_dkv(const AttnArgs& a, const Scope& sc, int64_t b, int kvh, int64_t j, float* k, float* v) {
    const wst_attention_desc& d = a.d;
    const int lane = threadIdx.x & 63, group = d.q_heads / d.k_heads;
    const T *kr = at<T>(d.k, d.k_strides, b, j, kvh), *vr = at<T>(d.v, d.v_strides, b, j, kvh);
    for (int x = lane; x < d.dim; x += 64) {
        k[x] = static_cast<float>(kr[x]);
        v[x] = static_cast<float>(vr[x]);
    }
    __builtin_amdgcn_wave_barrier();
    float dk[kPer] = {}, dv[kPer] = {};
    for (int h = kvh * group; h < (kvh + 1) * group; ++h) {
        const float slope = d.slopes ? d.slopes[h] : 0.f;
        for (int64_t i0 = 0; i0 < d.q_len; i0 += 64) {
            const int64_t i = i0 + lane;
            const int64_t row = (b * d.q_heads + h) * d.q_len + i;
            const bool see = i < d.q_len && sc.seen(i, j) && a.g.lse[row] != -INFINITY;
            float p = 0.f, dz = 0.f;
            if (see) {
                float grad;
                float s = capped(dot_row(k, at<T>(d.q, d.q_strides, b, i, h), d.dim) * d.scale, d.cap, grad);
                if (d.slopes) s -= slope * sc.distance(i, j);
                p = expf(s - a.g.lse[row]);
                dz = p * (dot_row(v, at<T>(a.g.d_o, a.g.do_strides, b, i, h), d.dim) - a.delta[row]) * grad * d.scale;
            }
            for (uint64_t w = __ballot(see); w; w &= w - 1) {
                const int e = __builtin_ctzll(w);
                const float pe = __shfl(p, e), ze = __shfl(dz, e);
                const T *q = at<T>(d.q, d.q_strides, b, i0 + e, h), *dr = at<T>(a.g.d_o, a.g.do_strides, b, i0 + e, h);
#pragma unroll
                for (int c = 0; c < kPer; ++c)
                    if (lane + 64 * c < d.dim) {
                        dk[c] += ze * static_cast<float>(q[lane + 64 * c]);
                        dv[c] += pe * static_cast<float>(dr[lane + 64 * c]);
                    }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < kPer; ++c)
        if (lane + 64 * c < d.dim) {
            if (a.g.dk) const_cast<T*>(at<T>(a.g.dk, a.g.dk_strides, b, j, kvh))[lane + 64 * c] = static_cast<T>(dk[c]);
            if (a.g.dv) const_cast<T*>(at<T>(a.g.dv, a.g.dv_strides, b, j, kvh))[lane + 64 * c] = static_cast<T>(dv[c]);
        }
}

template <typename T>
__global__ __launch_bounds__(256) void k_attn_rows(AttnArgs a) {
    __shared__ float q[4][kD];
    const int w = threadIdx.x >> 6, h = blockIdx.y;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + w, b = blockIdx.z;
    if (i >= a.d.q_len) return;
    row_forward<T>(a, Scope(a.d, b), b, h, i, q[w]);
}

// delta_i = sum_d do_id o_id, a wave a row
template <typename T>
__global__ __launch_bounds__(256) void k_attn_delta(AttnArgs a) {
    const wst_attention_desc& d = a.d;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6), b = blockIdx.z;
    const int h = blockIdx.y, lane = threadIdx.x & 63;
    if (i >= d.q_len) return;
    const T *o = at<T>(a.g.o, d.o_strides, b, i, h), *dr = at<T>(a.g.d_o, a.g.do_strides, b, i, h);
    float s = 0.f;
    for (int x = lane; x < d.dim; x += 64) s += static_cast<float>(o[x]) * static_cast<float>(dr[x]);
    s = wave_sum(s);
    if (lane == 0) a.delta[(b * d.q_heads + h) * d.q_len + i] = s;
}

template <typename T>
__global__ __launch_bounds__(256) void k_attn_dq_rows(AttnArgs a) {
    __shared__ float q[4][kD], dout[4][kD];
    const int w = threadIdx.x >> 6, h = blockIdx.y;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + w, b = blockIdx.z;
    if (i >= a.d.q_len) return;
    const float share = row_dq<T>(a, Scope(a.d, b), b, h, i, q[w], dout[w]);
    if (a.slope_part && (threadIdx.x & 63) == 0)
        a.slope_part[(static_cast<int64_t>(h) * a.d.batch + b) * a.slots + i] = share;
}

template <typename T>
__global__ __launch_bounds__(256) void k_attn_dkv_rows(AttnArgs a) {
    __shared__ float k[4][kD], v[4][kD];
    const int w = threadIdx.x >> 6;
    const int64_t j = static_cast<int64_t>(blockIdx.x) * 4 + w, b = blockIdx.z;
    if (j >= a.d.k_len) return;
    row_dkv<T>(a, Scope(a.d, b), b, blockIdx.y, j, k[w], v[w]);
}

// dslopes[h]: the partial sums of a head, added in a fixed order.
__global__ __launch_bounds__(1024) void k_attn_slopes(const float* part, int64_t count, float* out) {
    __shared__ float s[16];
    const float* p = part + static_cast<int64_t>(blockIdx.x) * count;
    float v = 0.f;
    for (int64_t i = threadIdx.x; i < count; i += 1024) v += p[i];
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 16; ++k) v += s[k];
        out[blockIdx.x] = v;
    }
}

template <typename T>
struct Tag {
    using type = T;
};
template <typename F>
int with_type(int dtype, F f) {
    if (dtype == WST_F32) return f(Tag<float>{});
    if (dtype == WST_BF16) return f(Tag<bf16>{});
    return f(Tag<f16>{});
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
    if (!(d->cap >= 0.f) || !std::isfinite(d->cap)) return fail(WST_ERR_INVALID, "attention: cap must be finite and not negative");
    if (!d->q_pos != !d->k_pos || !d->q_doc != !d->k_doc)
        return fail(WST_ERR_INVALID, "attention: positions and documents are given for queries and keys alike");
    if (d->q_pos && (d->axes < 1 || d->axes > WST_MAX_AXES)) return fail(WST_ERR_INVALID, "attention: 1 to %d axes", WST_MAX_AXES);
    if (d->prefix && !d->causal) return fail(WST_ERR_INVALID, "attention: a prefix needs causal order");
    if (d->batch > 65535 || d->q_heads > 65535) return fail(WST_ERR_UNSUPPORTED, "attention: more than 65535 sequences or heads");
    if (d->q_len > (1LL << 30) || d->k_len > (1LL << 30)) return fail(WST_ERR_UNSUPPORTED, "attention: more than 2^30 tokens");
    return WST_OK;
}

size_t rows_of(const wst_attention_desc& d) { return static_cast<size_t>(d.batch) * d.q_heads * d.q_len; }

size_t bytes_of(const wst_attention_desc& d, int backward) {
    if (!backward) return 0;
    return sizeof(float) * rows_of(d) * (d.slopes ? 2 : 1);
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
    a.d = *d;
    a.o = o;
    a.lse = lse;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    with_type(d->dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        k_attn_rows<T><<<dim3(static_cast<unsigned>((d->q_len + 3) / 4), d->q_heads, static_cast<unsigned>(d->batch)), dim3(256), 0, st>>>(a);
        return 0;
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
    a.delta = static_cast<float*>(workspace);
    if (g->dslopes) {
        a.slope_part = a.delta + rows_of(*d);
        a.slots = static_cast<int>(d->q_len);
    }
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    with_type(d->dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        const dim3 rows(static_cast<unsigned>((d->q_len + 3) / 4), d->q_heads, static_cast<unsigned>(d->batch));
        const dim3 keys(static_cast<unsigned>((d->k_len + 3) / 4), d->k_heads, static_cast<unsigned>(d->batch));
        k_attn_delta<T><<<rows, dim3(256), 0, st>>>(a);
        if (g->dq || g->dslopes) k_attn_dq_rows<T><<<rows, dim3(256), 0, st>>>(a);
        if (g->dk || g->dv) k_attn_dkv_rows<T><<<keys, dim3(256), 0, st>>>(a);
        return 0;
    });
    if (g->dslopes) k_attn_slopes<<<dim3(d->q_heads), dim3(1024), 0, st>>>(a.slope_part, d->batch * a.slots, g->dslopes);
    return launched("attention backward");
}

}  // extern "C"
