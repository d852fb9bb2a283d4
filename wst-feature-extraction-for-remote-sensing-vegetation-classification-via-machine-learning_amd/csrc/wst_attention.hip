// Attention on coefficient tokens, with scores capped by tanh, a bias that depends on distance, documents, order and a
// prefix (C ABI and formulas: include/wst_hip.h, "Token operators").
//
//   z = scale q.k;  z = cap tanh(z / cap);  s = z - slope * distance;  p = softmax(s over the keys seen);  o = p v
//   backward, with delta_i = sum_d do_id o_id:  dv = p^T do;  dp = do v^T;  ds = p (dp - delta);
//   dslope = -sum ds distance;  dz = ds (1 - (z / cap)^2) scale;  dq = dz k;  dk = dz^T q
#include <cmath>
#include <type_traits>

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
    float *part, *part_ml;   // forward: (splits, rows, dim) and (splits, rows, 2); backward: (parts, keys, 2, dim)
    int slots, splits, parts;
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

// ------------------------------------------------------------------------------------------ matrix instructions
// Heads of a multiple of 8 values up to 128 go through 32x32 matrix instructions, padded to DP = 32, 64, 96 or 128.
//
// Operand layout (16-bit: 32x32x16, eight values a lane; float32: 32x32x2, one value a lane): with h = lane / 32, an
// operand fragment holds, of row or column lane % 32, the eight inner indices 8 h .. 8 h + 7 of a step of 16. For float32
// the eight values feed eight instructions, one each; which inner index meets which instruction does not matter as long
// as both operands agree. The result holds column lane % 32 and rows 8 (r / 4) + 4 h + r % 4 for r = 0 .. 15.
//
// So a tile of scores taken as (keys x queries) has one query a lane: the softmax's maximum and sum are in-lane but for
// one exchange between the halves, and its sixteen registers are, rounded, the next product's operand for the keys
// 16 s + 8 (e / 4) + 4 h + e % 4 (step s, element e): the other operand reads the same keys in that order, so no score
// ever moves between lanes.
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
    typedef bf16 Frag __attribute__((ext_vector_type(8)));
    typedef bf16 Quad __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x16 mul(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<f16> {
    typedef f16 Frag __attribute__((ext_vector_type(8)));
    typedef f16 Quad __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x16 mul(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<float> {
    typedef float Frag __attribute__((ext_vector_type(8)));
    typedef float Quad __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x16 mul(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};
template <typename T>
using Frag = typename Mma<T>::Frag;
template <typename T>
using Quad = typename Mma<T>::Quad;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
#define WST_LDS __attribute__((address_space(3)))

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}

// max / sum with the lane 32 away
__device__ __forceinline__ float halves_max(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Rows of DP values in LDS, in units of 16 bytes. Unit u of a row lies at u ^ swizzle(row): reading 16 rows at one unit
// (row_frag) and 4 rows at 4 units (col_frag) both then touch every bank once. The swizzle depends on row % 16 alone, so
// a lane's is the same for all its rows.
template <typename T, int DP>
struct Tile {
    static constexpr int kElems = 16 / sizeof(T), kUnits = DP / kElems, kRowBytes = DP * sizeof(T);
    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (kUnits % 16 == 0) return ((row & 3) << 2) | ((row >> 2) & 3);        // a row spans all banks
        else if constexpr (kUnits % 8 == 0) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);   // two rows do
        else return (row >> 2) & 3;                                                        // four rows do
    }
    static __device__ __forceinline__ int at(int row, int unit) { return row * kRowBytes + ((unit ^ swizzle(row)) << 4); }

    // row row0 + lane % 32, values 16 c + 8 (lane / 32) .. + 7; row0 a multiple of 16
    static __device__ __forceinline__ Frag<T> row_frag(const char* t, int row0, int c) {
        const int lane = threadIdx.x & 63, row = lane & 31, h = lane >> 5;
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            f = *reinterpret_cast<const Frag<T>*>(t + row0 * kRowBytes + at(row, 2 * c + h));
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4*>(t + row0 * kRowBytes + at(row, 4 * c + 2 * h));
            const f32x4 b = *reinterpret_cast<const f32x4*>(t + row0 * kRowBytes + at(row, 4 * c + 2 * h + 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[e] = a[e];
                f[4 + e] = b[e];
            }
        }
        return f;
    }
    // value 32 db + lane % 32 of the eight rows row0 + 8 (e / 4) + 4 (lane / 32) + e % 4; row0 a multiple of 16
    static __device__ __forceinline__ Frag<T> col_frag(const char* t, int row0, int db) {
        const int lane = threadIdx.x & 63;
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            // the transposing read: sixteen lanes hand in four rows of sixteen values and get a column of four each
            const int g = lane >> 4, x = lane & 15, row = 4 * (g >> 1) + (x >> 2), unit = 4 * db + 2 * (g & 1) + ((x & 3) >> 1);
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            union {
                s16x4 q[2];
                Frag<T> f;
            } u;
#pragma unroll
            for (int k = 0; k < 2; ++k)
                u.q[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (WST_LDS s16x4*)(t + row0 * kRowBytes + at(8 * k + row, unit) + 8 * (x & 1)));
            f = u.f;
        } else {
            const int d = 32 * db + (lane & 31), h = lane >> 5;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                f[e] = *reinterpret_cast<const float*>(t + row0 * kRowBytes + at(8 * (e >> 2) + 4 * h + (e & 3), d >> 2) + 4 * (d & 3));
        }
        return f;
    }
};

// N rows of a tensor on their way to LDS: loaded into registers early, stored when the tile is free. A thread of TH takes
// units t, t + TH, ...; rows that do not exist or belong to no document, and values beyond the head, become zero.
template <typename T, int DP, int N, int TH>
struct Stage {
    using L = Tile<T, DP>;
    static constexpr int kCount = (N * L::kUnits + TH - 1) / TH;
    u32x4 v[kCount];

    __device__ __forceinline__ void load(const T* base, int64_t stride, int64_t row0, int64_t rows, const int32_t* doc, int dim, int t) {
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int id = t + i * TH, row = id / L::kUnits, unit = id % L::kUnits;
            bool ok = (N * L::kUnits % TH == 0 || row < N) && row0 + row < rows && unit * L::kElems < dim;
            if (doc) ok = ok && doc[row0 + (row0 + row < rows ? row : 0)] >= 0;
            v[i] = u32x4{0, 0, 0, 0};
            if (ok) __builtin_memcpy(&v[i], base + (row0 + row) * stride + unit * L::kElems, 16);
        }
    }
    __device__ __forceinline__ void store(char* tile, int t) const {
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int id = t + i * TH, row = id / L::kUnits, unit = id % L::kUnits;
            if (N * L::kUnits % TH == 0 || row < N) *reinterpret_cast<u32x4*>(tile + L::at(row, unit)) = v[i];
        }
    }
};

// N rows of a tensor straight into LDS, past the registers: each lane names the 16 bytes it wants, the sixteen-byte units
// of a wave land one after the other. Swizzling is done by choosing the source. What does not exist, or belongs to no
// document, is fetched from a line of zeros. The compiler does not know of these loads: arrived() waits for them.
__device__ const u32x4 g_zero = {0, 0, 0, 0};

template <typename T, int DP, int N, int TH>
struct Fetch {
    using L = Tile<T, DP>;
    static_assert(N * L::kUnits % TH == 0, "whole waves");
    static __device__ __forceinline__ void issue(const T* base, int64_t stride, int64_t row0, int64_t rows, const int32_t* doc, int dim,
                                                 const char* tile, int t) {
        const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((WST_LDS const char*)tile)) + (t & ~63) * 16;
#pragma unroll
        for (int i = 0; i < N * L::kUnits / TH; ++i) {
            const int id = t + i * TH, row = id / L::kUnits, unit = (id % L::kUnits) ^ L::swizzle(row);
            bool ok = row0 + row < rows && unit * L::kElems < dim;
            if (doc) ok = ok && doc[row0 + row < rows ? row0 + row : row0] >= 0;
            const void* src = ok ? static_cast<const void*>(base + (row0 + row) * stride + unit * L::kElems) : static_cast<const void*>(&g_zero);
            const uint32_t dst = __builtin_amdgcn_readfirstlane(lds + i * TH * 16);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(dst), "v"(src) : "memory", "m0");
        }
    }
};
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }

// Eight values of a row as an operand fragment, from memory; zero beyond the head or where the row is not to be read.
template <typename T, int DP>
__device__ __forceinline__ void row_frags(const T* row, bool ok, int dim, Frag<T> (&f)[DP / 16]) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
        if (ok && 16 * c + 8 * h < dim) {
            __builtin_memcpy(&f[c], row + 16 * c + 8 * h, sizeof(Frag<T>));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[c][e] = static_cast<T>(0.f);
        }
    }
}

// Sixteen result registers as the operands of two steps of the next product, rounded to the inputs' type: the products
// of weights are the one place where attention rounds before its end.
template <typename T>
__device__ __forceinline__ void to_frags(const f32x16& s, Frag<T> (&f)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) f[k][e] = static_cast<T>(s[8 * k + e]);
}

template <typename T>
__device__ __forceinline__ void store_quad(T* p, const float (&v)[4]) {
    store<4>(p, v);
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Scores in powers of two. The cap: tanh(x) = 1 - 2 / (e^2x + 1), whose error of 2^-24 or two of the cap is below what
// 16-bit weights keep; float32 takes the library's tanh, good to an ulp of the result.
struct Shape {
    float lin, cap2, twice;   // scale log2 e;  cap log2 e;  2 scale log2 e / cap
    float turn;               // scale / cap
    bool cap;
    __device__ __forceinline__ Shape(const wst_attention_desc& d) {
        cap = d.cap > 0.f;
        lin = d.scale * kLog2e;
        cap2 = d.cap * kLog2e;
        twice = cap ? 2.f * d.scale * kLog2e / d.cap : 0.f;
        turn = cap ? d.scale / d.cap : 0.f;
    }
    template <typename T>
    __device__ __forceinline__ float tanh_of(float dot) const {
        if constexpr (sizeof(T) == 4) return tanhf(dot * turn);
        else return 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(dot * twice) + 1.f);
    }
};

// What a lane's query (forward, dq) needs: the first key it may not see in order, its document and coordinates.
struct Query {
    int limit, doc;
    float place;
    uint32_t pos[WST_MAX_AXES];
};
constexpr uint32_t kPosBias = 0x40000000u;   // coordinates in +-2^29 as unsigned numbers

__device__ __forceinline__ Query query_of(const Scope& sc, int64_t i, bool ok) {
    Query q;
    q.limit = static_cast<int>(sc.length);
    if (sc.causal) {
        const int64_t place = i + sc.shift + 1, e = place > sc.prefix ? place : sc.prefix;
        q.limit = static_cast<int>(e < 0 ? 0 : e < sc.length ? e : sc.length);
    }
    if (!ok) q.limit = 0;
    q.doc = -1;
    if (sc.q_doc && ok) q.doc = sc.q_doc[i];
    if (sc.q_doc && q.doc < 0) q.limit = 0;
    q.place = static_cast<float>(i + sc.shift);
#pragma unroll
    for (int a = 0; a < WST_MAX_AXES; ++a)
        q.pos[a] = sc.q_pos && a < sc.axes && ok ? static_cast<uint32_t>(sc.q_pos[i * sc.axes + a]) + kPosBias : 0u;
    return q;
}

__device__ __forceinline__ uint32_t away(uint32_t a, uint32_t b, uint32_t sum) { return (a > b ? a - b : b - a) + sum; }

// Which 64-key (or 64-query) tiles a block has to visit. With documents: those where some token's document lies in the
// block's own range; and whether a tile's tokens all belong to the one document that all of the block's own do, so that
// no pair needs a look. Up to kWords * 64 tiles are marked, tiles beyond are visited.
constexpr int kWords = 64;
struct Marks {
    uint64_t any[kWords], full[kWords];
    int lo[4], hi[4], all;
};

// Range of the documents of `count` tokens from t0 on (valid ones), by the first wave's lanes and then to all.
__device__ __forceinline__ void scan_documents(Marks& m, const int32_t* own, int64_t own0, int own_count, int64_t own_rows,
                                               const int32_t* other, int64_t tile0, int64_t tile1, int64_t other_rows) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int lo = INT32_MAX, hi = -1;
    bool all = true;
    for (int x = lane; x < own_count && own0 + x < own_rows; x += 64) {
        const int v = own[own0 + x];
        all = all && v >= 0;
        if (v >= 0) {
            lo = v < lo ? v : lo;
            hi = v > hi ? v : hi;
        }
    }
#pragma unroll
    for (int k = 32; k; k >>= 1) {
        const int a = __shfl_xor(lo, k), b = __shfl_xor(hi, k);
        lo = a < lo ? a : lo;
        hi = b > hi ? b : hi;
    }
    const bool one = __all(all) && lo == hi;
    for (int64_t word = w; word < kWords && tile0 + word * 64 < tile1; word += blockDim.x >> 6) {
        uint64_t any = 0, full = 0;
        for (int k = 0; k < 64 && tile0 + word * 64 + k < tile1; ++k) {
            const int64_t j = (tile0 + word * 64 + k) * 64 + lane;
            const int v = j < other_rows ? other[j] : -1;
            if (__ballot(v >= lo && v <= hi)) any |= 1ull << k;
            if (one && __ballot(v == lo) == ~0ull) full |= 1ull << k;
        }
        if (lane == 0) {
            m.any[word] = any;
            m.full[word] = full;
        }
    }
}

// The next tile to visit after `t` (tiles tile0 .. tile1 - 1), tile1 when there is none.
__device__ __forceinline__ int64_t next_tile(const Marks& m, bool marked, int64_t t, int64_t tile0, int64_t tile1) {
    ++t;
    if (!marked) return t;
    while (t < tile1) {
        const int64_t k = t - tile0;
        if (k >= kWords * 64) return t;
        const uint64_t w = m.any[k >> 6] >> (k & 63);
        // uniform: the word comes from LDS, the same for all lanes
        const uint64_t u = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(w >> 32))) << 32 |
                           static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(w)));
        if (u) return t + __builtin_ctzll(u) < tile1 ? t + __builtin_ctzll(u) : tile1;
        t += 64 - (k & 63);
    }
    return tile1;
}
__device__ __forceinline__ bool full_tile(const Marks& m, int64_t k) {
    return k < kWords * 64 && __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(m.full[k >> 6] >> (k & 63)) & 1u);
}

// Columns (of a key tile) that go along with it in LDS: coordinates and documents, ready to compare.
struct Along {
    uint32_t pos[WST_MAX_AXES][64];
    int doc[64];
};

// Turns 32 x 32 dot products (rows: keys, column: the lane's query) into scores; `key0` is the tile's first key, sub
// the block of 32 within it. GRAD also keeps the cap's slope (1 - tanh^2) and the distances.
template <typename T, bool GRAD>
__device__ __forceinline__ void scores(f32x16& s, const Shape& sh, float slope2, bool bias, const Scope& sc, const Query& q,
                                       const Along& al, int64_t key0, int sub, bool masked, f32x16& grad, f32x16& far) {
    const int h = (threadIdx.x & 63) >> 5;
    if (sh.cap) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float t = sh.tanh_of<T>(s[r]);
            if constexpr (GRAD) grad[r] = 1.f - t * t;
            s[r] = sh.cap2 * t;
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= sh.lin;
    }
    if (bias) {
        if (sc.q_pos) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                uint32_t sum[4] = {0, 0, 0, 0};
                for (int a = 0; a < sc.axes; ++a) {
                    const u32x4 k = *reinterpret_cast<const u32x4*>(&al.pos[a][32 * sub + 8 * g + 4 * h]);
                    const uint32_t x = a == 0 ? q.pos[0] : a == 1 ? q.pos[1] : a == 2 ? q.pos[2] : q.pos[3];
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] = away(x, k[e], sum[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float f = static_cast<float>(sum[e]);
                    if constexpr (GRAD) far[4 * g + e] = f;
                    s[4 * g + e] -= slope2 * f;
                }
            }
        } else {
            const float base = q.place - static_cast<float>(key0 + 32 * sub + 4 * h);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float f = fabsf(base - static_cast<float>(8 * (r >> 2) + (r & 3)));
                if constexpr (GRAD) far[r] = f;
                s[r] -= slope2 * f;
            }
        }
    }
    if (masked) {
        const int64_t rel64 = static_cast<int64_t>(q.limit) - key0 - 32 * sub - 4 * h;
        const int rel = static_cast<int>(rel64 > 64 ? 64 : rel64 < 0 ? 0 : rel64);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (sc.q_doc) {
                const i32x4 k = *reinterpret_cast<const i32x4*>(&al.doc[32 * sub + 8 * g + 4 * h]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * g + e] = 8 * g + e < rel && k[e] == q.doc ? s[4 * g + e] : -INFINITY;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * g + e] = 8 * g + e < rel ? s[4 * g + e] : -INFINITY;
            }
        }
    }
}

// Loads what goes along with a key tile: thread t < 256 one coordinate, t < 64 one document.
struct AlongStage {
    uint32_t pos;
    int doc;
    __device__ __forceinline__ void load(const int32_t* p, const int32_t* d, int axes, int64_t row0, int64_t rows, int t) {
        const int64_t row = row0 + (t & 63);
        const bool ok = row < rows;
        pos = p && (t >> 6) < axes && ok ? static_cast<uint32_t>(p[row * axes + (t >> 6)]) + kPosBias : 0u;
        doc = d && t < 64 && ok ? d[row] : -2;    // -2 matches nobody; a key without a document holds a negative number,
        if (doc < 0) doc = -2;                    // and queries without one see nothing anyway
    }
    __device__ __forceinline__ void store(Along& al, int t) const {
        al.pos[t >> 6][t & 63] = pos;
        if (t < 64) al.doc[t] = doc;
    }
};

template <typename T, int DP>
__device__ __forceinline__ bool not_finite(const f32x16 (&o)[DP / 32]) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < DP / 32; ++k)
#pragma unroll
        for (int r = 0; r < 16; ++r) t = fmaf(o[k][r], 0.f, t);
    return t != t;
}

constexpr int kBQ = 128, kBK = 64;

// Forward pass: a block takes 128 queries of a head, 32 a wave, and walks the key tiles that any of them may see,
// keeping the running maximum, sum and output of the softmax in registers; keys and values of a tile are shared through
// LDS, the next tile on its way in registers meanwhile.
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void k_attn_fwd(AttnArgs a) {
    using L = Tile<T, DP>;
    __shared__ __attribute__((aligned(256))) char kt[2][kBK * L::kRowBytes], vt[2][kBK * L::kRowBytes];
    __shared__ Along al[2];
    __shared__ Marks marks;
    __shared__ float scratch[4][DP];
    const wst_attention_desc& d = a.d;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, hl = lane >> 5;
    const uint32_t cells = static_cast<uint32_t>(d.batch) * d.q_heads, bh = blockIdx.x % cells;
    const int64_t nq = (d.q_len + kBQ - 1) / kBQ, qt = nq - 1 - blockIdx.x / cells;   // long rows first
    const int64_t b = bh / d.q_heads;
    const int h = static_cast<int>(bh % d.q_heads), kvh = h / (d.q_heads / d.k_heads);
    const Scope sc(d, b);
    const Shape sh(d);
    const int64_t i0 = qt * kBQ, i = i0 + w * 32 + (lane & 31);
    const bool ok = i < d.q_len;
    const Query q = query_of(sc, i, ok);
    const float slope2 = d.slopes ? d.slopes[h] * kLog2e : 0.f;
    Frag<T> qf[DP / 16];
    row_frags<T, DP>(at<T>(d.q, d.q_strides, b, ok ? i : 0, h), ok && q.limit > 0, d.dim, qf);

    // keys below `end` may be seen by some query of the block, keys below `open` by all of its queries in order
    const int64_t last = (i0 + kBQ < d.q_len ? i0 + kBQ : d.q_len) - 1;
    int64_t end = sc.length, open = sc.length;
    if (sc.causal) {
        end = last + sc.shift + 1 > sc.prefix ? last + sc.shift + 1 : sc.prefix;
        open = i0 + sc.shift + 1 > sc.prefix ? i0 + sc.shift + 1 : sc.prefix;
        end = end < sc.length ? end : sc.length;
        open = open < sc.length ? open : sc.length;
    }
    const int64_t tiles = end > 0 ? (end + kBK - 1) / kBK : 0;
    const bool marked = sc.q_doc != nullptr;
    if (marked) {
        scan_documents(marks, sc.q_doc, i0, kBQ, d.q_len, sc.k_doc, 0, tiles, sc.length);
        __syncthreads();
    }
    f32x16 o[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) o[k] = zero16();
    float m = -INFINITY, l = 0.f;

    const T *kb = at<T>(d.k, d.k_strides, b, 0, kvh), *vb = at<T>(d.v, d.v_strides, b, 0, kvh);
    AlongStage as;
    auto fetch = [&](int64_t n, int buf) {
        Fetch<T, DP, kBK, 256>::issue(kb, d.k_strides[1], n * kBK, sc.length, sc.k_doc, d.dim, kt[buf], t);
        Fetch<T, DP, kBK, 256>::issue(vb, d.v_strides[1], n * kBK, sc.length, sc.k_doc, d.dim, vt[buf], t);
        as.load(sc.k_pos, sc.k_doc, sc.axes, n * kBK, sc.length, t);
    };
    int64_t tile = next_tile(marks, marked, -1, 0, tiles);
    int buf = 0;
    if (tile < tiles) {
        fetch(tile, 0);
        as.store(al[0], t);
    }
    while (tile < tiles) {
        const int64_t key0 = tile * kBK, next = next_tile(marks, marked, tile, 0, tiles);
        arrived();
        __syncthreads();                          // the tile is there, and nobody reads the other buffer any more
        if (next < tiles) fetch(next, buf ^ 1);
        const bool masked = key0 + kBK > open || (marked && !full_tile(marks, tile));
        const char *kc = kt[buf], *vc = vt[buf];
        f32x16 s[2], unused;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n] = zero16();
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) s[n] = Mma<T>::mul(L::row_frag(kc, 32 * n, c), qf[c], s[n]);
        }
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            scores<T, false>(s[n], sh, slope2, d.slopes != nullptr, sc, q, al[buf], key0, n, masked, unused, unused);
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[n][r]);
        }
        const float mn = fmaxf(m, halves_max(top));
        const float base = fmaxf(mn, -3.0e38f);        // nothing seen yet: exp2(-inf) = 0 either way
        if (__ballot(mn > m)) {
            const float f = __builtin_amdgcn_exp2f(m - base);
            l *= f;
#pragma unroll
            for (int k = 0; k < DP / 32; ++k)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[k][r] *= f;
        }
        m = mn;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[n][r] = __builtin_amdgcn_exp2f(s[n][r] - base);
                l += s[n][r];
            }
            Frag<T> p[2];
            to_frags<T>(s[n], p);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) o[db] = Mma<T>::mul(L::col_frag(vc, 32 * n + 16 * k, db), p[k], o[db]);
        }
        if (next < tiles) as.store(al[buf ^ 1], t);
        tile = next;
        buf ^= 1;
    }
    l = halves_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = const_cast<T*>(at<T>(a.o, d.o_strides, b, ok ? i : 0, h));
    if (ok) {
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int x = 32 * db + 8 * g + 4 * hl;
                const float v[4] = {o[db][4 * g] * inv, o[db][4 * g + 1] * inv, o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv};
                if (x < d.dim) store_quad(out + x, v);
            }
        if (hl == 0 && a.lse) a.lse[(b * d.q_heads + h) * d.q_len + i] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
    }
    // A value that is not finite, of a key that some query of the wave does not see, has reached that query as 0 * inf:
    // the queries whose output is not finite are done over, key by key. In ordinary data there are none.
    uint64_t bad = __ballot(ok && not_finite<T, DP>(o));
    for (bad = (bad | bad >> 32) & 0xffffffffu; bad; bad &= bad - 1)
        row_forward<T>(a, sc, b, h, i0 + w * 32 + __builtin_ctzll(bad), scratch[w]);
}

// Few queries over many keys: the queries of all heads that share a key head make up to 32 rows, and the keys are split
// over blocks, and in a block over its waves, each of which walks its own tiles of 32 keys through its own part of LDS
// with nothing to wait for. The parts are joined by their maxima and sums, in the block and then by k_attn_join.
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void k_attn_split(AttnArgs a) {
    using L = Tile<T, DP>;
    constexpr int kTile = 32 * L::kRowBytes, kLd = DP + 4;
    constexpr int kBytes = 8 * kTile > 32 * kLd * 4 ? 8 * kTile : 32 * kLd * 4;
    __shared__ __attribute__((aligned(256))) char pool[kBytes];
    __shared__ Along al[2];          // a wave's 32 keys in half of one
    __shared__ Marks marks;
    __shared__ float wm[4][32], wl[4][32];
    __shared__ float scratch[4][DP];
    const wst_attention_desc& d = a.d;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, hl = lane >> 5;
    const int group = d.q_heads / d.k_heads;
    const int64_t rows = group * d.q_len;
    // blocks: splits, then tiles of rows, then key heads, then sequences
    const uint32_t split = blockIdx.x % a.splits, cell = blockIdx.x / a.splits, row_tiles = static_cast<uint32_t>((rows + 31) / 32);
    const int64_t b = cell / row_tiles / d.k_heads;
    const int kvh = static_cast<int>(cell / row_tiles % d.k_heads);
    const int64_t r0 = static_cast<int64_t>(cell % row_tiles) * 32, r = r0 + (lane & 31);
    const bool ok = r < rows;
    const int64_t i = ok ? r % d.q_len : 0;
    const int h = kvh * group + static_cast<int>(ok ? r / d.q_len : 0);
    const Scope sc(d, b);
    const Shape sh(d);
    const Query q = query_of(sc, i, ok);
    const float slope2 = d.slopes ? d.slopes[h] * kLog2e : 0.f;
    Frag<T> qf[DP / 16];
    row_frags<T, DP>(at<T>(d.q, d.q_strides, b, i, h), ok && q.limit > 0, d.dim, qf);

    int64_t end = sc.length;
    if (sc.causal) {
        end = d.q_len + sc.shift > sc.prefix ? d.q_len + sc.shift : sc.prefix;
        end = end < sc.length ? end : sc.length;
    }
    // this split's keys, in whole groups of 128: a wave has 32 of each
    const int64_t groups = end > 0 ? (end + 127) / 128 : 0, per = (groups + a.splits - 1) / a.splits;
    const int64_t g0 = split * per < groups ? split * per : groups, g1 = g0 + per < groups ? g0 + per : groups;
    const bool marked = sc.q_doc != nullptr;
    if (marked) {
        scan_documents(marks, sc.q_doc, 0, static_cast<int>(d.q_len < 1024 ? d.q_len : 1024), d.q_len, sc.k_doc, 2 * g0, 2 * g1, sc.length);
        __syncthreads();
    }
    const bool skip = marked && d.q_len <= 1024;   // else the marks do not speak for all queries
    auto wanted = [&](int64_t g) {                  // the next group of 128 in whose 64 keys this wave has work
        for (; g < g1; ++g) {
            const int64_t k = 2 * (g - g0) + (w >> 1);
            if (!skip || k >= kWords * 64) return g;
            if (__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(marks.any[k >> 6] >> (k & 63)) & 1u)) return g;
        }
        return g1;
    };
    f32x16 o[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) o[k] = zero16();
    float m = -INFINITY, l = 0.f;
    const T *kb = at<T>(d.k, d.k_strides, b, 0, kvh), *vb = at<T>(d.v, d.v_strides, b, 0, kvh);
    char *kt = pool + 2 * w * kTile, *vt = kt + kTile;
    Stage<T, DP, 32, 64> ks, vs;
    uint32_t pos[WST_MAX_AXES];
    int doc = -2;
    auto fetch = [&](int64_t key0) {
        ks.load(kb, d.k_strides[1], key0, sc.length, sc.k_doc, d.dim, lane);
        vs.load(vb, d.v_strides[1], key0, sc.length, sc.k_doc, d.dim, lane);
        const int64_t j = key0 + (lane & 31);
        if (sc.k_pos)
#pragma unroll
            for (int x = 0; x < WST_MAX_AXES; ++x)
                pos[x] = x < sc.axes && j < sc.length ? static_cast<uint32_t>(sc.k_pos[j * sc.axes + x]) + kPosBias : 0u;
        if (sc.k_doc) {
            doc = j < sc.length ? sc.k_doc[j] : -2;
            if (doc < 0) doc = -2;
        }
    };
    Along& mine = al[w >> 1];
    const int sub = w & 1;
    int64_t g = wanted(g0);
    if (g < g1) fetch(g * 128 + 32 * w);
    while (g < g1) {
        const int64_t key0 = g * 128 + 32 * w;
        __builtin_amdgcn_wave_barrier();
        ks.store(kt, lane);
        vs.store(vt, lane);
        if (lane < 32) {
            if (sc.k_pos)
#pragma unroll
                for (int x = 0; x < WST_MAX_AXES; ++x) mine.pos[x][32 * sub + lane] = pos[x];
            mine.doc[32 * sub + lane] = doc;
        }
        __builtin_amdgcn_wave_barrier();
        const int64_t next = wanted(g + 1);
        if (next < g1) fetch(next * 128 + 32 * w);
        f32x16 s = zero16(), unused;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) s = Mma<T>::mul(L::row_frag(kt, 0, c), qf[c], s);
        scores<T, false>(s, sh, slope2, d.slopes != nullptr, sc, q, mine, key0 - 32 * sub, sub, true, unused, unused);
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < 16; ++x) top = fmaxf(top, s[x]);
        const float mn = fmaxf(m, halves_max(top)), base = fmaxf(mn, -3.0e38f);
        if (__ballot(mn > m)) {
            const float f = __builtin_amdgcn_exp2f(m - base);
            l *= f;
#pragma unroll
            for (int k = 0; k < DP / 32; ++k)
#pragma unroll
                for (int x = 0; x < 16; ++x) o[k][x] *= f;
        }
        m = mn;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            s[x] = __builtin_amdgcn_exp2f(s[x] - base);
            l += s[x];
        }
        Frag<T> p[2];
        to_frags<T>(s, p);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) o[db] = Mma<T>::mul(L::col_frag(vt, 16 * k, db), p[k], o[db]);
        g = next;
    }
    // join the waves
    l = halves_sum(l);
    if (hl == 0) {
        wm[w][lane] = m;
        wl[w][lane] = l;
    }
    __syncthreads();               // and every wave is done with its tiles
    const int x = lane & 31;
    const float mm = fmaxf(fmaxf(wm[0][x], wm[1][x]), fmaxf(wm[2][x], wm[3][x])), base = fmaxf(mm, -3.0e38f);
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) total += wl[k][x] * __builtin_amdgcn_exp2f(wm[k][x] - base);
    const float f = __builtin_amdgcn_exp2f(m - base);
    float* sum = reinterpret_cast<float*>(pool);
    for (int turn = 0; turn < 4; ++turn) {
        if (turn == w) {
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f32x4* c = reinterpret_cast<f32x4*>(sum + x * kLd + 32 * db + 8 * e + 4 * hl);
                    f32x4 v = turn ? *c : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int y = 0; y < 4; ++y) v[y] += o[db][4 * e + y] * f;
                    *c = v;
                }
        }
        __syncthreads();
    }
    // a wave writes eight rows
    for (int y = w * 8; y < w * 8 + 8 && r0 + y < rows; ++y) {
        const int64_t ii = (r0 + y) % d.q_len;
        const int hh = kvh * group + static_cast<int>((r0 + y) / d.q_len);
        const int64_t row = (b * d.q_heads + hh) * d.q_len + ii;
        const float my = __shfl(mm, y), ly = __shfl(total, y);
        if (a.splits > 1) {
            const int64_t all = d.batch * d.q_heads * d.q_len, slot = split * all + row;
            for (int e = lane; e < d.dim; e += 64) a.part[slot * d.dim + e] = sum[y * kLd + e];
            if (lane == 0) {
                a.part_ml[2 * slot] = my;
                a.part_ml[2 * slot + 1] = ly;
            }
        } else {
            const float inv = ly == 0.f ? 0.f : 1.f / ly;
            T* out = const_cast<T*>(at<T>(a.o, d.o_strides, b, ii, hh));
            bool bad = false;
            for (int e = lane; e < d.dim; e += 64) {
                const float v = sum[y * kLd + e] * inv;
                bad = bad || !(fabsf(v) < INFINITY);
                out[e] = static_cast<T>(v);
            }
            if (lane == 0 && a.lse) a.lse[row] = ly == 0.f ? -INFINITY : my * kLn2 + logf(ly);
            if (__ballot(bad)) row_forward<T>(a, sc, b, hh, ii, scratch[w]);   // see k_attn_fwd
        }
    }
}

// Joins the splits of a row, a wave a row.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a) {
    __shared__ float scratch[4][kD];
    const wst_attention_desc& d = a.d;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t all = d.batch * d.q_heads * d.q_len, row = static_cast<int64_t>(blockIdx.x) * 4 + w;
    if (row >= all) return;
    const int64_t i = row % d.q_len, bh = row / d.q_len, b = bh / d.q_heads;
    const int h = static_cast<int>(bh % d.q_heads);
    float m = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.part_ml[2 * (s * all + row)]);
    m = wave_max(m);
    const float base = fmaxf(m, -3.0e38f);
    float l = 0.f, v[2] = {0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
        const int64_t slot = s * all + row;
        const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * slot] - base);
        l += f * a.part_ml[2 * slot + 1];
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (lane + 64 * e < d.dim) v[e] += f * a.part[slot * d.dim + lane + 64 * e];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = const_cast<T*>(at<T>(a.o, d.o_strides, b, i, h));
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < d.dim) {
            bad = bad || !(fabsf(v[e] * inv) < INFINITY);
            out[lane + 64 * e] = static_cast<T>(v[e] * inv);
        }
    if (lane == 0 && a.lse) a.lse[row] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
    if (__ballot(bad)) row_forward<T>(a, Scope(d, b), b, h, i, scratch[w]);
}

// Float16 loses small numbers before large ones: weights and score gradients are held 2^6 times as large there, so that
// they keep their precision down to 2^-20; a score gradient beyond 2^10 then overflows, and its row is done over in
// float32 like any that is not finite.
template <typename T>
constexpr float kUp = 1.f;
template <>
constexpr float kUp<f16> = 64.f;

// dq, the slopes' shares and delta: walks the keys as the forward pass does. Scores come back as (keys x queries), so
// their gradient is the operand of dq^T = k^T dz^T as it stands; keys are read from LDS both ways.
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void k_attn_dq(AttnArgs a) {
    using L = Tile<T, DP>;
    __shared__ __attribute__((aligned(256))) char kt[2][kBK * L::kRowBytes], vt[2][kBK * L::kRowBytes];
    __shared__ Along al[2];
    __shared__ Marks marks;
    __shared__ float scratch[4][2][DP];
    const wst_attention_desc& d = a.d;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, hl = lane >> 5;
    const uint32_t cells = static_cast<uint32_t>(d.batch) * d.q_heads, bh = blockIdx.x % cells;
    const int64_t nq = (d.q_len + kBQ - 1) / kBQ, qt = nq - 1 - blockIdx.x / cells;
    const int64_t b = bh / d.q_heads;
    const int h = static_cast<int>(bh % d.q_heads), kvh = h / (d.q_heads / d.k_heads);
    const Scope sc(d, b);
    const Shape sh(d);
    const int64_t i0 = qt * kBQ, i = i0 + w * 32 + (lane & 31), row = (b * d.q_heads + h) * d.q_len + i;
    const bool ok = i < d.q_len;
    const Query q = query_of(sc, i, ok);
    const float slope2 = d.slopes ? d.slopes[h] * kLog2e : 0.f;
    const float lse = ok ? a.g.lse[row] : -INFINITY;
    const bool live = ok && q.limit > 0 && lse != -INFINITY;
    const float lse2 = live ? lse * kLog2e : INFINITY;         // of a query that sees nothing every weight is 0
    Frag<T> qf[DP / 16], df[DP / 16];
    float delta = 0.f;
    {
        Frag<T> of[DP / 16];
        row_frags<T, DP>(at<T>(a.g.d_o, a.g.do_strides, b, ok ? i : 0, h), live, d.dim, df);
        row_frags<T, DP>(at<T>(a.g.o, d.o_strides, b, ok ? i : 0, h), live, d.dim, of);
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta += static_cast<float>(df[c][e]) * static_cast<float>(of[c][e]);
        delta = halves_sum(delta);
        if (ok && hl == 0) a.delta[row] = delta;
    }
    row_frags<T, DP>(at<T>(d.q, d.q_strides, b, ok ? i : 0, h), live, d.dim, qf);

    const int64_t last = (i0 + kBQ < d.q_len ? i0 + kBQ : d.q_len) - 1;
    int64_t end = sc.length, open = sc.length;
    if (sc.causal) {
        end = last + sc.shift + 1 > sc.prefix ? last + sc.shift + 1 : sc.prefix;
        open = i0 + sc.shift + 1 > sc.prefix ? i0 + sc.shift + 1 : sc.prefix;
        end = end < sc.length ? end : sc.length;
        open = open < sc.length ? open : sc.length;
    }
    const int64_t tiles = end > 0 ? (end + kBK - 1) / kBK : 0;
    const bool marked = sc.q_doc != nullptr;
    if (marked) {
        scan_documents(marks, sc.q_doc, i0, kBQ, d.q_len, sc.k_doc, 0, tiles, sc.length);
        __syncthreads();
    }
    f32x16 dq[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) dq[k] = zero16();
    // -sum ds far = -(sum p dp far - (sum p dp) (sum p far)): from delta as the row itself gives it, in 32 bits, since
    // delta out of the rounded output would be multiplied by a mean distance
    float pdf = 0.f, pd = 0.f, pf = 0.f;

    const T *kb = at<T>(d.k, d.k_strides, b, 0, kvh), *vb = at<T>(d.v, d.v_strides, b, 0, kvh);
    AlongStage as;
    auto fetch = [&](int64_t n, int buf) {
        Fetch<T, DP, kBK, 256>::issue(kb, d.k_strides[1], n * kBK, sc.length, sc.k_doc, d.dim, kt[buf], t);
        Fetch<T, DP, kBK, 256>::issue(vb, d.v_strides[1], n * kBK, sc.length, sc.k_doc, d.dim, vt[buf], t);
        as.load(sc.k_pos, sc.k_doc, sc.axes, n * kBK, sc.length, t);
    };
    int64_t tile = next_tile(marks, marked, -1, 0, tiles);
    int buf = 0;
    if (tile < tiles) {
        fetch(tile, 0);
        as.store(al[0], t);
    }
    while (tile < tiles) {
        const int64_t key0 = tile * kBK, next = next_tile(marks, marked, tile, 0, tiles);
        arrived();
        __syncthreads();
        if (next < tiles) fetch(next, buf ^ 1);
        const bool masked = key0 + kBK > open || (marked && !full_tile(marks, tile));
        const char *kc = kt[buf], *vc = vt[buf];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            f32x16 s = zero16(), dp = zero16(), grad, far;
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) s = Mma<T>::mul(L::row_frag(kc, 32 * n, c), qf[c], s);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) dp = Mma<T>::mul(L::row_frag(vc, 32 * n, c), df[c], dp);
            scores<T, true>(s, sh, slope2, d.slopes != nullptr, sc, q, al[buf], key0, n, masked, grad, far);
            if (masked) {     // a weight of 0 may meet a value that is not finite
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] = s[r] == -INFINITY ? 0.f : dp[r];
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - lse2);
            if (a.slope_part) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    pf += s[r] * far[r];
                    pd += s[r] * dp[r];
                    pdf += s[r] * dp[r] * far[r];
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] = s[r] * (dp[r] - delta);
            if (sh.cap) {
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] *= grad[r];
            }
            if constexpr (kUp<T> != 1.f) {
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] *= kUp<T>;
            }
            Frag<T> z[2];
            to_frags<T>(dp, z);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) dq[db] = Mma<T>::mul(L::col_frag(kc, 32 * n + 16 * k, db), z[k], dq[db]);
        }
        if (next < tiles) as.store(al[buf ^ 1], t);
        tile = next;
        buf ^= 1;
    }
    const float mul = d.scale / kUp<T>;
    if (ok && a.g.dq) {
        T* out = const_cast<T*>(at<T>(a.g.dq, a.g.dq_strides, b, i, h));
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int x = 32 * db + 8 * g + 4 * hl;
                const float v[4] = {dq[db][4 * g] * mul, dq[db][4 * g + 1] * mul, dq[db][4 * g + 2] * mul, dq[db][4 * g + 3] * mul};
                if (x < d.dim) store_quad(out + x, v);
            }
    }
    if (a.slope_part) {
        const float share = halves_sum(pd) * halves_sum(pf) - halves_sum(pdf), sum = wave_sum(hl ? 0.f : share);
        if (lane == 0) a.slope_part[(static_cast<int64_t>(h) * d.batch + b) * a.slots + qt * 4 + w] = sum;
    }
    uint64_t bad = __ballot(ok && not_finite<T, DP>(dq));      // see k_attn_fwd
    for (bad = (bad | bad >> 32) & 0xffffffffu; bad; bad &= bad - 1) {
        __builtin_amdgcn_wave_barrier();
        row_dq<T>(a, sc, b, h, i0 + w * 32 + __builtin_ctzll(bad), scratch[w][0], scratch[w][1]);
    }
}

// What goes along with a tile of 64 queries.
struct Rows {
    float lse2[64], delta[64], place[64];
    int limit[64], doc[64];
    uint32_t pos[WST_MAX_AXES][64];
};

// dk and dv: a block takes 128 keys of a key head, 32 a wave, held as operands in registers, and walks tiles of 64
// queries of the heads that share it. Scores come as (queries x keys), one key a lane, so weights and score gradients
// are the operands of dv^T = do^T p and dk^T = q^T dz as they stand. With few key tiles the walk is split in parts whose
// sums k_attn_dkv_join adds in order.
template <typename T, int DP>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && DP <= 64) ? 2 : 1) void k_attn_dkv(AttnArgs a) {
    using L = Tile<T, DP>;
    constexpr int kRows = 64;
    __shared__ __attribute__((aligned(256))) char qt[2][kRows * L::kRowBytes], dt[2][kRows * L::kRowBytes];
    __shared__ Rows rows[2];
    __shared__ Marks marks;
    __shared__ float scratch[4][2][DP];
    const wst_attention_desc& d = a.d;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, hl = lane >> 5, group = d.q_heads / d.k_heads;
    const uint32_t cells = static_cast<uint32_t>(d.batch) * d.k_heads, bh = blockIdx.x % cells, part = blockIdx.y;
    const int64_t kt = blockIdx.x / cells, b = bh / d.k_heads;   // early keys are seen by most: first
    const int kvh = static_cast<int>(bh % d.k_heads);
    const Scope sc(d, b);
    const Shape sh(d);
    const int64_t j0 = kt * kBQ, j = j0 + w * 32 + (lane & 31);
    const bool exists = j < d.k_len, ok = j < sc.length && (!sc.k_doc || sc.k_doc[j] >= 0);
    const int kdoc = ok && sc.k_doc ? sc.k_doc[j] : -2;
    uint32_t kpos[WST_MAX_AXES];
#pragma unroll
    for (int x = 0; x < WST_MAX_AXES; ++x)
        kpos[x] = ok && sc.k_pos && x < sc.axes ? static_cast<uint32_t>(sc.k_pos[j * sc.axes + x]) + kPosBias : 0u;
    Frag<T> kf[DP / 16], vf[DP / 16];
    row_frags<T, DP>(at<T>(d.k, d.k_strides, b, ok ? j : 0, kvh), ok, d.dim, kf);
    row_frags<T, DP>(at<T>(d.v, d.v_strides, b, ok ? j : 0, kvh), ok, d.dim, vf);
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) dk[k] = dv[k] = zero16();

    // queries from `first` on may see one of the block's keys; keys past the length are seen by none
    const int64_t nqt = (d.q_len + kRows - 1) / kRows, keys = sc.length - j0 < kBQ ? sc.length - j0 : kBQ;
    int64_t first = 0;
    if (sc.causal && j0 >= sc.prefix) first = j0 - sc.shift > 0 ? j0 - sc.shift : 0;
    const int64_t tile0 = first / kRows, tiles = keys > 0 ? nqt : 0;
    const bool marked = sc.q_doc != nullptr;
    if (marked && tile0 < tiles) {
        scan_documents(marks, sc.k_doc, j0, kBQ, sc.length, sc.q_doc, tile0, tiles, d.q_len);
        __syncthreads();
    }
    float r_lse = 0.f, r_delta = 0.f, r_place = 0.f;
    int r_limit = 0, r_doc = -1;
    uint32_t r_pos = 0;
    int g = 0;
    auto fetch = [&](int64_t tile, int buf) {
        const int h = kvh * group + g;
        Fetch<T, DP, kRows, 256>::issue(at<T>(d.q, d.q_strides, b, 0, h), d.q_strides[1], tile * kRows, d.q_len, sc.q_doc, d.dim, qt[buf], t);
        Fetch<T, DP, kRows, 256>::issue(at<T>(a.g.d_o, a.g.do_strides, b, 0, h), a.g.do_strides[1], tile * kRows, d.q_len, sc.q_doc, d.dim, dt[buf], t);
        const int64_t i = tile * kRows + (t & 63), row = (b * d.q_heads + h) * d.q_len + i;
        const bool in = i < d.q_len;
        if (t < 64) {
            const Query q = query_of(sc, i, in);
            const float lse = in ? a.g.lse[row] : -INFINITY;
            r_lse = lse == -INFINITY || q.limit == 0 ? INFINITY : lse * kLog2e;
            r_delta = in ? a.delta[row] : 0.f;
            r_limit = q.limit;
            r_doc = q.doc;
            r_place = q.place;
        }
        r_pos = sc.q_pos && (t >> 6) < sc.axes && in ? static_cast<uint32_t>(sc.q_pos[i * sc.axes + (t >> 6)]) + kPosBias : 0u;
    };
    // items: the visited tiles of head 0, then of head 1, ...; this part takes every a.parts-th
    int64_t tile = tile0 - 1;
    auto step = [&]() {
        tile = next_tile(marks, marked, tile, tile0, tiles);
        while (tile >= tiles && g + 1 < group) {
            ++g;
            tile = next_tile(marks, marked, tile0 - 1, tile0, tiles);
            if (tile >= tiles) g = group;    // nothing to visit in any head
        }
    };
    auto skip = [&](int n) {
        for (int k = 0; k < n && tile < tiles; ++k) step();
    };
    if (tile0 < tiles) {
        step();
        skip(part);
    } else {
        tile = tiles;
    }
    auto put = [&](Rows& rw) {
        if (t < 64) {
            rw.lse2[t] = r_lse;
            rw.delta[t] = r_delta;
            rw.limit[t] = r_limit;
            rw.doc[t] = r_doc;
            rw.place[t] = r_place;
        }
        rw.pos[t >> 6][t & 63] = r_pos;
    };
    int buf = 0;
    if (tile < tiles) {
        fetch(tile, 0);
        put(rows[0]);
    }
    while (tile < tiles) {
        const int64_t row0 = tile * kRows;
        const float slope2 = d.slopes ? d.slopes[kvh * group + g] * kLog2e : 0.f;
        const Rows& rw = rows[buf];
        const char *qc = qt[buf], *dc = dt[buf];
        arrived();
        __syncthreads();
        // in order for every pair: the tile's first query sees the block's last key, and all rows and keys exist
        bool masked = row0 + kRows > d.q_len || keys < kBQ || (marked && !full_tile(marks, tile - tile0));
        if (sc.causal) {
            const int64_t place = row0 + sc.shift + 1, lim = place > sc.prefix ? place : sc.prefix;
            masked = masked || lim < j0 + kBQ;
        }
        skip(a.parts);
        if (tile < tiles) fetch(tile, buf ^ 1);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            f32x16 s = zero16(), dp = zero16(), grad;
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) s = Mma<T>::mul(L::row_frag(qc, 32 * n, c), kf[c], s);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) dp = Mma<T>::mul(L::row_frag(dc, 32 * n, c), vf[c], dp);
            if (sh.cap) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float x = sh.tanh_of<T>(s[r]);
                    grad[r] = 1.f - x * x;
                    s[r] = sh.cap2 * x;
                }
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= sh.lin;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int y = 32 * n + 8 * c + 4 * hl;
                if (d.slopes) {
                    if (sc.q_pos) {
                        uint32_t sum[4] = {0, 0, 0, 0};
                        for (int x = 0; x < sc.axes; ++x) {
                            const u32x4 v = *reinterpret_cast<const u32x4*>(&rw.pos[x][y]);
                            const uint32_t mine = x == 0 ? kpos[0] : x == 1 ? kpos[1] : x == 2 ? kpos[2] : kpos[3];
#pragma unroll
                            for (int e = 0; e < 4; ++e) sum[e] = away(mine, v[e], sum[e]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * c + e] -= slope2 * static_cast<float>(sum[e]);
                    } else {
                        const f32x4 v = *reinterpret_cast<const f32x4*>(&rw.place[y]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * c + e] -= slope2 * fabsf(v[e] - static_cast<float>(j));
                    }
                }
                const f32x4 lse2 = *reinterpret_cast<const f32x4*>(&rw.lse2[y]), delta = *reinterpret_cast<const f32x4*>(&rw.delta[y]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(s[4 * c + e] - lse2[e]);
                    dp[4 * c + e] = p * (dp[4 * c + e] - delta[e]);
                    s[4 * c + e] = p;
                }
                if (masked) {
                    const i32x4 lim = *reinterpret_cast<const i32x4*>(&rw.limit[y]), doc = *reinterpret_cast<const i32x4*>(&rw.doc[y]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool see = j < lim[e] && (!sc.q_doc || kdoc == doc[e]);
                        s[4 * c + e] = see ? s[4 * c + e] : 0.f;
                        dp[4 * c + e] = see ? dp[4 * c + e] : 0.f;
                    }
                }
            }
            if (sh.cap) {
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] *= grad[r];
            }
            if constexpr (kUp<T> != 1.f) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] *= kUp<T>;
                    dp[r] *= kUp<T>;
                }
            }
            Frag<T> p[2], z[2];
            to_frags<T>(s, p);
            to_frags<T>(dp, z);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) {
                    dv[db] = Mma<T>::mul(L::col_frag(dc, 32 * n + 16 * k, db), p[k], dv[db]);
                    dk[db] = Mma<T>::mul(L::col_frag(qc, 32 * n + 16 * k, db), z[k], dk[db]);
                }
        }
        if (tile < tiles) put(rows[buf ^ 1]);
        buf ^= 1;
    }
    const float up = 1.f / kUp<T>, mul = d.scale * up;
    if (a.parts > 1) {
        if (exists) {
            const int64_t row = ((static_cast<int64_t>(part) * d.batch + b) * d.k_heads + kvh) * d.k_len + j;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int x = 32 * db + 8 * g4 + 4 * hl;
                    if (x < d.dim) {
                        float u[4], v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            u[e] = dk[db][4 * g4 + e] * mul;
                            v[e] = dv[db][4 * g4 + e] * up;
                        }
                        store<4>(a.part + (2 * row) * d.dim + x, u);
                        store<4>(a.part + (2 * row + 1) * d.dim + x, v);
                    }
                }
        }
        return;
    }
    if (exists) {
        T* ok_ = a.g.dk ? const_cast<T*>(at<T>(a.g.dk, a.g.dk_strides, b, j, kvh)) : nullptr;
        T* ov = a.g.dv ? const_cast<T*>(at<T>(a.g.dv, a.g.dv_strides, b, j, kvh)) : nullptr;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int x = 32 * db + 8 * g4 + 4 * hl;
                if (x < d.dim) {
                    float u[4], v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        u[e] = dk[db][4 * g4 + e] * mul;
                        v[e] = dv[db][4 * g4 + e] * up;
                    }
                    if (ok_) store_quad(ok_ + x, u);
                    if (ov) store_quad(ov + x, v);
                }
            }
    }
    uint64_t bad = __ballot(exists && (not_finite<T, DP>(dk) || not_finite<T, DP>(dv)));      // see k_attn_fwd
    for (bad = (bad | bad >> 32) & 0xffffffffu; bad; bad &= bad - 1) {
        __builtin_amdgcn_wave_barrier();
        row_dkv<T>(a, sc, b, kvh, j0 + w * 32 + __builtin_ctzll(bad), scratch[w][0], scratch[w][1]);
    }
}

// Adds the parts of a key's gradients, a wave a key.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dkv_join(AttnArgs a) {
    __shared__ float scratch[4][2][kD];
    const wst_attention_desc& d = a.d;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t j = static_cast<int64_t>(blockIdx.x) * 4 + w, b = blockIdx.z;
    const int kvh = blockIdx.y;
    if (j >= d.k_len) return;
    float v[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
    for (int p = 0; p < a.parts; ++p) {
        const float* s = a.part + 2 * (((p * d.batch + b) * d.k_heads + kvh) * d.k_len + j) * d.dim;
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (lane + 64 * e < d.dim) {
                v[0][e] += s[lane + 64 * e];
                v[1][e] += s[d.dim + lane + 64 * e];
            }
    }
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < d.dim) {
            bad = bad || !(fabsf(v[0][e]) < INFINITY) || !(fabsf(v[1][e]) < INFINITY);
            if (a.g.dk) const_cast<T*>(at<T>(a.g.dk, a.g.dk_strides, b, j, kvh))[lane + 64 * e] = static_cast<T>(v[0][e]);
            if (a.g.dv) const_cast<T*>(at<T>(a.g.dv, a.g.dv_strides, b, j, kvh))[lane + 64 * e] = static_cast<T>(v[1][e]);
        }
    if (__ballot(bad)) row_dkv<T>(a, Scope(d, b), b, kvh, j, scratch[w][0], scratch[w][1]);
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
    // blocks of every kernel are counted in 31 bits: a tile or row of each has at most eight splits or so in flight
    if (static_cast<double>(d->batch) * d->q_heads * (static_cast<double>(d->q_len) / 4 + static_cast<double>(d->k_len) / 4 + 512) > 2147483647.0)
        return fail(WST_ERR_UNSUPPORTED, "attention: too many rows for one call");
    if (d->q_len > (1LL << 30) || d->k_len > (1LL << 30)) return fail(WST_ERR_UNSUPPORTED, "attention: more than 2^30 tokens");
    return WST_OK;
}

size_t rows_of(const wst_attention_desc& d) { return static_cast<size_t>(d.batch) * d.q_heads * d.q_len; }

// How a call runs.
struct Plan {
    bool tiles;                 // matrix instructions; else a row at a time (heads of other widths, rows not lined up to 16 bytes)
    int splits;                 // forward: 0 = k_attn_fwd, else blocks along the keys of k_attn_split
    int parts, slots;           // backward: parts of dk and dv; partial slope sums of a head and sequence
    size_t forward, backward;   // workspace, in floats
};

// Rows that can be fetched 16 bytes at a time.
bool lined_up(const wst_attention_desc& d, const void* p, const int64_t (&s)[3]) {
    const int64_t size = d.dtype == WST_F32 ? 4 : 2;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] * size % 16 == 0 && s[1] * size % 16 == 0 && s[2] * size % 16 == 0;
}

bool can_tile(const wst_attention_desc& d) {
    return d.dim % 8 == 0 && d.dim <= 128 && lined_up(d, d.q, d.q_strides) && lined_up(d, d.k, d.k_strides) && lined_up(d, d.v, d.v_strides);
}

Plan plan_of(const wst_attention_desc& d, bool tiles) {
    Plan p{};
    p.tiles = tiles;
    const int64_t rows = static_cast<int64_t>(rows_of(d)), group = d.q_heads / d.k_heads;
    p.slots = static_cast<int>(d.q_len);
    p.parts = 1;
    if (p.tiles && rows) {
        const int64_t blocks = d.batch * d.q_heads * ((d.q_len + kBQ - 1) / kBQ);
        const int64_t row_tiles = (group * d.q_len + 31) / 32, cells = d.batch * d.k_heads * row_tiles;
        if (d.q_len <= 32 || (blocks < 128 && d.k_len >= 1024)) {
            int64_t s = (1024 + cells - 1) / cells, most = (d.k_len + 255) / 256;
            s = s < most ? s : most;
            p.splits = static_cast<int>(s < 1 ? 1 : s > 256 ? 256 : s);
            if (p.splits > 1) p.forward = static_cast<size_t>(p.splits) * rows * (d.dim + 2);
        }
        const int64_t items = group * ((d.q_len + 63) / 64), keys = d.batch * d.k_heads * ((d.k_len + kBQ - 1) / kBQ);
        int64_t parts = keys ? (512 + keys - 1) / keys : 1;
        parts = parts < items / 2 ? parts : items / 2;
        p.parts = static_cast<int>(parts < 1 ? 1 : parts > 64 ? 64 : parts);
        p.slots = static_cast<int>((d.q_len + kBQ - 1) / kBQ * 4);
        if (p.parts > 1) p.backward = static_cast<size_t>(p.parts) * d.batch * d.k_heads * d.k_len * 2 * d.dim;
    }
    p.backward += rows;
    if (d.slopes) p.backward += static_cast<size_t>(d.q_heads) * d.batch * p.slots;
    return p;
}

size_t bytes_of(const wst_attention_desc& d, int backward) {
    // either way of running: the gradient of the output, which decides with the rest, is not known here
    const Plan p = plan_of(d, true), q = plan_of(d, false);
    const size_t b = p.backward > q.backward ? p.backward : q.backward;
    return sizeof(float) * (backward ? b : p.forward);
}

template <typename F>
void with_width(int dim, F f) {
    if (dim <= 32) f(std::integral_constant<int, 32>{});
    else if (dim <= 64) f(std::integral_constant<int, 64>{});
    else if (dim <= 96) f(std::integral_constant<int, 96>{});
    else f(std::integral_constant<int, 128>{});
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
    const Plan p = plan_of(*d, can_tile(*d));
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
            with_width(d->dim, [&](auto w) {
                constexpr int DP = decltype(w)::value;
                if (p.splits) {
                    const int64_t row_tiles = (d->q_heads / d->k_heads * d->q_len + 31) / 32;
                    k_attn_split<T, DP><<<dim3(static_cast<unsigned>(p.splits * row_tiles * d->batch * d->k_heads)), dim3(256), 0, st>>>(a);
                } else {
                    const int64_t blocks = d->batch * d->q_heads * ((d->q_len + kBQ - 1) / kBQ);
                    k_attn_fwd<T, DP><<<dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st>>>(a);
                }
            });
            if (p.splits > 1) k_attn_join<T><<<dim3(static_cast<unsigned>((rows_of(*d) + 3) / 4)), dim3(256), 0, st>>>(a);
            return 0;
        }
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
    const Plan p = plan_of(*d, can_tile(*d) && lined_up(*d, g->d_o, g->do_strides));
    a.delta = static_cast<float*>(workspace);
    a.slots = p.slots;
    a.parts = p.parts;
    float* rest = a.delta + rows_of(*d);
    if (d->slopes) {
        if (g->dslopes) a.slope_part = rest;
        rest += static_cast<size_t>(d->q_heads) * d->batch * p.slots;
    }
    a.part = rest;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    with_type(d->dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        const dim3 rows(static_cast<unsigned>((d->q_len + 3) / 4), d->q_heads, static_cast<unsigned>(d->batch));
        const dim3 keys(static_cast<unsigned>((d->k_len + 3) / 4), d->k_heads, static_cast<unsigned>(d->batch));
        if (p.tiles) {
            if (!g->dq && !g->dslopes) k_attn_delta<T><<<rows, dim3(256), 0, st>>>(a);
            with_width(d->dim, [&](auto w) {
                constexpr int DP = decltype(w)::value;
                const int64_t q_blocks = d->batch * d->q_heads * ((d->q_len + kBQ - 1) / kBQ);
                const int64_t k_blocks = d->batch * d->k_heads * ((d->k_len + kBQ - 1) / kBQ);
                if (g->dq || g->dslopes) k_attn_dq<T, DP><<<dim3(static_cast<unsigned>(q_blocks)), dim3(256), 0, st>>>(a);   // and delta
                if (g->dk || g->dv) k_attn_dkv<T, DP><<<dim3(static_cast<unsigned>(k_blocks), p.parts), dim3(256), 0, st>>>(a);
            });
            if (p.parts > 1 && (g->dk || g->dv)) k_attn_dkv_join<T><<<keys, dim3(256), 0, st>>>(a);
            return 0;
        }
        k_attn_delta<T><<<rows, dim3(256), 0, st>>>(a);
        if (g->dq || g->dslopes) k_attn_dq_rows<T><<<rows, dim3(256), 0, st>>>(a);
        if (g->dk || g->dv) k_attn_dkv_rows<T><<<keys, dim3(256), 0, st>>>(a);
        return 0;
    });
    if (g->dslopes) k_attn_slopes<<<dim3(d->q_heads), dim3(1024), 0, st>>>(a.slope_part, d->batch * a.slots, g->dslopes);
    return launched("attention backward");
}

}  // extern "C"
