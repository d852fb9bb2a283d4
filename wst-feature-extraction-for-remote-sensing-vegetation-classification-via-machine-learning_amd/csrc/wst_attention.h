// Attention on coefficient tokens, with scores capped by tanh, a bias that depends on distance, documents, order and a
// prefix (C ABI and formulas: include/wst_hip.h, "Token operators").
//
//   z = scale q.k;  z = cap tanh(z / cap);  s = z - slope * distance;  p = softmax(s over the keys seen);  o = p v
//   backward, with delta_i = sum_d do_id o_id:  dv = p^T do;  dp = do v^T;  ds = p (dp - delta);
//   dslope = -sum ds distance;  dz = ds (1 - (z / cap)^2) scale;  dq = dz k;  dk = dz^T q
//
// Kernels as templates over the element type; wst_attention_t.hip instantiates one type, wst_attention.hip checks the
// arguments and chooses.
#ifndef WST_ATTENTION_H
#define WST_ATTENTION_H

#include <cfloat>
#include <type_traits>

#include "wst_tokens.h"

namespace wst_tok {

// How a call runs.
struct AttnPlan {
    bool tiles;                 // matrix instructions; else a row at a time (other widths, rows not lined up to 16 bytes)
    int splits;                 // forward: 0 = k_attn_fwd, else blocks along the keys of k_attn_split
    int parts, slots;           // backward: parts of dk and dv; partial slope sums of a head and sequence
    size_t forward, backward;   // workspace, in floats
};

struct AttnArgs {
    wst_attention_desc d;
    wst_attention_grads g;
    void* o;
    float* lse;
    float* delta;        // (batch, heads, q_len)
    float* unit;         // float32: (batch, heads, q_len), 1 / the sum of the weights that the backward pass rebuilds; else null
    float* slope_part;   // (heads, batch, slots)
    float *part, *part_ml;   // forward: (splits, rows, dim) and (splits, rows, 2); backward: (parts, keys, 2, dim)
    int slots, splits, parts;
};

// What one batch entry's keys and queries may see.
struct Scope {
    int length, shift, prefix;   // keys that exist; place(i) = i + shift; keys below prefix are seen out of order
    const int32_t *q_doc, *k_doc, *q_pos, *k_pos;
    bool causal;
    int axes;

    __device__ __forceinline__ Scope(const wst_attention_desc& d, int64_t b) {
        length = static_cast<int>(d.k_len);
        if (d.k_lengths) {
            const int l = d.k_lengths[b];
            length = l < 0 ? 0 : l < length ? l : length;
        }
        shift = length - static_cast<int>(d.q_len);
        prefix = d.prefix ? d.prefix[b] : 0;
        prefix = prefix < 0 ? 0 : prefix < length ? prefix : length;
        causal = d.causal != 0;
        axes = d.axes;
        q_doc = d.q_doc ? d.q_doc + b * d.q_doc_stride : nullptr;
        k_doc = d.k_doc ? d.k_doc + b * d.k_doc_stride : nullptr;
        q_pos = d.q_pos ? d.q_pos + b * d.q_pos_stride : nullptr;
        k_pos = d.k_pos ? d.k_pos + b * d.k_pos_stride : nullptr;
    }
    __device__ __forceinline__ bool seen(int i, int j) const {
        if (j >= length) return false;
        if (causal && j > i + shift && j >= prefix) return false;
        if (q_doc) {
            const int32_t x = q_doc[i];
            return x >= 0 && x == k_doc[j];
        }
        return true;
    }
    // first key that query i does not see in order
    __device__ __forceinline__ int limit(int i) const {
        if (!causal) return length;
        const int e = i + shift + 1 > prefix ? i + shift + 1 : prefix;
        return e < length ? e : length;
    }
    __device__ __forceinline__ float distance(int i, int j) const {
        if (!q_pos) return static_cast<float>(i + shift > j ? i + shift - j : j - i - shift);
        float s = 0.f;
        for (int a = 0; a < axes; ++a) {
            const int64_t x = static_cast<int64_t>(q_pos[static_cast<int64_t>(i) * axes + a]) - k_pos[static_cast<int64_t>(j) * axes + a];
            s += static_cast<float>(x < 0 ? -x : x);
        }
        return s;
    }
};

constexpr int kAxes = WST_MAX_DISTANCE_AXES;
constexpr int kD = WST_MAX_HEAD_DIM, kPer = kD / 64;   // values of a row a lane holds: d = lane + 64 c

template <typename T>
__device__ __forceinline__ const T* at(const void* p, const int64_t (&s)[3], int64_t b, int64_t t, int h) {
    return static_cast<const T*>(p) + b * s[0] + t * s[1] + h * s[2];
}

// What rounding v to T takes from it. The backward pass has it from the forward pass (o_rest): delta = sum do o taken
// from the rounded output alone is off by its rounding, which a row with few large weights meets as a whole, since there
// all of its do.v_j lie close to delta.
template <typename T>
__device__ __forceinline__ T lost(float v) {
    return static_cast<T>(v - static_cast<float>(static_cast<T>(v)));
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
__device__ void row_forward(const AttnArgs& a, const Scope& sc, int64_t b, int h, int i, float* q) {
    const wst_attention_desc& d = a.d;
    const int lane = threadIdx.x & 63, kvh = h / (d.q_heads / d.k_heads);
    const T* qr = at<T>(d.q, d.q_strides, b, i, h);
    for (int x = lane; x < d.dim; x += 64) q[x] = static_cast<float>(qr[x]);
    __builtin_amdgcn_wave_barrier();
    const float slope = d.slopes ? d.slopes[h] : 0.f;
    float m = -INFINITY, l = 0.f, acc[kPer] = {};
    for (int j0 = 0; j0 < sc.length; j0 += 64) {
        const int j = j0 + lane;
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
        if (lane + 64 * c < d.dim) {
            o[lane + 64 * c] = static_cast<T>(acc[c] * inv);
            if (d.o_rest) static_cast<T*>(d.o_rest)[o - static_cast<T*>(a.o) + lane + 64 * c] = lost<T>(acc[c] * inv);
        }
    if (lane == 0 && a.lse) a.lse[(b * d.q_heads + h) * d.q_len + i] = l == 0.f ? -INFINITY : m + logf(l);
}

// What makes a row's rebuilt weights add up to 1. They come as exp(s - lse), and lse is a float32 number: its rounding is
// half an ulp of the largest score, the same for all weights of the row (and in powers of two once more). 16-bit weights lose
// more when they are rounded, and only the slopes' gradients take it there; float32 gradients are the nearer to the exact ones so (256 keys: dq 3.9e-7 for 5.0e-7, dk 3.2
// for 4.5, dv 3.0 for 4.5; 16 x 256, 4 heads x 32: dk/dv 23.5 us for 22.6, dq no slower), most of all where scores stand far
// from 0 (at 1e5 a log-sum-exp of float32 is off by 4e-3).
__device__ __forceinline__ float unit_of(float sum) { return sum > 0.f && sum < INFINITY ? 1.f / sum : 1.f; }

// The gradient of one query, and its share of -sum ds distance. LDS: q and do of the row.
template <typename T>
__device__ float row_dq(const AttnArgs& a, const Scope& sc, int64_t b, int h, int i, float* q, float* dout) {
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
    float acc[kPer] = {}, sum = 0.f, pf = 0.f, e0 = 0.f, e1 = 0.f;      // as in k_attn_dq
    if (lse != -INFINITY)
        for (int j0 = 0; j0 < sc.length; j0 += 64) {
            const int j = j0 + lane;
            const bool see = sc.seen(i, j);
            float dz = 0.f;
            if (see) {
                float grad;
                float s = capped(dot_row(q, at<T>(d.k, d.k_strides, b, j, kvh), d.dim) * d.scale, d.cap, grad);
                const float far = d.slopes ? sc.distance(i, j) : 0.f;
                s -= slope * far;
                const float p = expf(s - lse);
                sum += p;
                const float ds = p * (dot_row(dout, at<T>(d.v, d.v_strides, b, j, kvh), d.dim) - delta);
                pf += p * far;
                e0 += ds;
                e1 += ds * far;
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
    const float unit = unit_of(wave_sum(sum));
    if (a.unit && lane == 0) a.unit[row] = unit;
    if (a.g.dq) {
        T* o = const_cast<T*>(at<T>(a.g.dq, a.g.dq_strides, b, i, h));
#pragma unroll
        for (int c = 0; c < kPer; ++c)
            if (lane + 64 * c < d.dim) o[lane + 64 * c] = static_cast<T>(acc[c] * unit);
    }
    return (wave_sum(e0) * (wave_sum(pf) * unit) - wave_sum(e1)) * unit;
}

// The gradients of one key and value, over all queries of the heads that share it. LDS: k and v of the row.
template <typename T>
__device__ void row_dkv(const AttnArgs& a, const Scope& sc, int64_t b, int kvh, int j, float* k, float* v) {
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
        for (int i0 = 0; i0 < d.q_len; i0 += 64) {
            const int i = i0 + lane;
            const int64_t row = (b * d.q_heads + h) * d.q_len + i;
            const bool see = i < d.q_len && sc.seen(i, j) && a.g.lse[row] != -INFINITY;
            float p = 0.f, dz = 0.f;
            if (see) {
                float grad;
                float s = capped(dot_row(k, at<T>(d.q, d.q_strides, b, i, h), d.dim) * d.scale, d.cap, grad);
                if (d.slopes) s -= slope * sc.distance(i, j);
                p = expf(s - a.g.lse[row]) * (a.unit ? a.unit[row] : 1.f);
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
    const int i = static_cast<int>(blockIdx.x) * 4 + w;
    const int64_t b = blockIdx.z;
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
    const T* rest = d.o_rest ? static_cast<const T*>(d.o_rest) + (o - static_cast<const T*>(a.g.o)) : nullptr;
    for (int x = lane; x < d.dim; x += 64) s += (static_cast<float>(o[x]) + (rest ? static_cast<float>(rest[x]) : 0.f)) * static_cast<float>(dr[x]);
    s = wave_sum(s);
    if (lane == 0) a.delta[(b * d.q_heads + h) * d.q_len + i] = s;
}

template <typename T>
__global__ __launch_bounds__(256) void k_attn_dq_rows(AttnArgs a) {
    __shared__ float q[4][kD], dout[4][kD];
    const int w = threadIdx.x >> 6, h = blockIdx.y;
    const int i = static_cast<int>(blockIdx.x) * 4 + w;
    const int64_t b = blockIdx.z;
    if (i >= a.d.q_len) return;
    const float share = row_dq<T>(a, Scope(a.d, b), b, h, i, q[w], dout[w]);
    if (a.slope_part && (threadIdx.x & 63) == 0)
        a.slope_part[(static_cast<int64_t>(h) * a.d.batch + b) * a.slots + i] = share;
}

template <typename T>
__global__ __launch_bounds__(256) void k_attn_dkv_rows(AttnArgs a) {
    __shared__ float k[4][kD], v[4][kD];
    const int w = threadIdx.x >> 6;
    const int j = static_cast<int>(blockIdx.x) * 4 + w;
    const int64_t b = blockIdx.z;
    if (j >= a.d.k_len) return;
    row_dkv<T>(a, Scope(a.d, b), b, blockIdx.y, j, k[w], v[w]);
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

__device__ __forceinline__ float sum16(const f32x16& x) {      // as a tree: a chain would wait for each addition
    float s[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) s[r] = x[r] + x[r + 8];
    return ((s[0] + s[4]) + (s[2] + s[6])) + ((s[1] + s[5]) + (s[3] + s[7]));
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

    // Where a lane reads in a tile. Unit indexes enter the swizzle by exclusive or, so every fragment's address is the
    // lane's own, exclusive-or a constant, plus a constant that the instruction adds: one operation a read, and one
    // register kept. (Taken as a sum, the compiler keeps the address of every fragment in a register, and spills.)
    struct Lane {
        uint32_t row, col;
        // anew for each tile, and in a way the compiler does not see through, or it would keep them all again
        __device__ __forceinline__ Lane at_tile(const char* tile) const {
            const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((WST_LDS const char*)tile));
            Lane l{row + base, col + base};
            asm volatile("" : "+v"(l.row), "+v"(l.col));
            return l;
        }
    };
    static __device__ __forceinline__ Lane lane() {
        const int x = threadIdx.x & 63, h = x >> 5;
        Lane l;
        if constexpr (sizeof(T) == 2) {
            l.row = at(x & 31, h);
            // the transposing read: sixteen lanes hand in four rows of sixteen values and get a column of four each
            const int g = x >> 4, y = x & 15;
            l.col = at(4 * (g >> 1) + (y >> 2), 2 * (g & 1) + ((y & 3) >> 1)) + 8 * (y & 1);
        } else {
            l.row = at(x & 31, 2 * h);
            l.col = 4 * h * kRowBytes + 4 * (x & 31);      // unswizzled
        }
        return l;
    }
    // of a constant unit offset: the bits the swizzle reaches, and the rest
    static constexpr int kBits = kUnits % 16 == 0 ? 15 : kUnits % 8 == 0 ? 7 : 3;
    static __device__ __forceinline__ uint32_t to(uint32_t lane, int row, int unit) {
        return (lane ^ ((unit & kBits) << 4)) + row * kRowBytes + ((unit & ~kBits) << 4);
    }

    // row row0 + lane % 32, values 16 c + 8 (lane / 32) .. + 7; row0 a multiple of 16
    static __device__ __forceinline__ Frag<T> row_frag(const Lane& l, int row0, int c) {
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            f = *(WST_LDS const Frag<T>*)(to(l.row, row0, 2 * c));
        } else {
            const f32x4 a = *(WST_LDS const f32x4*)(to(l.row, row0, 4 * c));
            const f32x4 b = *(WST_LDS const f32x4*)(to(l.row, row0, 4 * c + 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[e] = a[e];
                f[4 + e] = b[e];
            }
        }
        return f;
    }
    // value 32 db + lane % 32 of the eight rows row0 + 8 (e / 4) + 4 (lane / 32) + e % 4; row0 a multiple of 16
    static __device__ __forceinline__ Frag<T> col_frag(const Lane& l, int row0, int db) {
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            union {
                s16x4 q[2];
                Frag<T> f;
            } u;
#pragma unroll
            for (int k = 0; k < 2; ++k)      // eight rows on, swizzle bit 1 turns
                u.q[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((WST_LDS s16x4*)(to(l.col, row0 + 8 * k, 4 * db + 2 * k)));
            f = u.f;
        } else {
            const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int row = 8 * (e >> 2) + (e & 3);
                const uint32_t swz = (swizzle(row) << 4) ^ (swizzle(4 * h) << 4);
                f[e] = *(WST_LDS const float*)(((l.col + db * 128) ^ swz) + (row0 + row) * kRowBytes);
            }
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

// A pointer that is the same for all lanes, as a scalar.
template <typename T>
__device__ __forceinline__ T* uniform(T* p) {
    const uint64_t x = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<T*>(static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32))) << 32 |
                                static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x))));
}

// The kernel's arguments, read again: what only the end of a kernel needs then takes no scalar registers before (the
// compiler loads all arguments at the start, and at about a hundred scalars spills them to vector lanes in the loop).
__device__ __forceinline__ const AttnArgs& again() {
    auto p = (const __attribute__((address_space(4))) AttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const AttnArgs*)p;
}

// N rows of a tensor straight into LDS, past the registers, by 256 threads: each lane names the 16 bytes it wants, and a
// wave's land one after the other, so the swizzle is in the choice of the source. A lane's offsets from the tile's first
// row are the same for every tile; what moves is the scalar base. Lanes whose row does not exist or belongs to no
// document, and those beyond the head's width, fetch nothing and leave what is there: zeros at first (clear()), later
// perhaps an earlier tile's row, which the mask keeps out like any other. The compiler does not know of these loads:
// arrived() waits for them.
template <typename T, int DP, int N>
struct Fetch {
    using L = Tile<T, DP>;
    static constexpr int kCount = N * L::kUnits / 256;
    static_assert(N * L::kUnits % 256 == 0, "whole waves");
    static constexpr int kStep = 256 / L::kUnits;                                     // rows from one count to the next
    static constexpr bool kSame = 256 % L::kUnits == 0 && kStep % 16 == 0;            // the same unit and swizzle in each
    static constexpr int kOff = kSame ? 1 : kCount;
    uint32_t off[kOff], live;
    int64_t stride;
    uint32_t wave;          // this wave's part of a tile

    __device__ __forceinline__ void init(int64_t stride_, int dim, int t) {
        stride = stride_;
        wave = __builtin_amdgcn_readfirstlane(t >> 6) * 1024;
        live = 0;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int id = t + i * 256, row = id / L::kUnits, unit = (id % L::kUnits) ^ L::swizzle(row);
            if (i < kOff) off[i] = static_cast<uint32_t>(row * stride * sizeof(T)) + unit * 16;
            live |= static_cast<uint32_t>(unit * L::kElems < dim) << i;
        }
    }
    // base: the tile's first row; whole: all its rows exist, and belong to some document; left: rows that exist from
    // there on; doc: the rows' documents in LDS, or nullptr
    __device__ __forceinline__ void issue(const T* base, bool whole, int left, const int* doc, const char* tile, int t) const {
        const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((WST_LDS const char*)tile)) + wave;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int row = (t + i * 256) / L::kUnits;
            const T* b = kSame ? base + i * kStep * stride : base;
            if (whole || ((live >> i & 1) && row < left && (!doc || doc[row] >= 0)))
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                             : : "s"(__builtin_amdgcn_readfirstlane(lds + i * 4096)), "v"(off[kSame ? 0 : i]), "s"(uniform(b)) : "memory", "m0");
        }
    }
};
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }

template <int BYTES, int TH = 256>
__device__ __forceinline__ void clear(char* p, int t) {
    for (int i = t * 16; i < BYTES; i += TH * 16) *reinterpret_cast<u32x4*>(p + i) = u32x4{0, 0, 0, 0};
}

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
template <typename T, int DP>
__device__ __forceinline__ void negate(Frag<T> (&f)[DP / 16]) {
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) f[c] = -f[c];
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

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Caps up to here, in 16-bit types, are taken as -1 / (e + 1) (Shape), which is off by about 2^-23 of the cap whatever the
// score: a weight is off by 2^-17 of itself at most, a thirty-second of a rounding to float16 and less of one to bfloat16.
// The error grows with the cap (at 1e6 a weight would be off by a tenth, from 1e8 on all scores be equal), so beyond the
// tanh is taken to a relative error (bend, FINE), in a kernel for all kinds of biases. 8192 x 8 heads x 128 in order,
// bfloat16, cap 64 and 65: forward 212 and 259 us, with its backward pass 811 and 1170; 64 wide 160 and 216, 599 and 829.
constexpr float kNearCap = 64.f;

// Scores in powers of two, as an affine function of what the tiles hold: score = mul * x + add. Plainly x is the dot
// product and mul = scale log2 e, so that scaling costs nothing beyond the subtraction of the maximum. Capped, with
// e = exp(2 z / cap), tanh = 1 - 2 / (e + 1), x is -1 / (e + 1): the cap's slope is 1 - tanh^2 = -4 x (1 + x); for caps
// beyond kNearCap x is the tanh itself; float32 takes the library's tanh, good to an ulp. With a
// bias x is the score itself, mul = log2 e: slopes times log2 e, rounded, would be the slopes of a network a little way
// off. For a maximum over x mul must not be negative: there a negative
// scale turns q over instead (sign = false).
struct Shape {
    float raw, mul, add;      // of the score before the bias
    float twice, turn;        // 2 |scale| log2 e / cap;  |scale| / cap
    bool cap;
    template <typename T>
    static __device__ __forceinline__ Shape of(const wst_attention_desc& d, bool sign = false, bool fine = false) {
        Shape s;
        const float scale = sign ? d.scale : fabsf(d.scale);
        s.cap = d.cap > 0.f;
        // held to finite numbers: a dot product of 0 stays 0 under the smallest caps
        s.twice = s.cap ? fminf(fmaxf(2.f * scale * kLog2e / d.cap, -FLT_MAX), FLT_MAX) : 0.f;
        s.turn = s.cap ? fminf(fmaxf(scale / d.cap, -FLT_MAX), FLT_MAX) : 0.f;
        s.raw = !s.cap ? scale : sizeof(T) == 4 || fine ? d.cap : 2.f * d.cap;
        s.mul = d.slopes ? kLog2e : s.raw * kLog2e;
        s.add = s.cap && sizeof(T) != 4 && !fine ? d.cap * kLog2e : 0.f;
        return s;
    }
    // dot products to x before the bias, and the cap's slope
    // FINE: x is the tanh itself, for caps beyond kNearCap and for the slopes' gradient, a float32 sum that keeps what
    // 16-bit weights do not. Its series to y^9 up to 1/4 (the next term is below 2^-26 of it there), beyond
    // 1 - 2 / (e + 1), off by 6 roundings of 1 and so by 24 of itself or fewer.
    template <typename T, bool GRAD, bool FINE = false>
    __device__ __forceinline__ void bend(f32x16& x, f32x16& grad) const {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if constexpr (sizeof(T) == 4) {
                x[r] = tanhf(x[r] * turn);
                if constexpr (GRAD) grad[r] = 1.f - x[r] * x[r];
            } else if constexpr (FINE) {
                const float y = x[r] * turn, y2 = y * y;
                const float series = fmaf(y * y2, fmaf(y2, fmaf(y2, fmaf(y2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), y);
                const float outer = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x[r] * twice)), 1.f);
                x[r] = fabsf(y) < 0.25f ? series : outer;
                if constexpr (GRAD) grad[r] = fmaf(-x[r], x[r], 1.f);
            } else {
                x[r] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(x[r] * twice));
                if constexpr (GRAD) {
                    const float y = -4.f * x[r];
                    grad[r] = fmaf(y, x[r], y);
                }
            }
        }
    }
};

// What a lane's query (forward, dq) needs: the first key it may not see in order, its document and coordinates.
struct Query {
    int limit, doc, place;
    uint32_t pos[kAxes];
};
constexpr uint32_t kPosBias = 0x40000000u;   // coordinates in +-2^29 as unsigned numbers

__device__ __forceinline__ Query query_of(const Scope& sc, int i, bool ok) {
    Query q;
    q.limit = ok ? sc.limit(i) : 0;
    q.doc = sc.q_doc && ok ? sc.q_doc[i] : -1;
    if (sc.q_doc && q.doc < 0) q.limit = 0;
    q.place = i + sc.shift;
#pragma unroll
    for (int a = 0; a < kAxes; ++a)
        q.pos[a] = sc.q_pos && a < sc.axes && ok ? static_cast<uint32_t>(sc.q_pos[static_cast<int64_t>(i) * sc.axes + a]) + kPosBias : 0u;
    return q;
}

__device__ __forceinline__ uint32_t away(uint32_t a, uint32_t b, uint32_t sum) { return (a > b ? a - b : b - a) + sum; }

// Which tiles of 64 tokens a block has to visit. With documents: those where some token's document lies in the block's
// own range; and whether a tile's tokens all belong to the one document that all of the block's own do, so that no pair
// needs a look. Up to kWords * 64 tiles are marked, tiles beyond are visited.
constexpr int kWords = 64;
struct Marks {
    uint64_t any[kWords], full[kWords], stray[kWords];       // stray: some token belongs to no document, or does not exist

    // Whether all rows of tile k can be fetched without a look at their documents, which in a tile takes about as long
    // as its products (2 x 4096 x 8 heads x 64, one document: 144 us, 132 without).
    __device__ __forceinline__ bool clean(int k) const {
        return k < kWords * 64 && !(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(stray)[k >> 4])) >> (k & 15) & 1u);
    }
};

// own: the documents of the block's tokens own0 .. own0 + own_count - 1 (those below own_rows exist); other: of the tiles
// tile0 .. tile1 - 1, tokens below other_rows. A wave takes sixteen tiles at a time, all loads on their way at once.
__device__ __forceinline__ void scan_documents(Marks& m, const int32_t* own, int own0, int own_count, int own_rows,
                                               const int32_t* other, int tile0, int tile1, int other_rows, int waves = 4) {
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
    const int count = tile1 - tile0 < kWords * 64 ? tile1 - tile0 : kWords * 64;
    for (int k0 = w * 16; k0 < count; k0 += 16 * waves) {
        int v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int j = (tile0 + k0 + k) * 64 + lane;
            v[k] = k0 + k < count && j < other_rows ? other[j] : -1;
        }
        // a lane's own bits first, a bit a tile, then all lanes' together (48 ballots at once take all scalar registers)
        uint32_t some = 0, not_full = 0;                     // bits 16 .. 31 of some: of no document
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            some |= static_cast<uint32_t>(v[k] >= lo && v[k] <= hi) << k | static_cast<uint32_t>(v[k] < 0) << (16 + k);
            not_full |= static_cast<uint32_t>(v[k] != lo) << k;
        }
#pragma unroll
        for (int k = 32; k; k >>= 1) {
            some |= __shfl_xor(some, k);
            not_full |= __shfl_xor(not_full, k);
        }
        if (lane == 0) {
            reinterpret_cast<uint16_t*>(m.any)[k0 >> 4] = static_cast<uint16_t>(some);
            reinterpret_cast<uint16_t*>(m.full)[k0 >> 4] = static_cast<uint16_t>(one ? ~not_full : 0u);
            reinterpret_cast<uint16_t*>(m.stray)[k0 >> 4] = static_cast<uint16_t>(some >> 16);
        }
    }
}

// The order of a block's tiles: first those in which no pair needs a look (full), then the others, so that each kind has
// a loop of its own. (One loop that chooses its body costs registers: where the bodies meet the compiler keeps two copies
// of the sums.) Tiles full0 .. full1 - 1 are full as far as lengths and order go; with documents, those of them that the
// marks say so.
struct Walk {
    int tile0, tile1, full0, full1;
    bool marked;
};
struct Step {
    int tile, rest;       // rest: 0 among the full tiles, 1 among the others

    __device__ __forceinline__ bool done(const Walk& w) const { return tile >= w.tile1; }
    __device__ __forceinline__ void find(const Walk& w, const Marks& m) {
        int t = tile + 1;
        if (!w.marked) {
            if (rest) t = t >= w.full0 && t < w.full1 ? w.full1 : t;
            else t = max(t, w.full0) < w.full1 ? max(t, w.full0) : w.tile1;
            tile = t < w.tile1 ? t : w.tile1;
            return;
        }
        tile = w.tile1;
        while (t < w.tile1) {
            const int k = t - w.tile0, first = t - (k & 15);
            if (k >= kWords * 64) {
                if (rest) tile = t;
                return;
            }
            // sixteen tiles' marks; those past the last are never set
            uint32_t any = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint16_t*>(m.any)[k >> 4]);
            uint32_t full = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint16_t*>(m.full)[k >> 4]);
            const int a = w.full0 - first, b = w.full1 - first;
            full &= (a <= 0 ? ~0u : a >= 16 ? 0u : ~0u << a) & (b >= 16 ? ~0u : b <= 0 ? 0u : ~(~0u << b));
            any = (rest ? any & ~full : full) >> (k & 15);
            if (any) {
                tile = t + __builtin_ctz(any);
                return;
            }
            t = first + 16;
        }
    }
    __device__ __forceinline__ void go(const Walk& w, const Marks& m) {
        find(w, m);
        if (tile >= w.tile1 && !rest) {
            rest = 1;
            tile = w.tile0 - 1;
            find(w, m);
        }
    }
};

// What goes along with a key tile in LDS: coordinates and documents, ready to compare.
struct Along {
    uint32_t pos[kAxes][64];
    int doc[64];
};

// One thread's share of it on its way: t < 192 one coordinate, t < 64 one document.
struct AlongStage {
    uint32_t pos;
    int doc;
    __device__ __forceinline__ void load(const int32_t* p, const int32_t* d, int axes, int row0, int rows, int t) {
        const int row = row0 + (t & 63);
        const bool ok = row < rows;
        if (p) pos = (t >> 6) < axes && ok ? static_cast<uint32_t>(p[static_cast<int64_t>(row) * axes + (t >> 6)]) + kPosBias : 0u;
        if (d) {
            doc = t < 64 && ok ? d[row] : -2;    // -2 matches nobody; a key without a document holds a negative number,
            if (doc < 0) doc = -2;               // and queries without one see nothing anyway
        }
    }
    __device__ __forceinline__ void store(Along& al, const int32_t* p, const int32_t* d, int t) const {
        if (p && t < 64 * kAxes) al.pos[t >> 6][t & 63] = pos;
        if (d && t < 64) al.doc[t] = doc;
    }
};

// The kinds of scores a kernel is compiled for: CAP 0 or 1; BIAS 0 none, 1 by place, 2 by coordinates; 2 and 3 stand for
// "as the call says". Branches on these inside the loop over tiles cost more than the branch: the compiler moves whole
// tiles of registers where the ways meet (forward, 8192 x 8 heads x 128, no cap, no bias: 318 us with such branches, 300
// without, in one process).
// float32, whose products take sixteen times as long, has the one general kernel, and 16-bit types one for caps beyond
// kNearCap.
struct Kind {
    bool cap, bias, coordinates;
};
template <int CAP, int BIAS>
__device__ __forceinline__ Kind kind_of(const wst_attention_desc& d) {
    Kind k;
    k.cap = CAP == 2 ? d.cap > 0.f : CAP == 1;
    k.bias = BIAS == 3 ? d.slopes != nullptr : BIAS != 0;
    k.coordinates = BIAS == 3 ? d.q_pos != nullptr : BIAS == 2;
    return k;
}

// Whether scores are capped by the tanh itself (Shape::bend) in 16-bit types.
template <typename T, int CAP>
constexpr bool kFar = sizeof(T) == 2 && CAP == 2;

// Turns 32 x 32 dot products (rows: keys key0 + 32 sub .., column: the lane's query) into x of Shape, -inf where the
// query does not see the key. GRAD: also the cap's slope and the distances.
template <typename T, bool GRAD, int MASK, bool FINE = false>
__device__ __forceinline__ void scores(f32x16& x, const Kind& kind, const Shape& sh, float slope, const Query& q, const Along& al,
                                       int key0, int sub, f32x16& grad, f32x16& far) {
    const int h = (threadIdx.x & 63) >> 5;
    if (kind.cap) sh.bend<T, GRAD, FINE>(x, grad);
    if (kind.bias) {
        if (kind.coordinates) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                uint32_t sum[4] = {0, 0, 0, 0};
#pragma unroll
                for (int a = 0; a < kAxes; ++a) {
                    const u32x4 k = *reinterpret_cast<const u32x4*>(&al.pos[a][32 * sub + 8 * g + 4 * h]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] = away(q.pos[a], k[e], sum[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float f = static_cast<float>(sum[e]);
                    if constexpr (GRAD) far[4 * g + e] = f;
                    x[4 * g + e] = fmaf(-slope, f, x[4 * g + e] * sh.raw);
                }
            }
        } else {
            const float base = static_cast<float>(q.place - (key0 + 32 * sub + 4 * h));
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float f = fabsf(base - static_cast<float>(8 * (r >> 2) + (r & 3)));
                if constexpr (GRAD) far[r] = f;
                x[r] = fmaf(-slope, f, x[r] * sh.raw);
            }
        }
    }
    if constexpr (MASK != 0) {
        const int rel = q.limit - (key0 + 32 * sub + 4 * h);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if constexpr (MASK == 2) {
                const i32x4 k = *reinterpret_cast<const i32x4*>(&al.doc[32 * sub + 8 * g + 4 * h]);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * g + e] = ((8 * g + e < rel) & (k[e] == q.doc)) ? x[4 * g + e] : -INFINITY;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * g + e] = 8 * g + e < rel ? x[4 * g + e] : -INFINITY;
            }
        }
    }
}

template <typename T, int DP>
__device__ __forceinline__ bool not_finite(const f32x16 (&o)[DP / 32]) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < DP / 32; ++k)
#pragma unroll
        for (int r = 0; r < 16; ++r) t = fmaf(o[k][r], 0.f, t);
    return t != t;
}

template <typename T>
inline constexpr float kSlack = 40.f;
template <>
inline constexpr float kSlack<f16> = 12.f;     // weights below 2^13 times the sum's rounding to float16

// The order of LDS reads and matrix instructions in a product of STEPS instructions that take READS reads each: AHEAD
// instructions' operands are read before the first, then each instruction is followed by the reads of a later one.
// Left to itself the compiler reads either one operand at a time, and waits for each, or all of them, and spills.
template <int STEPS, int READS, int AHEAD>
__device__ __forceinline__ void paced() {
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
    for (int i = 0; i < STEPS - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
    __builtin_amdgcn_sched_barrier(0);
}

constexpr int kBQ = 128, kBK = 64;

// Two teams a block (k_attn_fwd, k_attn_dq) where the rows are of many lengths; float32 has no room in LDS for two.
inline bool two_teams(const wst_attention_desc& d) { return d.dtype != WST_F32 && d.causal && d.k_len > 2 * kBK; }

// Forward pass: a block takes 128 queries of a head, 32 a wave, and walks the key tiles that any of them may see, keeping
// the running maximum, sum and output of the softmax in registers; keys and values of a tile are shared through LDS.
// The maximum is that of the first tile that shows the query anything, and stays as long as no score exceeds it by
// kSlack powers of two: larger weights cost neither sums nor roundings anything, and the output is not scaled. A wave
// that meets such a score goes on in loops that move the maximum with every tile. (As a branch inside the loop the
// scaling costs as much when it is not taken: where the ways meet, the compiler copies all sums between registers.)
//
// TEAMS: one or two teams of four waves. Two share the queries and take every other tile, each through its own part of
// LDS, and join their maxima, sums and outputs at the end: the block with the longest rows of an order does not run on
// alone at half the rate. Where all blocks are as long, two independent blocks are better than two teams that wait for
// each other at every tile (8192 x 8 heads x 128: in order 238 -> 201 us, dq 283 -> 250; not in order 327 -> 379).
//
// Bound by the matrix units and, with a cap or a bias, as much by what a score takes besides: 8192 x 8 heads of 128
// 327 us, 840 TFLOP/s; in order 201 us; with cap 50 and a prefix 262 us.
template <typename T, int DP, int CAP, int BIAS, int TEAMS>
__global__ __launch_bounds__(256 * TEAMS, sizeof(T) == 2 ? 2 : 1) void k_attn_fwd(AttnArgs a) {
    using L = Tile<T, DP>;
    constexpr int kTile = kBK * L::kRowBytes;
    __shared__ __attribute__((aligned(256))) char pool[TEAMS * 4 * kTile];
    __shared__ Along alongs[TEAMS][3];
    __shared__ Marks marks;
    __shared__ float scratch[4][DP];
    const wst_attention_desc& d = a.d;
    const int team = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
    const int t = threadIdx.x & 255, lane = t & 63, w = t >> 6, hl = lane >> 5;
    char *kt = pool + team * 4 * kTile, *vt = kt + 2 * kTile;
    Along* al = alongs[team];
    const uint32_t cells = static_cast<uint32_t>(d.batch) * d.q_heads, bh = blockIdx.x % cells;
    const int nq = static_cast<int>((d.q_len + kBQ - 1) / kBQ), i0 = (nq - 1 - static_cast<int>(blockIdx.x / cells)) * kBQ;   // long rows first
    const int64_t b = bh / d.q_heads;
    const int h = static_cast<int>(bh % d.q_heads), kvh = h / (d.q_heads / d.k_heads);
    const Scope sc(d, b);
    const Shape sh = Shape::of<T>(d, false, kFar<T, CAP>);
    const Kind kind = kind_of<CAP, BIAS>(d);
    const int i = i0 + w * 32 + (lane & 31);
    const bool ok = i < d.q_len;
    const Query q = query_of(sc, i, ok);
    const float slope = d.slopes ? d.slopes[h] : 0.f;
    Frag<T> qf[DP / 16];
    row_frags<T, DP>(at<T>(d.q, d.q_strides, b, ok ? i : 0, h), ok && q.limit > 0, d.dim, qf);
    if (d.scale < 0.f) negate<T, DP>(qf);

    // keys below `end` may be seen by some query of the block, keys below `open` by all of its queries in order
    const int last = i0 + kBQ < d.q_len ? i0 + kBQ - 1 : static_cast<int>(d.q_len) - 1;
    const int end = sc.limit(last), open = sc.limit(i0);
    const int tiles = end > 0 ? (end + kBK - 1) / kBK : 0;
    const bool marked = sc.q_doc != nullptr, along = sc.q_doc || sc.q_pos;
    if (marked) scan_documents(marks, sc.q_doc, i0, kBQ, static_cast<int>(d.q_len), sc.k_doc, 0, tiles, sc.length, 4 * TEAMS);
    if (marked || d.dim != DP || sc.length % kBK) {
        clear<4 * kTile>(kt, t);
    }
    f32x16 o[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) o[k] = zero16();
    float m = -INFINITY, l = 0.f;

    const T *kb = at<T>(d.k, d.k_strides, b, 0, kvh), *vb = at<T>(d.v, d.v_strides, b, 0, kvh);
    const int64_t ks = d.k_strides[1], vs = d.v_strides[1];
    Fetch<T, DP, kBK> kf, vf;
    kf.init(ks, d.dim, t);
    vf.init(vs, d.dim, t);
    // a tile's keys and values are on their way while the tile before is worked on, its documents and coordinates (which
    // decide what to fetch) one tile earlier still
    auto fetch = [&](int n, int buf, const Along& with) {
        const int* doc = marked ? with.doc : nullptr;
        const int left = sc.length - n * kBK;
        const bool whole = d.dim == DP && left >= kBK && (!marked || marks.clean(n));
        kf.issue(kb + static_cast<int64_t>(n) * kBK * ks, whole, left, doc, kt + buf * kTile, t);
        vf.issue(vb + static_cast<int64_t>(n) * kBK * vs, whole, left, doc, vt + buf * kTile, t);
    };
    AlongStage as{};
    if (marked) __syncthreads();       // the marks
    const Walk walk{0, tiles, 0, open / kBK, marked};
    bool behind = false;               // the first team has a tile after the second one's last
    auto go = [&](Step& x) {           // over the other team's tile to the next of this one's
        x.go(walk, marks);
        if constexpr (TEAMS > 1) {
            if (x.done(walk)) return;
            x.go(walk, marks);
            behind = x.done(walk);
        }
    };
    Step cur{-1, 0};
    if (team) go(cur);
    else cur.go(walk, marks);
    Step next = cur;
    if (!cur.done(walk)) go(next);
    if (along) {
        if (!cur.done(walk)) {
            as.load(sc.k_pos, sc.k_doc, sc.axes, cur.tile * kBK, sc.length, t);
            as.store(al[0], sc.k_pos, sc.k_doc, t);
        }
        if (!next.done(walk)) {
            as.load(sc.k_pos, sc.k_doc, sc.axes, next.tile * kBK, sc.length, t);
            as.store(al[1], sc.k_pos, sc.k_doc, t);
        }
    }
    __syncthreads();                   // documents and zeros
    if (!cur.done(walk)) fetch(cur.tile, 0, al[0]);
    const typename L::Lane lanes = L::lane();
    int buf = 0, turn = 0;
    int turn1 = 0, turn2 = 0;
    Step after = next;
    auto enter = [&]() {               // the tile is there, and nobody reads the other buffer any more
        turn1 = turn == 2 ? 0 : turn + 1;
        turn2 = turn1 == 2 ? 0 : turn1 + 1;
        arrived();
        __syncthreads();
        after = next;
        if (!next.done(walk)) {
            fetch(next.tile, buf ^ 1, al[turn1]);
            go(after);
            if (along && !after.done(walk)) as.load(sc.k_pos, sc.k_doc, sc.axes, after.tile * kBK, sc.length, t);
        }
    };
    auto leave = [&]() {
        if (along && !after.done(walk)) as.store(al[turn2], sc.k_pos, sc.k_doc, t);
        cur = next;
        next = after;
        buf ^= 1;
        turn = turn1;
    };
    // x of a tile, and the query's largest
    auto look = [&](auto mask, f32x16 (&x)[2]) {
        const typename L::Lane kc = lanes.at_tile(kt + buf * kTile);
        x[0] = x[1] = zero16();
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
#pragma unroll
            for (int n = 0; n < 2; ++n) x[n] = Mma<T>::mul(L::row_frag(kc, 32 * n, c), qf[c], x[n]);
        if constexpr (sizeof(T) == 2) paced<DP / 8, 1, 4>();
        f32x16 unused;
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            scores<T, false, decltype(mask)::value, kFar<T, CAP>>(x[n], kind, sh, slope, q, al[turn], cur.tile * kBK, n, unused, unused);
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, x[n][r]);
        }
        return halves_max(top) * sh.mul;
    };
    auto add = [&](f32x16 (&x)[2]) {
        const typename L::Lane vc = lanes.at_tile(vt + buf * kTile);
        const float base = fmaxf(m, -3.0e38f);         // nothing seen yet: exp2(-inf) = 0 either way
        Frag<T> p[2][2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) x[n][r] = __builtin_amdgcn_exp2f(fmaf(x[n][r], sh.mul, -base));
            l += sum16(x[n]);
            to_frags<T>(x[n], p[n]);
        }
        if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) o[db] = Mma<T>::mul(L::col_frag(vc, 32 * n + 16 * k, db), p[n][k], o[db]);
        if constexpr (sizeof(T) == 2) paced<DP / 8, 2, 3>();
    };
    bool slow = false;                 // of the wave: a score has come that the maximum must move for
    auto fast = [&](auto mask) {
        enter();
        f32x16 x[2];
        const float mn = look(mask, x);
        m = m == -INFINITY ? mn : m;
        slow = __ballot(mn > m + kSlack<T>) != 0;
        if (slow) return;
        add(x);
        leave();
    };
    bool entered = false;
    auto careful = [&](auto mask) {
        if (!entered) enter();
        entered = false;
        f32x16 x[2];
        const float m1 = fmaxf(m, look(mask, x)), f = __builtin_amdgcn_exp2f(m - fmaxf(m1, -3.0e38f));
        m = m1;
        l *= f;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[k][r] *= f;
        add(x);
        leave();
    };
    while (!cur.done(walk) && !cur.rest && !slow) fast(std::integral_constant<int, 0>{});
    while (!cur.done(walk) && !marked && !slow) fast(std::integral_constant<int, 1>{});
    while (!cur.done(walk) && !slow) fast(std::integral_constant<int, 2>{});
    entered = slow;
    while (!cur.done(walk) && !marked) careful(std::integral_constant<int, 1>{});
    while (!cur.done(walk)) careful(std::integral_constant<int, 2>{});
    l = halves_sum(l);
    if constexpr (TEAMS > 1) {         // a lane's registers go to the lane that has the same place in the first team
        static_assert(sizeof(pool) >= 4 * (DP / 2 + 2) * 64 * sizeof(float), "room for the sums");
        float* sums = reinterpret_cast<float*>(pool) + w * ((DP / 2 + 2) * 64) + lane;
        if (team && behind) __syncthreads();           // as many waits as the first team's
        __syncthreads();
        if (team) {
#pragma unroll
            for (int k = 0; k < DP / 32; ++k)
#pragma unroll
                for (int r = 0; r < 16; ++r) sums[(16 * k + r) * 64] = o[k][r];
            sums[(DP / 2) * 64] = m;
            sums[(DP / 2 + 1) * 64] = l;
        }
        __syncthreads();
        if (team) return;
        const float m2 = sums[(DP / 2) * 64], top = fmaxf(m, m2), base = fmaxf(top, -3.0e38f);
        const float f = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
        l = l * f + sums[(DP / 2 + 1) * 64] * f2;
        m = top;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[k][r] = o[k][r] * f + sums[(16 * k + r) * 64] * f2;
    }
    const AttnArgs& z = again();
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (ok) {
        T* out = const_cast<T*>(at<T>(z.o, z.d.o_strides, b, i, h));
        T* rest = z.d.o_rest ? static_cast<T*>(z.d.o_rest) + (out - static_cast<T*>(z.o)) : nullptr;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * db + 8 * g + 4 * hl;
                float v[4] = {o[db][4 * g] * inv, o[db][4 * g + 1] * inv, o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv};
                if (c >= z.d.dim) continue;
                store<4>(out + c, v);
                if (rest) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(lost<T>(v[e]));
                    store<4>(rest + c, v);
                }
            }
        if (hl == 0 && z.lse) z.lse[(b * z.d.q_heads + h) * z.d.q_len + i] = l == 0.f ? -INFINITY : (m + sh.add) * kLn2 + logf(l);
    }
    // A value that is not finite, of a key that some query of the wave does not see, has reached that query as 0 * inf:
    // the queries whose output is not finite are done over, key by key. In ordinary data there are none.
    uint64_t bad = __ballot(ok && not_finite<T, DP>(o));
    for (bad = (bad | bad >> 32) & 0xffffffffu; bad; bad &= bad - 1)
        row_forward<T>(z, Scope(z.d, b), b, h, i0 + w * 32 + __builtin_ctzll(bad), scratch[w]);
}

// Few queries over many keys: the queries of all heads that share a key head make up to 32 rows, and the keys are split
// over blocks, and in a block over its waves, each of which walks its own tiles of 32 keys through its own part of LDS
// with nothing to wait for. The parts are joined by their maxima and sums, in the block and then by k_attn_join. Bound by
// memory: 64 queries of 8 heads over 64 x 3/4 of 4096 keys of 2 x 64 in bfloat16, 100 MB: 29 us, 3.5 TB/s.
template <typename T, int DP, int CAP, int BIAS>
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
    const int i = static_cast<int>(ok ? r % d.q_len : 0);
    const int h = kvh * group + static_cast<int>(ok ? r / d.q_len : 0);
    const Scope sc(d, b);
    const Shape sh = Shape::of<T>(d, false, kFar<T, CAP>);
    const Kind kind = kind_of<CAP, BIAS>(d);
    const Query q = query_of(sc, i, ok);
    const float slope = d.slopes ? d.slopes[h] : 0.f;
    Frag<T> qf[DP / 16];
    row_frags<T, DP>(at<T>(d.q, d.q_strides, b, i, h), ok && q.limit > 0, d.dim, qf);
    const int end = sc.limit(static_cast<int>(d.q_len) - 1);
    // this split's keys, in whole groups of 128: a wave has 32 of each
    const int groups = end > 0 ? (end + 127) / 128 : 0, per = (groups + a.splits - 1) / a.splits;
    const int g0 = min(static_cast<int>(split) * per, groups), g1 = min(g0 + per, groups);
    const bool marked = sc.q_doc != nullptr;
    if (marked) {
        scan_documents(marks, sc.q_doc, 0, static_cast<int>(d.q_len < 1024 ? d.q_len : 1024), static_cast<int>(d.q_len), sc.k_doc, 2 * g0, 2 * g1, sc.length);
        __syncthreads();
    }
    const bool skip = marked && d.q_len <= 1024;   // else the marks do not speak for all queries
    auto wanted = [&](int g) {                  // the next group of 128 in whose 64 keys this wave has work
        for (; g < g1; ++g) {
            const int k = 2 * (g - g0) + (w >> 1);
            if (!skip || k >= kWords * 64) return g;
            if (__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(marks.any)[k >> 4]) >> (k & 15) & 1u)) return g;
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
    uint32_t pos[kAxes];
    int doc = -2;
    auto fetch = [&](int key0) {
        ks.load(kb, d.k_strides[1], key0, sc.length, sc.k_doc, d.dim, lane);
        vs.load(vb, d.v_strides[1], key0, sc.length, sc.k_doc, d.dim, lane);
        const int j = key0 + (lane & 31);
        if (sc.k_pos)
#pragma unroll
            for (int x = 0; x < kAxes; ++x)
                pos[x] = x < sc.axes && j < sc.length ? static_cast<uint32_t>(sc.k_pos[static_cast<int64_t>(j) * sc.axes + x]) + kPosBias : 0u;
        if (sc.k_doc) {
            doc = j < sc.length ? sc.k_doc[j] : -2;
            if (doc < 0) doc = -2;
        }
    };
    Along& mine = al[w >> 1];
    const int sub = w & 1;
    const typename L::Lane lanes = L::lane();
    int g = wanted(g0);
    if (g < g1) fetch(g * 128 + 32 * w);
    if (d.scale < 0.f) negate<T, DP>(qf);      // after the keys' loads: it waits for the queries
    while (g < g1) {
        const int key0 = g * 128 + 32 * w;
        __builtin_amdgcn_wave_barrier();
        ks.store(kt, lane);
        vs.store(vt, lane);
        if (lane < 32) {
            if (sc.k_pos)
#pragma unroll
                for (int x = 0; x < kAxes; ++x) mine.pos[x][32 * sub + lane] = pos[x];
            mine.doc[32 * sub + lane] = doc;
        }
        __builtin_amdgcn_wave_barrier();
        const int next = wanted(g + 1);
        if (next < g1) fetch(next * 128 + 32 * w);
        const typename L::Lane kc = lanes.at_tile(kt), vc = lanes.at_tile(vt);
        f32x16 s = zero16(), unused;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) s = Mma<T>::mul(L::row_frag(kc, 0, c), qf[c], s);
        if (marked) scores<T, false, 2, kFar<T, CAP>>(s, kind, sh, slope, q, mine, key0 - 32 * sub, sub, unused, unused);
        else scores<T, false, 1, kFar<T, CAP>>(s, kind, sh, slope, q, mine, key0 - 32 * sub, sub, unused, unused);
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < 16; ++x) top = fmaxf(top, s[x]);
        const float mn = halves_max(top) * sh.mul;
        const float m1 = fmaxf(m, mn), f = __builtin_amdgcn_exp2f(m - fmaxf(m1, -3.0e38f));
        m = m1;
        l *= f;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k)
#pragma unroll
            for (int x = 0; x < 16; ++x) o[k][x] *= f;
        const float base = fmaxf(m, -3.0e38f);
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], sh.mul, -base));
        l += sum16(s);
        Frag<T> p[2];
        to_frags<T>(s, p);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) o[db] = Mma<T>::mul(L::col_frag(vc, 16 * k, db), p[k], o[db]);
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
        const int ii = static_cast<int>((r0 + y) % d.q_len);
        const int hh = kvh * group + static_cast<int>((r0 + y) / d.q_len);
        const int64_t row = (b * d.q_heads + hh) * d.q_len + ii;
        const float my = __shfl(mm, y), ly = __shfl(total, y);
        if (a.splits > 1) {
            const int64_t all = d.batch * d.q_heads * d.q_len, slot = split * all + row;
            for (int e = lane; e < d.dim; e += 64) a.part[slot * d.dim + e] = sum[y * kLd + e];
            if (lane == 0) {
                a.part_ml[2 * slot] = my + sh.add;
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
                if (d.o_rest) static_cast<T*>(d.o_rest)[out - static_cast<T*>(a.o) + e] = lost<T>(v);
            }
            if (lane == 0 && a.lse) a.lse[row] = ly == 0.f ? -INFINITY : (my + sh.add) * kLn2 + logf(ly);
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
    const int64_t bh = row / d.q_len, b = bh / d.q_heads;
    const int i = static_cast<int>(row % d.q_len);
    const int h = static_cast<int>(bh % d.q_heads);
    float m = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.part_ml[2 * (s * all + row)]);
    m = wave_max(m);
    const float base = fmaxf(m, -3.0e38f);
    float l = 0.f, v[2] = {0.f, 0.f};
    for (int s0 = 0; s0 < a.splits; s0 += 64) {
        const int count = min(a.splits - s0, 64);
        float mine = 0.f;              // the lane's split's factor
        if (lane < count) {
            const int64_t slot = (s0 + lane) * all + row;
            mine = __builtin_amdgcn_exp2f(a.part_ml[2 * slot] - base);
            l = fmaf(mine, a.part_ml[2 * slot + 1], l);
        }
        for (int s = 0; s < count; s += 8) {           // eight splits' loads at a time
            float x[8][2];
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    x[u][e] = s + u < count && lane + 64 * e < d.dim ? a.part[((s0 + s + u) * all + row) * d.dim + lane + 64 * e] : 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < 2; ++e) v[e] = fmaf(__shfl(mine, (s + u) & 63), x[u][e], v[e]);
        }
    }
    l = wave_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = const_cast<T*>(at<T>(a.o, d.o_strides, b, i, h));
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < d.dim) {
            bad = bad || !(fabsf(v[e] * inv) < INFINITY);
            out[lane + 64 * e] = static_cast<T>(v[e] * inv);
            if (d.o_rest) static_cast<T*>(d.o_rest)[out - static_cast<T*>(a.o) + lane + 64 * e] = lost<T>(v[e] * inv);
        }
    if (lane == 0 && a.lse) a.lse[row] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
    if (__ballot(bad)) row_forward<T>(a, Scope(d, b), b, h, i, scratch[w]);
}

// Float16 loses small numbers before large ones: weights and score gradients are held 2^6 times as large there, so that
// they keep their precision down to 2^-20; a score gradient beyond 2^10 then overflows, and its row is done over in
// float32 like any that is not finite. That is for the odd row: 1024 tokens, 8 heads x 64, backward 100 us, 450 with output
// gradients of 2^10 and 5300 with 2^13, where nearly all rows and keys overflow.
template <typename T>
inline constexpr float kUp = 1.f;
template <>
inline constexpr float kUp<f16> = 64.f;

// dq, the slopes' shares and delta: walks the keys as the forward pass does. Scores come back as (keys x queries), so
// their gradient is the operand of dq^T = k^T dz^T as it stands; keys are read from LDS both ways. delta goes in as the
// product's starting value. 8192 x 8 heads of 128: 400 us, 1030 TFLOP/s; in order 250 us; with cap 50 and a prefix 327.
template <typename T, int DP, int CAP, int BIAS, int TEAMS>
__global__ __launch_bounds__(256 * TEAMS, sizeof(T) == 2 ? 2 : 1) void k_attn_dq(AttnArgs a) {
    using L = Tile<T, DP>;
    constexpr int kTile = kBK * L::kRowBytes;
    __shared__ __attribute__((aligned(256))) char pool[TEAMS * 4 * kTile];
    __shared__ Along alongs[TEAMS][3];
    __shared__ Marks marks;
    __shared__ float scratch[4][2][DP];
    const wst_attention_desc& d = a.d;
    const int team = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
    const int t = threadIdx.x & 255, lane = t & 63, w = t >> 6, hl = lane >> 5;
    char *kt = pool + team * 4 * kTile, *vt = kt + 2 * kTile;
    Along* al = alongs[team];
    const uint32_t cells = static_cast<uint32_t>(d.batch) * d.q_heads, bh = blockIdx.x % cells;
    const int nq = static_cast<int>((d.q_len + kBQ - 1) / kBQ), qt = nq - 1 - static_cast<int>(blockIdx.x / cells), i0 = qt * kBQ;
    const int64_t b = bh / d.q_heads;
    const int h = static_cast<int>(bh % d.q_heads), kvh = h / (d.q_heads / d.k_heads);
    const Scope sc(d, b);
    constexpr bool kFine = kFar<T, CAP> || (sizeof(T) == 2 && BIAS != 0);
    const Shape sh = Shape::of<T>(d, false, kFine);
    const Kind kind = kind_of<CAP, BIAS>(d);
    const int i = i0 + w * 32 + (lane & 31);
    const int64_t row = (b * d.q_heads + h) * d.q_len + i;
    const bool ok = i < d.q_len;
    const Query q = query_of(sc, i, ok);
    const float slope = d.slopes ? d.slopes[h] : 0.f;
    const float lse = ok ? a.g.lse[row] : -INFINITY;
    const bool live = ok && q.limit > 0 && lse != -INFINITY;
    const float base = live ? sh.add - lse * kLog2e : -INFINITY;         // of a query that sees nothing every weight is 0
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
        if (d.o_rest) {
            row_frags<T, DP>(at<T>(d.o_rest, d.o_strides, b, ok ? i : 0, h), live, d.dim, of);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) delta += static_cast<float>(df[c][e]) * static_cast<float>(of[c][e]);
        }
        delta = halves_sum(delta);
        if (ok && hl == 0 && !team) a.delta[row] = delta;
    }
    row_frags<T, DP>(at<T>(d.q, d.q_strides, b, ok ? i : 0, h), live, d.dim, qf);
    if (d.scale < 0.f) negate<T, DP>(qf);

    // keys below `end` may be seen by some query of the block, keys below `open` by all of its queries in order
    const int last = i0 + kBQ < d.q_len ? i0 + kBQ - 1 : static_cast<int>(d.q_len) - 1;
    const int end = sc.limit(last), open = sc.limit(i0);
    const int tiles = end > 0 ? (end + kBK - 1) / kBK : 0;
    const bool marked = sc.q_doc != nullptr, along = sc.q_doc || sc.q_pos;
    if (marked) scan_documents(marks, sc.q_doc, i0, kBQ, static_cast<int>(d.q_len), sc.k_doc, 0, tiles, sc.length, 4 * TEAMS);
    if (marked || d.dim != DP || sc.length % kBK) {
        clear<4 * kTile>(kt, t);
    }
    f32x16 dq[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) dq[k] = zero16();
    // The slopes' share, -sum ds far. delta comes from the rounded output, and its error would meet a mean distance: with
    // e = sum ds (0, were delta exact) the share is -(sum ds far - e sum p far), the weights made to add up to 1 in every
    // type: it is a float32 sum that stays (bfloat16, 25 x 4001 in order: 8.9e-7 from the exact one before, 0.9e-7 so; dq
    // 86 us and 87.5).
    float pf = 0.f, e0 = 0.f, e1 = 0.f, whole_p = 0.f;      // whole_p: the sum of the weights (unit_of)
    const bool slopes_too = a.slope_part != nullptr;

    const T *kb = at<T>(d.k, d.k_strides, b, 0, kvh), *vb = at<T>(d.v, d.v_strides, b, 0, kvh);
    const int64_t ks = d.k_strides[1], vs = d.v_strides[1];
    Fetch<T, DP, kBK> kf, vf;
    kf.init(ks, d.dim, t);
    vf.init(vs, d.dim, t);
    // a tile's keys and values are on their way while the tile before is worked on, its documents and coordinates (which
    // decide what to fetch) one tile earlier still
    auto fetch = [&](int n, int buf, const Along& with) {
        const int* doc = marked ? with.doc : nullptr;
        const int left = sc.length - n * kBK;
        const bool whole = d.dim == DP && left >= kBK && (!marked || marks.clean(n));
        kf.issue(kb + static_cast<int64_t>(n) * kBK * ks, whole, left, doc, kt + buf * kTile, t);
        vf.issue(vb + static_cast<int64_t>(n) * kBK * vs, whole, left, doc, vt + buf * kTile, t);
    };
    AlongStage as{};
    if (marked) __syncthreads();       // the marks
    const Walk walk{0, tiles, 0, open / kBK, marked};
    bool behind = false;               // teams as in k_attn_fwd
    auto go = [&](Step& x) {
        x.go(walk, marks);
        if constexpr (TEAMS > 1) {
            if (x.done(walk)) return;
            x.go(walk, marks);
            behind = x.done(walk);
        }
    };
    Step cur{-1, 0};
    if (team) go(cur);
    else cur.go(walk, marks);
    Step next = cur;
    if (!cur.done(walk)) go(next);
    if (along) {
        if (!cur.done(walk)) {
            as.load(sc.k_pos, sc.k_doc, sc.axes, cur.tile * kBK, sc.length, t);
            as.store(al[0], sc.k_pos, sc.k_doc, t);
        }
        if (!next.done(walk)) {
            as.load(sc.k_pos, sc.k_doc, sc.axes, next.tile * kBK, sc.length, t);
            as.store(al[1], sc.k_pos, sc.k_doc, t);
        }
    }
    __syncthreads();                   // documents and zeros
    if (!cur.done(walk)) fetch(cur.tile, 0, al[0]);
    const typename L::Lane lanes = L::lane();
    int buf = 0, turn = 0;
    auto work = [&](auto mask) {       // a tile; compiled without, with the ordinary and with the documents' mask
        constexpr int MASK = decltype(mask)::value;
        const int key0 = cur.tile * kBK;
        const int turn1 = turn == 2 ? 0 : turn + 1, turn2 = turn1 == 2 ? 0 : turn1 + 1;
        arrived();
        __syncthreads();               // the tile is there, and nobody reads the other buffer any more
        Step after = next;
        if (!next.done(walk)) {
            fetch(next.tile, buf ^ 1, al[turn1]);
            go(after);
            if (along && !after.done(walk)) as.load(sc.k_pos, sc.k_doc, sc.axes, after.tile * kBK, sc.length, t);
        }
        const typename L::Lane kc = lanes.at_tile(kt + buf * kTile), vc = lanes.at_tile(vt + buf * kTile);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            f32x16 x = zero16(), dp, grad, far;
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] = -delta;
            if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                x = Mma<T>::mul(L::row_frag(kc, 32 * n, c), qf[c], x);
                dp = Mma<T>::mul(L::row_frag(vc, 32 * n, c), df[c], dp);
            }
            if constexpr (sizeof(T) == 2) paced<DP / 8, 1, 4>();
            scores<T, true, MASK, kFine>(x, kind, sh, slope, q, al[turn], key0, n, grad, far);
            if constexpr (MASK != 0) {     // a weight of 0 may meet a value that is not finite
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] = x[r] == -INFINITY ? 0.f : dp[r];
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], sh.mul, base));
                dp[r] *= x[r];
            }
            if constexpr (sizeof(T) == 4) whole_p += sum16(x);
            if (kind.bias && slopes_too) {
                float u = 0.f, v = 0.f, y = 0.f;       // sums of their own first: thousands of terms lose little so
                if constexpr (sizeof(T) == 2) whole_p += sum16(x);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    u = fmaf(x[r], far[r], u);
                    v += dp[r];
                    y = fmaf(dp[r], far[r], y);
                }
                pf += u;
                e0 += v;
                e1 += y;
            }
            if (kind.cap) {
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] *= grad[r];
            }
            if constexpr (kUp<T> != 1.f) {
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] *= kUp<T>;
            }
            Frag<T> z[2];
            to_frags<T>(dp, z);
            if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) dq[db] = Mma<T>::mul(L::col_frag(kc, 32 * n + 16 * k, db), z[k], dq[db]);
            if constexpr (sizeof(T) == 2) paced<DP / 16, 2, 2>();
        }
        if (along && !after.done(walk)) as.store(al[turn2], sc.k_pos, sc.k_doc, t);
        cur = next;
        next = after;
        buf ^= 1;
        turn = turn1;
    };
    while (!cur.done(walk) && !cur.rest) work(std::integral_constant<int, 0>{});
    while (!cur.done(walk) && !marked) work(std::integral_constant<int, 1>{});
    while (!cur.done(walk)) work(std::integral_constant<int, 2>{});
    if constexpr (TEAMS > 1) {
        static_assert(sizeof(pool) >= 4 * (DP / 2 + 4) * 64 * sizeof(float), "room for the sums");
        float* sums = reinterpret_cast<float*>(pool) + w * ((DP / 2 + 4) * 64) + lane;
        if (team && behind) __syncthreads();
        __syncthreads();
        if (team) {
#pragma unroll
            for (int k = 0; k < DP / 32; ++k)
#pragma unroll
                for (int r = 0; r < 16; ++r) sums[(16 * k + r) * 64] = dq[k][r];
            sums[(DP / 2) * 64] = pf;
            sums[(DP / 2 + 1) * 64] = e0;
            sums[(DP / 2 + 2) * 64] = e1;
            sums[(DP / 2 + 3) * 64] = whole_p;
        }
        __syncthreads();
        if (team) return;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) dq[k][r] += sums[(16 * k + r) * 64];
        pf += sums[(DP / 2) * 64];
        e0 += sums[(DP / 2 + 1) * 64];
        e1 += sums[(DP / 2 + 2) * 64];
        whole_p += sums[(DP / 2 + 3) * 64];
    }
    const AttnArgs& z = again();
    float mul = z.d.scale / kUp<T>;
    const float unit = unit_of(halves_sum(whole_p));
    if constexpr (sizeof(T) == 4) {
        mul *= unit;
        if (ok && hl == 0) z.unit[row] = unit;
    }
    if (ok && z.g.dq) {
        T* out = const_cast<T*>(at<T>(z.g.dq, z.g.dq_strides, b, i, h));
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * db + 8 * g + 4 * hl;
                const float v[4] = {dq[db][4 * g] * mul, dq[db][4 * g + 1] * mul, dq[db][4 * g + 2] * mul, dq[db][4 * g + 3] * mul};
                if (c < z.d.dim) store<4>(out + c, v);
            }
    }
    if (z.slope_part) {
        const float share = (halves_sum(e0) * (halves_sum(pf) * unit) - halves_sum(e1)) * unit, sum = wave_sum(hl ? 0.f : share);
        if (lane == 0) z.slope_part[(static_cast<int64_t>(h) * z.d.batch + b) * z.slots + qt * 4 + w] = sum;
    }
    uint64_t bad = __ballot(ok && not_finite<T, DP>(dq));      // see k_attn_fwd
    for (bad = (bad | bad >> 32) & 0xffffffffu; bad; bad &= bad - 1) {
        __builtin_amdgcn_wave_barrier();
        row_dq<T>(z, Scope(z.d, b), b, h, i0 + w * 32 + __builtin_ctzll(bad), scratch[w][0], scratch[w][1]);
    }
}

// What goes along with a tile of 64 queries.
struct Rows {
    float base[64], delta[64];     // add - lse log2 e; -delta
    int limit[64], doc[64], place[64];
    uint32_t pos[kAxes][64];
};

// Threads of k_attn_dkv, by the width of a value and of a head.
constexpr int dkv_threads(int size, int dim) { return size == 2 && dim > 64 ? 512 : 256; }

// dk and dv: a block takes 128 keys of a key head, 32 a wave, and walks tiles of 64 queries of the heads that share it.
// Scores come as (queries x keys), one key a lane, so weights and score gradients are the operands of dv^T = do^T p and
// dk^T = q^T dz as they stand. With few key tiles the walk is split in parts whose sums k_attn_dkv_join adds in order.
//
// Heads up to 64 wide (and float32): four waves, keys and values held as operands in registers. Wider ones would then
// leave room for one wave a SIMD, which waits for LDS most of its time (8192 x 8 heads x 128, cap and prefix: 870 us,
// with eight waves 694). They take eight waves: keys and values stay in LDS, two waves share 32 keys and take half of
// each tile's queries, and add their sums at the end.
//
// Bound by the matrix units and, with a cap or a bias, as much by what a score takes besides. 8192 x 8 heads of 128:
// 670 us, 820 TFLOP/s, of 1137 that a library product of 8192^3 reaches here.
template <typename T, int DP, int CAP, int BIAS>
__global__ __launch_bounds__(dkv_threads(sizeof(T), DP), sizeof(T) == 2 ? 2 : 1) void k_attn_dkv(AttnArgs a) {
    using L = Tile<T, DP>;
    constexpr int kRows = 64, TH = dkv_threads(sizeof(T), DP), kTile = kRows * L::kRowBytes;
    constexpr bool kWide = TH == 512;
    constexpr int kOwn = kBQ * L::kRowBytes;                          // the block's keys (or values)
    __shared__ __attribute__((aligned(256))) char pool[4 * kTile + (kWide ? 2 * kOwn : 0)];
    char *qt = pool, *dt = pool + 2 * kTile, *kt = pool + 4 * kTile, *vt = kt + kOwn;
    __shared__ Rows rows[3];
    constexpr bool kUnit = sizeof(T) == 4;
    __shared__ __attribute__((aligned(16))) float units[3][kUnit ? 64 : 4];
    __shared__ Marks marks;
    __shared__ float scratch[TH / 64][2][DP];
    const wst_attention_desc& d = a.d;
    const int t = threadIdx.x, lane = t & 63, w = (t >> 6) & 3, half = t >> 8, hl = lane >> 5;
    const int group = d.q_heads / d.k_heads;
    const uint32_t cells = static_cast<uint32_t>(d.batch) * d.k_heads, slot = blockIdx.x % (cells * a.parts);
    const uint32_t bh = slot % cells, part = slot / cells;
    const int j0 = static_cast<int>(blockIdx.x / (cells * a.parts)) * kBQ;         // early keys are seen by most: first
    const int64_t b = bh / d.k_heads;
    const int kvh = static_cast<int>(bh % d.k_heads);
    const Scope sc(d, b);
    const Shape sh = Shape::of<T>(d, true, kFar<T, CAP>);
    const Kind kind = kind_of<CAP, BIAS>(d);
    const int j = j0 + w * 32 + (lane & 31), q_len = static_cast<int>(d.q_len);
    const bool exists = j < d.k_len, ok = j < sc.length && (!sc.k_doc || sc.k_doc[j] >= 0);
    const int kdoc = ok && sc.k_doc ? sc.k_doc[j] : -2;
    uint32_t kpos[kAxes];
#pragma unroll
    for (int x = 0; x < kAxes; ++x)
        kpos[x] = ok && sc.k_pos && x < sc.axes ? static_cast<uint32_t>(sc.k_pos[static_cast<int64_t>(j) * sc.axes + x]) + kPosBias : 0u;
    Frag<T> kf[DP / 16], vf[DP / 16];
    if constexpr (!kWide) {
        row_frags<T, DP>(at<T>(d.k, d.k_strides, b, ok ? j : 0, kvh), ok, d.dim, kf);
        row_frags<T, DP>(at<T>(d.v, d.v_strides, b, ok ? j : 0, kvh), ok, d.dim, vf);
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) dk[k] = dv[k] = zero16();

    // queries from `first` on may see one of the block's keys; keys past the length are seen by none
    const int nqt = (q_len + kRows - 1) / kRows, keys = min(sc.length - j0, kBQ);
    const int first = sc.causal && j0 >= sc.prefix ? max(j0 - sc.shift, 0) : 0;
    const int tile0 = first / kRows, tiles = keys > 0 ? nqt : 0;
    const bool marked = sc.q_doc != nullptr;
    if (marked && tile0 < tiles) scan_documents(marks, sc.k_doc, j0, kBQ, sc.length, sc.q_doc, tile0, tiles, q_len, TH / 64);
    if (marked || d.dim != DP || q_len % kRows || keys < kBQ) clear<sizeof(pool), TH>(pool, t);
    const int64_t qs = d.q_strides[1], ds = a.g.do_strides[1];
    Fetch<T, DP, kRows> qfetch, dfetch;
    qfetch.init(qs, d.dim, t);
    dfetch.init(ds, d.dim, t);

    // no pair needs a look when all rows and keys exist and the tile's first query sees the block's last key: from the
    // first such tile to the last whole one
    int full0 = tile0, full1 = keys == kBQ ? q_len / kRows : 0;
    if (sc.causal && j0 + kBQ > sc.prefix) full0 = max(tile0, (max(j0 + kBQ - 1 - sc.shift, 0) + kRows - 1) / kRows);
    const Walk walk{tile0, tiles, full0, max(full0, full1), marked};
    // Items of work: the full tiles of the first head, then of the next, ..., then the others. Parts take heads of their
    // own where that comes out even, so that the blocks of an XCD (blocks 8 apart) read the same queries at a time (8192
    // in order, 8 heads x 128 sharing 2: 560 -> 356 us; with cap and prefix 659 -> 442); what is left of the number of
    // parts takes every so many-th item.
    int g0 = 0, g1 = group, ahead = static_cast<int>(part), stride = a.parts;
    if (a.parts % group == 0) {
        g0 = ahead % group;
        g1 = g0 + 1;
        ahead /= group;
        stride /= group;
    } else if (group % a.parts == 0) {
        g0 = ahead * (group / a.parts);
        g1 = g0 + group / a.parts;
        ahead = 0;
        stride = 1;
    }
    struct Item {
        Step s;
        int g;
    };
    auto step = [&](Item x) {
        x.s.find(walk, marks);
        for (int k = 0; x.s.done(walk) && k < 2 * group; ++k) {       // bounded: there may be no tile at all
            if (x.g + 1 < g1) {
                ++x.g;
            } else if (!x.s.rest) {
                x.g = g0;
                x.s.rest = 1;
            } else {
                break;
            }
            x.s.tile = tile0 - 1;
            x.s.find(walk, marks);
        }
        return x;
    };
    auto skip = [&](Item x, int n) {
        for (int k = 0; k < n && !x.s.done(walk); ++k) x = step(x);
        return x;
    };
    float r_base = -INFINITY, r_delta = 0.f, r_unit = 1.f;
    int r_limit = 0, r_doc = -1, r_place = 0;
    uint32_t r_pos = 0;
    auto load = [&](Item x) {
        const int h = kvh * group + x.g, i = x.s.tile * kRows + (t & 63);
        const bool in = i < q_len;
        if (t < 64) {
            const int64_t row = (b * d.q_heads + h) * d.q_len + i;
            const float lse = in ? a.g.lse[row] : -INFINITY;
            r_limit = in ? sc.limit(i) : 0;
            r_doc = sc.q_doc && in ? sc.q_doc[i] : -1;
            if (sc.q_doc && r_doc < 0) r_limit = 0;
            r_base = lse == -INFINITY || r_limit <= 0 ? -INFINITY : sh.add - lse * kLog2e;
            r_delta = in ? -a.delta[row] : 0.f;
            if constexpr (kUnit) r_unit = in ? a.unit[row] : 1.f;
            r_place = i + sc.shift;
        }
        if (sc.q_pos) r_pos = (t >> 6) < sc.axes && in ? static_cast<uint32_t>(sc.q_pos[static_cast<int64_t>(i) * sc.axes + (t >> 6)]) + kPosBias : 0u;
    };
    auto put = [&](int n) {
        Rows& rw = rows[n];
        if (t < 64) {
            if constexpr (kUnit) units[n][t] = r_unit;
            rw.base[t] = r_base;
            rw.delta[t] = r_delta;
            rw.limit[t] = r_limit;
            rw.doc[t] = r_doc;
            rw.place[t] = r_place;
        }
        if (sc.q_pos && t < 64 * kAxes) rw.pos[t >> 6][t & 63] = r_pos;
    };
    auto fetch = [&](Item x, int buf, const Rows& with) {
        const int h = kvh * group + x.g, i = x.s.tile * kRows;
        const int* doc = marked ? with.doc : nullptr;
        const bool whole = d.dim == DP && q_len - i >= kRows && (!marked || marks.clean(x.s.tile - tile0));
        if (kWide && half) return;
        qfetch.issue(at<T>(d.q, d.q_strides, b, i, h), whole, q_len - i, doc, qt + buf * kTile, t);
        dfetch.issue(at<T>(a.g.d_o, a.g.do_strides, b, i, h), whole, q_len - i, doc, dt + buf * kTile, t);
    };
    if (marked) __syncthreads();       // the marks
    Item cur{{tile0 - 1, 0}, g0};
    if (tile0 < tiles) cur = skip(step(cur), ahead);
    else cur.s.tile = tiles;
    Item nxt = skip(cur, stride);
    if (!cur.s.done(walk)) {
        load(cur);
        put(0);
    }
    if (!nxt.s.done(walk)) {
        load(nxt);
        put(1);
    }
    __syncthreads();
    if (!cur.s.done(walk)) fetch(cur, 0, rows[0]);
    if constexpr (kWide) {
        // Only where a tile follows: its wait is the one for these loads too. A part without tiles (in order, the last
        // keys; documents that no query has) reads no key, and the sums below lie where the keys would land.
        if (!half && !cur.s.done(walk)) {
            Fetch<T, DP, kBQ> own;
            const bool whole = !marked && d.dim == DP && keys >= kBQ;
            own.init(d.k_strides[1], d.dim, t);
            own.issue(at<T>(d.k, d.k_strides, b, j0, kvh), whole, keys, marked ? sc.k_doc + j0 : nullptr, kt, t);
            own.init(d.v_strides[1], d.dim, t);
            own.issue(at<T>(d.v, d.v_strides, b, j0, kvh), whole, keys, marked ? sc.k_doc + j0 : nullptr, vt, t);
        }
    }
    const typename L::Lane lanes = L::lane();
    const int row_half = kWide ? 32 * __builtin_amdgcn_readfirstlane(half) : 0;      // this wave's first row of a tile
    int buf = 0, turn = 0;
    auto work = [&](auto mask) {
        constexpr int MASK = decltype(mask)::value;
        const int turn1 = turn == 2 ? 0 : turn + 1, turn2 = turn1 == 2 ? 0 : turn1 + 1;
        const float slope = kind.bias ? d.slopes[kvh * group + cur.g] : 0.f;
        const Rows& rw = rows[turn];
        const typename L::Lane qc = lanes.at_tile(qt + buf * kTile + row_half * L::kRowBytes);
        const typename L::Lane dc = lanes.at_tile(dt + buf * kTile + row_half * L::kRowBytes);
        arrived();
        __syncthreads();
        if (!nxt.s.done(walk)) fetch(nxt, buf ^ 1, rows[turn1]);
        const Item after = skip(nxt, stride);
        if (!after.s.done(walk)) load(after);
#pragma unroll
        for (int n = 0; n < (kWide ? 1 : 2); ++n) {
            f32x16 x = zero16(), dp, grad;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(&rw.delta[row_half + 32 * n + 8 * c + 4 * hl]);
#pragma unroll
                for (int e = 0; e < 4; ++e) dp[4 * c + e] = v[e];
            }
            if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
            if constexpr (kWide) {
                const typename L::Lane kc = lanes.at_tile(kt + 32 * w * L::kRowBytes), vc = lanes.at_tile(vt + 32 * w * L::kRowBytes);
                // one step's operands are read while the step before multiplies; said step by step, since with most
                // registers taken the compiler does not follow paced()
                Frag<T> f[2][4];
                auto read = [&](int c) {
                    f[c & 1][0] = L::row_frag(qc, 0, c);
                    f[c & 1][1] = L::row_frag(kc, 0, c);
                    f[c & 1][2] = L::row_frag(dc, 0, c);
                    f[c & 1][3] = L::row_frag(vc, 0, c);
                };
                read(0);
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    if (c + 1 < DP / 16) read(c + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    x = Mma<T>::mul(f[c & 1][0], f[c & 1][1], x);
                    dp = Mma<T>::mul(f[c & 1][2], f[c & 1][3], dp);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    x = Mma<T>::mul(L::row_frag(qc, 32 * n, c), kf[c], x);
                    dp = Mma<T>::mul(L::row_frag(dc, 32 * n, c), vf[c], dp);
                }
                if constexpr (sizeof(T) == 2) paced<DP / 8, 1, 6>();
            }
            if (kind.cap) sh.bend<T, true, kFar<T, CAP>>(x, grad);
            if (kind.bias) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int y = row_half + 32 * n + 8 * c + 4 * hl;
                    float f[4];
                    if (kind.coordinates) {
                        uint32_t sum[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int k = 0; k < kAxes; ++k) {
                            const u32x4 v = *reinterpret_cast<const u32x4*>(&rw.pos[k][y]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) sum[e] = away(kpos[k], v[e], sum[e]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[e] = static_cast<float>(sum[e]);
                    } else {
                        const i32x4 v = *reinterpret_cast<const i32x4*>(&rw.place[y]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[e] = fabsf(static_cast<float>(v[e] - j));
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[4 * c + e] = fmaf(-slope, f[e], x[4 * c + e] * sh.raw);
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(&rw.base[row_half + 32 * n + 8 * c + 4 * hl]);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * c + e] = __builtin_amdgcn_exp2f(fmaf(x[4 * c + e], sh.mul, v[e]));
                if constexpr (kUnit) {
                    const f32x4 u = *reinterpret_cast<const f32x4*>(&units[turn][row_half + 32 * n + 8 * c + 4 * hl]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[4 * c + e] *= u[e];
                }
            }
            if constexpr (MASK != 0) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int y = row_half + 32 * n + 8 * c + 4 * hl;
                    const i32x4 lim = *reinterpret_cast<const i32x4*>(&rw.limit[y]);
                    i32x4 doc;
                    if constexpr (MASK == 2) doc = *reinterpret_cast<const i32x4*>(&rw.doc[y]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        bool see = j < lim[e];
                        if constexpr (MASK == 2) see &= kdoc == doc[e];
                        x[4 * c + e] = see ? x[4 * c + e] : 0.f;
                        dp[4 * c + e] = see ? dp[4 * c + e] : 0.f;
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                x[r] *= kUp<T>;
                dp[r] *= x[r];
            }
            if (kind.cap) {
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] *= grad[r];
            }
            Frag<T> p[2], z[2];
            to_frags<T>(x, p);
            to_frags<T>(dp, z);
            if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
            if constexpr (kWide) {
                Frag<T> f[2][2];
                auto read = [&](int c) {
                    f[c & 1][0] = L::col_frag(dc, 16 * (c / (DP / 32)), c % (DP / 32));
                    f[c & 1][1] = L::col_frag(qc, 16 * (c / (DP / 32)), c % (DP / 32));
                };
                read(0);
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    if (c + 1 < DP / 16) read(c + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    const int k = c / (DP / 32), db = c % (DP / 32);
                    dv[db] = Mma<T>::mul(f[c & 1][0], p[k], dv[db]);
                    dk[db] = Mma<T>::mul(f[c & 1][1], z[k], dk[db]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) {
                        dv[db] = Mma<T>::mul(L::col_frag(dc, 32 * n + 16 * k, db), p[k], dv[db]);
                        dk[db] = Mma<T>::mul(L::col_frag(qc, 32 * n + 16 * k, db), z[k], dk[db]);
                    }
                if constexpr (sizeof(T) == 2) paced<DP / 8, 2, 4>();
            }
        }
        if (!after.s.done(walk)) put(turn2);
        cur = nxt;
        nxt = after;
        buf ^= 1;
        turn = turn1;
    };
    while (!cur.s.done(walk) && !cur.s.rest) work(std::integral_constant<int, 0>{});
    while (!cur.s.done(walk) && !marked) work(std::integral_constant<int, 1>{});
    while (!cur.s.done(walk)) work(std::integral_constant<int, 2>{});
    if constexpr (kWide) {             // the second four waves hand their sums over, a lane its own registers
        float* sums = reinterpret_cast<float*>(pool) + w * (DP * 64) + lane;
        static_assert(sizeof(pool) >= 4 * DP * 64 * sizeof(float), "room for the sums");
        arrived();                     // nothing may land in the pool any more
        __syncthreads();
        if (half) {
#pragma unroll
            for (int k = 0; k < DP / 32; ++k)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    sums[(32 * k + 2 * r) * 64] = dk[k][r];
                    sums[(32 * k + 2 * r + 1) * 64] = dv[k][r];
                }
        }
        __syncthreads();
        if (half) return;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                dk[k][r] += sums[(32 * k + 2 * r) * 64];
                dv[k][r] += sums[(32 * k + 2 * r + 1) * 64];
            }
    }
    const AttnArgs& z = again();
    const float up = 1.f / kUp<T>, mul = z.d.scale * up;
    if (z.parts > 1) {
        if (exists) {
            const int64_t row = ((static_cast<int64_t>(part) * z.d.batch + b) * z.d.k_heads + kvh) * z.d.k_len + j;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int x = 32 * db + 8 * g4 + 4 * hl;
                    if (x < z.d.dim) {
                        float u[4], v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            u[e] = dk[db][4 * g4 + e] * mul;
                            v[e] = dv[db][4 * g4 + e] * up;
                        }
                        store<4>(z.part + (2 * row) * z.d.dim + x, u);
                        store<4>(z.part + (2 * row + 1) * z.d.dim + x, v);
                    }
                }
        }
        return;
    }
    if (exists) {
        T* out_k = z.g.dk ? const_cast<T*>(at<T>(z.g.dk, z.g.dk_strides, b, j, kvh)) : nullptr;
        T* out_v = z.g.dv ? const_cast<T*>(at<T>(z.g.dv, z.g.dv_strides, b, j, kvh)) : nullptr;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int x = 32 * db + 8 * g4 + 4 * hl;
                if (x < z.d.dim) {
                    float u[4], v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        u[e] = dk[db][4 * g4 + e] * mul;
                        v[e] = dv[db][4 * g4 + e] * up;
                    }
                    if (out_k) store<4>(out_k + x, u);
                    if (out_v) store<4>(out_v + x, v);
                }
            }
    }
    uint64_t bad = __ballot(exists && (not_finite<T, DP>(dk) || not_finite<T, DP>(dv)));      // see k_attn_fwd
    for (bad = (bad | bad >> 32) & 0xffffffffu; bad; bad &= bad - 1) {
        __builtin_amdgcn_wave_barrier();
        row_dkv<T>(z, Scope(z.d, b), b, kvh, j0 + w * 32 + __builtin_ctzll(bad), scratch[w][0], scratch[w][1]);
    }
}

// dslopes[h] by one block: the partial sums of a head, added in a fixed order. s: a float a wave.
__device__ __forceinline__ void add_slopes(const AttnArgs& a, int h, float* s) {
    const int64_t count = a.d.batch * static_cast<int64_t>(a.slots);
    const float* p = a.slope_part + h * count;
    float v = 0.f;
    for (int64_t i = threadIdx.x; i < count; i += blockDim.x) v += p[i];
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t k = 1; k < blockDim.x / 64; ++k) v += s[k];
        a.g.dslopes[h] = v;
    }
}

// Adds the parts of a key's gradients, a wave a key; blocks behind those of the keys, one a head that shares the key head,
// add the slopes' partial sums, which saves a launch.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dkv_join(AttnArgs a) {
    __shared__ float scratch[4][2][kD];
    const wst_attention_desc& d = a.d;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t b = blockIdx.z, behind = static_cast<int64_t>(blockIdx.x) - (d.k_len + 3) / 4;
    const int kvh = blockIdx.y;
    if (behind >= 0) {
        if (b == 0) add_slopes(a, kvh * (d.q_heads / d.k_heads) + static_cast<int>(behind), &scratch[0][0][0]);
        return;
    }
    const int j = static_cast<int>(blockIdx.x) * 4 + w;
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
void launch_delta(const AttnArgs& a, hipStream_t st) {
    const dim3 rows(static_cast<unsigned>((a.d.q_len + 3) / 4), a.d.q_heads, static_cast<unsigned>(a.d.batch));
    k_attn_delta<T><<<rows, dim3(256), 0, st>>>(a);
}

// Launches through matrix instructions, for one element type and padded width (wst_attention_t.hip).
template <typename T, int DP>
__attribute__((visibility("hidden"))) void attend(const AttnArgs& a, const AttnPlan& p, hipStream_t st);
template <typename T, int DP>
__attribute__((visibility("hidden"))) void attend_backward(const AttnArgs& a, const AttnPlan& p, hipStream_t st);

}  // namespace wst_tok

#endif  // WST_ATTENTION_H
