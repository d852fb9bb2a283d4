// The attention kernels of one element type: compiled once for each with -DWST_ATTN_TYPE=float, bf16 or f16.
#include "wst_attention.h"

namespace wst_tok {

template <typename T>
void attend(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    const wst_attention_desc& d = a.d;
    if (!p.tiles) {
        k_attn_rows<T><<<dim3(static_cast<unsigned>((d.q_len + 3) / 4), d.q_heads, static_cast<unsigned>(d.batch)), dim3(256), 0, st>>>(a);
        return;
    }
    with_width(d.dim, [&](auto w) {
        constexpr int DP = decltype(w)::value;
        if (p.splits) {
            const int64_t row_tiles = (d.q_heads / d.k_heads * d.q_len + 31) / 32;
            k_attn_split<T, DP><<<dim3(static_cast<unsigned>(p.splits * row_tiles * d.batch * d.k_heads)), dim3(256), 0, st>>>(a);
        } else {
            const int64_t blocks = d.batch * d.q_heads * ((d.q_len + kBQ - 1) / kBQ);
            k_attn_fwd<T, DP><<<dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st>>>(a);
        }
    });
    const int64_t rows = d.batch * d.q_heads * d.q_len;
    if (p.splits > 1) k_attn_join<T><<<dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, st>>>(a);
}

template <typename T>
void attend_backward(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    const wst_attention_desc& d = a.d;
    const bool want_q = a.g.dq || a.g.dslopes, want_k = a.g.dk || a.g.dv;
    const dim3 rows(static_cast<unsigned>((d.q_len + 3) / 4), d.q_heads, static_cast<unsigned>(d.batch));
    const dim3 keys(static_cast<unsigned>((d.k_len + 3) / 4), d.k_heads, static_cast<unsigned>(d.batch));
    if (!p.tiles || !want_q) k_attn_delta<T><<<rows, dim3(256), 0, st>>>(a);
    if (!p.tiles) {
        if (want_q) k_attn_dq_rows<T><<<rows, dim3(256), 0, st>>>(a);
        if (want_k) k_attn_dkv_rows<T><<<keys, dim3(256), 0, st>>>(a);
        return;
    }
    with_width(d.dim, [&](auto w) {
        constexpr int DP = decltype(w)::value;
        const int64_t q_blocks = d.batch * d.q_heads * ((d.q_len + kBQ - 1) / kBQ);
        const int64_t k_blocks = d.batch * d.k_heads * ((d.k_len + kBQ - 1) / kBQ);
        if (want_q) k_attn_dq<T, DP><<<dim3(static_cast<unsigned>(q_blocks)), dim3(256), 0, st>>>(a);   // and delta
        if (want_k) k_attn_dkv<T, DP><<<dim3(static_cast<unsigned>(k_blocks), p.parts), dim3(256), 0, st>>>(a);
    });
    if (p.parts > 1 && want_k) k_attn_dkv_join<T><<<keys, dim3(256), 0, st>>>(a);
}

template void attend<WST_ATTN_TYPE>(const AttnArgs&, const AttnPlan&, hipStream_t);
template void attend_backward<WST_ATTN_TYPE>(const AttnArgs&, const AttnPlan&, hipStream_t);

}  // namespace wst_tok
