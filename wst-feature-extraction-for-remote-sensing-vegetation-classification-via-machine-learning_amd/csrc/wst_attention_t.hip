// The attention kernels of one element type and one padded width of heads: compiled once for each with
// -DWST_ATTN_TYPE=float, bf16 or f16 and -DWST_ATTN_WIDTH=32, 64, 96 or 128.
#include "wst_attention.h"

namespace wst_tok {

// calls f(cap, bias) with the kinds of scores as constants (wst_attention.h, Kind)
template <typename T, typename F>
void with_kind(const wst_attention_desc& d, F f) {
    if constexpr (sizeof(T) == 4) {
        f(std::integral_constant<int, 2>{}, std::integral_constant<int, 3>{});
    } else {
        auto bias = [&](auto cap) {
            if (!d.slopes) f(cap, std::integral_constant<int, 0>{});
            else if (!d.q_pos) f(cap, std::integral_constant<int, 1>{});
            else f(cap, std::integral_constant<int, 2>{});
        };
        if (d.cap > kNearCap) f(std::integral_constant<int, 2>{}, std::integral_constant<int, 3>{});
        else if (d.cap > 0.f) bias(std::integral_constant<int, 1>{});
        else bias(std::integral_constant<int, 0>{});
    }
}

template <typename T, typename F>
void with_teams(const wst_attention_desc& d, F f) {
    if constexpr (sizeof(T) == 2) {
        if (two_teams(d)) return f(std::integral_constant<int, 2>{});
    }
    f(std::integral_constant<int, 1>{});
}

template <typename T, int DP>
void attend(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    const wst_attention_desc& d = a.d;
    with_kind<T>(d, [&](auto cap, auto bias) {
        constexpr int CAP = decltype(cap)::value, BIAS = decltype(bias)::value;
        if (p.splits) {
            const int64_t row_tiles = (d.q_heads / d.k_heads * d.q_len + 31) / 32;
            k_attn_split<T, DP, CAP, BIAS><<<dim3(static_cast<unsigned>(p.splits * row_tiles * d.batch * d.k_heads)), dim3(256), 0, st>>>(a);
        } else {
            const int64_t blocks = d.batch * d.q_heads * ((d.q_len + kBQ - 1) / kBQ);
            with_teams<T>(d, [&](auto teams) {
                constexpr int TEAMS = decltype(teams)::value;
                k_attn_fwd<T, DP, CAP, BIAS, TEAMS><<<dim3(static_cast<unsigned>(blocks)), dim3(256 * TEAMS), 0, st>>>(a);
            });
        }
    });
    const int64_t rows = d.batch * d.q_heads * d.q_len;
    if (p.splits > 1) k_attn_join<T><<<dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, st>>>(a);
}

template <typename T, int DP>
void attend_backward(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    const wst_attention_desc& d = a.d;
    // float32: what makes the weights add up to 1 comes from the walk over the keys too
    const bool want_q = a.g.dq || a.g.dslopes || a.unit, want_k = a.g.dk || a.g.dv;
    if (!want_q) launch_delta<T>(a, st);
    with_kind<T>(d, [&](auto cap, auto bias) {
        constexpr int CAP = decltype(cap)::value, BIAS = decltype(bias)::value;
        const int64_t q_blocks = d.batch * d.q_heads * ((d.q_len + kBQ - 1) / kBQ);
        const int64_t k_blocks = d.batch * d.k_heads * ((d.k_len + kBQ - 1) / kBQ);
        if (want_q)
            with_teams<T>(d, [&](auto teams) {
                constexpr int TEAMS = decltype(teams)::value;
                k_attn_dq<T, DP, CAP, BIAS, TEAMS><<<dim3(static_cast<unsigned>(q_blocks)), dim3(256 * TEAMS), 0, st>>>(a);   // and delta
            });
        if (want_k) k_attn_dkv<T, DP, CAP, BIAS><<<dim3(static_cast<unsigned>(k_blocks * p.parts)), dim3(dkv_threads(sizeof(T), DP)), 0, st>>>(a);
    });
    if (p.parts > 1 && want_k) {
        const int64_t behind = a.slope_part ? d.q_heads / d.k_heads : 0;
        const dim3 keys(static_cast<unsigned>((d.k_len + 3) / 4 + behind), d.k_heads, static_cast<unsigned>(d.batch));
        k_attn_dkv_join<T><<<keys, dim3(256), 0, st>>>(a);
    }
}

template void attend<WST_ATTN_TYPE, WST_ATTN_WIDTH>(const AttnArgs&, const AttnPlan&, hipStream_t);
template void attend_backward<WST_ATTN_TYPE, WST_ATTN_WIDTH>(const AttnArgs&, const AttnPlan&, hipStream_t);

}  // namespace wst_tok
