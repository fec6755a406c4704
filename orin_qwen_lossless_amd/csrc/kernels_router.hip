// The router's selection with softmax or sigmoid scores, a bias for balance and experts in groups (gfx950).
#include "dev_common.h"
#include "launchers.h"

namespace bf16n {
namespace dev {

namespace {

// the same lanes' sums as wave_sum_dpp, in 64 bits; every lane gets the result
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double dpp_add64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int) u, CTRL, ROW_MASK, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int) (u >> 32), CTRL, ROW_MASK, 0xf, false);
    return v + __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
}
__device__ __forceinline__ double wave_add(double v) {
    v = dpp_add64<0xB1, 0xf>(v);
    v = dpp_add64<0x4E, 0xf>(v);
    v = dpp_add64<0x141, 0xf>(v);
    v = dpp_add64<0x140, 0xf>(v);
    v = dpp_add64<0x142, 0xa>(v);
    v = dpp_add64<0x143, 0xc>(v);
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int) u, 63), hi = __builtin_amdgcn_readlane((int) (u >> 32), 63);
    return __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, dpp_take<0xB1, 0xf>(v));
    v = max(v, dpp_take<0x4E, 0xf>(v));
    v = max(v, dpp_take<0x141, 0xf>(v));
    v = max(v, dpp_take<0x140, 0xf>(v));
    v = max(v, dpp_take<0x142, 0xa>(v));
    v = max(v, dpp_take<0x143, 0xc>(v));
    return __builtin_amdgcn_readlane((int) v, 63);
}
// an unsigned number in the values' order (zeros of either sign are one value; not for NaN); 0 is below all of them
__device__ __forceinline__ uint64_t order_of(double v) {
    const int64_t u = __builtin_bit_cast(int64_t, v + 0.0);
    return (uint64_t) (u < 0 ? ~u : u | INT64_MIN);
}

// One wavefront to a token, expert lane + 64 q in its registers.
//   p_e = softmax(logits)_e or 1 / (1 + exp(-logit_e));  c_e = p_e + bias_e
// Groups are ranked by their largest c or the sum of their two largest, the first topk_groups stay open, and the k largest open
// c are taken, ties to the lower index.  Scores and sums are held in 64 bits: which of two near experts is larger must not
// hang on the order of 32-bit roundings.  A NaN logit has the score 0 and comes last, as -inf does; ids are always distinct
// experts of open groups, whatever the values.
// A pick is a maximum over the lanes of the upper half of c as an ordered number, on the VALU alone; only where more than one expert
// has it do the lower halves decide, then the index, from the lanes' votes.  (With maxima of doubles through LDS one token of
// 256 experts took 7.8 us and 8192 tokens 24.8, now 5.8 and 16.9.)  Bound by the length of that chain for few tokens, by the
// exponentials' and the picks' instructions for many.
template <int NQ>
__global__ void __launch_bounds__(256) k_router_grouped(const router_grouped_args a, int n_tok) {
    constexpr int PLACES = NQ * 64 + 64; // group g begins g places later than its first expert: its lanes' reads find different banks
    __shared__ double lds[4][PLACES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int token = blockIdx.x * 4 + wave;
    if (token >= n_tok) {
        return;
    }
    double * const mine = lds[wave];
    const float * lg = a.logits + token * a.stride;
    double score[NQ], choice[NQ];
    uint64_t open[NQ]; // experts that may still be taken
    float logit[NQ], bias[NQ];
    float mx = -INFINITY;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const int e = lane + 64 * q;
        const bool in = e < a.n_experts;
        logit[q] = in ? lg[e] : -INFINITY;
        bias[q] = in && a.bias ? a.bias[e] : 0.f;
        logit[q] = logit[q] == logit[q] ? logit[q] : -INFINITY;
        mx = fmaxf(mx, logit[q]);
        open[q] = __ballot(in);
    }
    if (a.sigmoid) {
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            score[q] = 1.0 / (1.0 + exp(-(double) logit[q]));
        }
    } else {
        mx = lane63(wave_max_dpp(mx));
        double sum = 0;
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            score[q] = logit[q] == -INFINITY ? 0.0 : logit[q] == mx ? 1.0 : exp((double) logit[q] - (double) mx);
            sum += score[q];
        }
        sum = wave_add(sum);
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            score[q] = sum > 0 ? score[q] / sum : 0.0;
        }
    }
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const double c = logit[q] == -INFINITY ? -INFINITY : score[q] + (double) bias[q];
        choice[q] = c == c ? c : -INFINITY;
    }
    const auto lds_order = [] { // this wavefront's lanes read what others of them wrote
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    if (a.topk_groups < a.n_groups) {
        const int size = a.group_size;
        const auto group_of = [&](int e) { return (int) ((uint32_t) e * a.group_factor >> 21); };
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const int e = lane + 64 * q;
            if (e < a.n_experts) {
                mine[e + group_of(e)] = choice[q];
            }
        }
        lds_order();
        // `per` lanes look at a group, then join their largest two
        const int log2 = 31 - __builtin_clz(64 / a.n_groups), per = 1 << log2;
        const int g = lane >> log2;
        double first = -INFINITY, second = -INFINITY;
        if (g < a.n_groups) {
            for (int i = lane & (per - 1); i < size; i += per) {
                const double v = mine[g * size + g + i];
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
        }
        for (int o = 1; o < per; o <<= 1) {
            const double f = __shfl_xor(first, o, 64), s = __shfl_xor(second, o, 64);
            second = fmax(fmin(first, f), fmax(second, s));
            first = fmax(first, f);
        }
        double rank = a.top2 && size > 1 ? first + second : first;
        rank = rank == rank ? rank : -INFINITY;
        // a group's place: how many come before it
        const uint64_t r = order_of(rank);
        int before = 0;
        for (int i = 0; i < a.n_groups; i++) {
            const int at = i << log2;
            const uint32_t lo = __builtin_amdgcn_readlane((int) r, at), hi = __builtin_amdgcn_readlane((int) (r >> 32), at);
            const uint64_t v = (uint64_t) hi << 32 | lo;
            before += v > r || (v == r && i < g);
        }
        const uint64_t kept = __ballot(g < a.n_groups && before < a.topk_groups); // by lanes
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const int e = lane + 64 * q;
            open[q] = __ballot(e < a.n_experts && (kept >> (group_of(e) << log2) & 1));
        }
        lds_order();
    }
    uint32_t hi[NQ], lo[NQ]; // 0: not to be taken (any more)
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const uint64_t o = open[q] >> lane & 1 ? order_of(choice[q]) : 0;
        hi[q] = (uint32_t) (o >> 32);
        lo[q] = (uint32_t) o;
        mine[lane + 64 * q] = score[q];
    }
    lds_order();
    int mine_id = 0;
    for (int j = 0; j < a.k; j++) {
        uint32_t best = hi[0];
#pragma unroll
        for (int q = 1; q < NQ; q++) {
            best = max(best, hi[q]);
        }
        best = wave_max(best);
        uint64_t who[NQ];
        int n = 0;
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            who[q] = __ballot(hi[q] == best) & open[q];
            n += __popcll(who[q]);
        }
        if (n > 1) {
            uint32_t low = 0;
#pragma unroll
            for (int q = 0; q < NQ; q++) {
                low = max(low, hi[q] == best ? lo[q] : 0);
            }
            low = wave_max(low);
#pragma unroll
            for (int q = 0; q < NQ; q++) {
                who[q] &= __ballot(lo[q] == low);
            }
        }
        int id = 0;
#pragma unroll
        for (int q = NQ - 1; q >= 0; q--) {
            id = who[q] ? 64 * q + (int) __builtin_ctzll(who[q]) : id;
        }
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            open[q] &= ~((id >> 6) == q ? 1ull << (id & 63) : 0ull);
            hi[q] = lane + 64 * q == id ? 0 : hi[q];
        }
        mine_id = lane == j ? id : mine_id; // k <= 64
    }
    const double p = lane < a.k ? mine[mine_id] : 0.0;
    const double top = a.renorm ? wave_add(p) : 1.0;
    if (lane < a.k) {
        a.ids[token * a.out_stride + lane] = mine_id;
        a.weights[token * a.out_stride + lane] = (float) ((a.renorm ? top > 0 ? p / top : 0.0 : p) * (double) a.scale);
    }
}

} // namespace

void launch_router_topk_grouped(router_grouped_args a, int n_tok, hipStream_t stream) {
    a.group_size = a.n_experts / a.n_groups;
    a.group_factor = (uint32_t) (((1u << 21) + a.group_size - 1) / a.group_size); // e * factor >> 21 = e / group_size for all e < 1024
    const int grid = (n_tok + 3) / 4;
    const int e = a.n_experts;
    (e <= 64 ? k_router_grouped<1> : e <= 128 ? k_router_grouped<2> : e <= 256 ? k_router_grouped<4> : e <= 512 ? k_router_grouped<8> : k_router_grouped<16>)
        <<<grid, 256, 0, stream>>>(a, n_tok);
}

} // namespace dev
} // namespace bf16n
