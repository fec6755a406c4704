// The router's selection with softmax or sigmoid scores, a bias for balance and experts in groups (gfx950).
#include "dev_common.h"
#include "launchers.h"

namespace bf16n {
namespace dev {

namespace {

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        v = fmax(v, __shfl_xor(v, o, 64));
    }
    return v;
}
__device__ __forceinline__ double wave_add(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        v += __shfl_xor(v, o, 64);
    }
    return v;
}

// One wavefront to a token, expert lane + 64 q in its registers.
//   p_e = softmax(logits)_e or 1 / (1 + exp(-logit_e));  c_e = p_e + bias_e
// Groups are ranked by their largest c or the sum of their two largest, the first topk_groups stay open, and the k largest open
// c are taken, ties to the lower index.  Scores and sums are held in 64 bits: which of two near experts is larger must not
// hang on the order of 32-bit roundings.  A NaN logit has the score 0 and comes last, as -inf does; ids are always distinct
// experts of open groups, whatever the values.
template <int NQ>
__global__ void __launch_bounds__(256) k_router_grouped(const router_grouped_args a, int n_tok) {
    __shared__ double choice_lds[4][NQ * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int token = blockIdx.x * 4 + wave;
    if (token >= n_tok) {
        return;
    }
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
    if (a.topk_groups < a.n_groups) {
        double * c = choice_lds[wave];
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            c[lane + 64 * q] = choice[q];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); // the wavefront reads what its other lanes wrote
        __builtin_amdgcn_wave_barrier();
        const int size = a.n_experts / a.n_groups;
        double first = -INFINITY, second = -INFINITY;
        if (lane < a.n_groups) {
            for (int i = 0; i < size; i++) {
                const double v = c[lane * size + i];
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
        }
        double rank = a.top2 && size > 1 ? first + second : first;
        rank = rank == rank ? rank : -INFINITY;
        int before = 0;
        for (int g = 0; g < a.n_groups; g++) {
            const double v = __shfl(rank, g, 64);
            before += v > rank || (v == rank && g < lane);
        }
        const uint64_t kept = __ballot(lane < a.n_groups && before < a.topk_groups);
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const int e = lane + 64 * q;
            const bool is = e < a.n_experts && (kept >> (e / size) & 1);
            open[q] = __ballot(is);
            choice[q] = is ? choice[q] : -INFINITY;
        }
    }
    double mine = 0;
    int mine_id = 0;
    for (int j = 0; j < a.k; j++) {
        double best = choice[0];
#pragma unroll
        for (int q = 1; q < NQ; q++) {
            best = fmax(best, choice[q]);
        }
        best = wave_max(best);
        uint32_t id = 0;
#pragma unroll
        for (int q = NQ - 1; q >= 0; q--) {
            const uint64_t at = __ballot(choice[q] == best) & open[q];
            id = at ? 64 * q + (uint32_t) __builtin_ctzll(at) : id;
        }
        double s = 0;
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const bool here = (id >> 6) == (uint32_t) q;
            open[q] &= ~(here ? 1ull << (id & 63) : 0ull);
            s = here ? score[q] : s;
            choice[q] = (uint32_t) (lane + 64 * q) == id ? -INFINITY : choice[q];
        }
        s = __shfl(s, id & 63, 64);
        mine = lane == j ? s : mine; // k <= 64
        mine_id = lane == j ? (int) id : mine_id;
    }
    const double top = wave_add(lane < a.k ? mine : 0.0);
    if (lane < a.k) {
        a.ids[token * a.out_stride + lane] = mine_id;
        a.weights[token * a.out_stride + lane] = (float) ((a.renorm ? top > 0 ? mine / top : 0.0 : mine) * (double) a.scale);
    }
}

} // namespace

void launch_router_topk_grouped(const router_grouped_args & a, int n_tok, hipStream_t stream) {
    const int grid = (n_tok + 3) / 4;
    const int e = a.n_experts;
    (e <= 64 ? k_router_grouped<1> : e <= 128 ? k_router_grouped<2> : e <= 256 ? k_router_grouped<4> : e <= 512 ? k_router_grouped<8> : k_router_grouped<16>)
        <<<grid, 256, 0, stream>>>(a, n_tok);
}

} // namespace dev
} // namespace bf16n
