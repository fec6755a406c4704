// Products in 8-bit floating point with a scale for every block of 128, and what makes rows of that form (gfx950).
#include "dev_fp8.h"
#include "launch_dims.h"
#include "launchers.h"

#include <algorithm>
#include <string>
#include <type_traits>

namespace bf16n {
namespace dev {

namespace {

enum { CODES = BF16N_FP8_CODES, BF16 = BF16N_FP8_BF16, F32 = BF16N_FP8_F32 };

struct fp8_launch {
    const uint8_t * w, * up;                // codes
    const void * ws, * ups;                 // scales
    bool scales_bf16;
    int K, KB, nrows, NB;                   // columns and their blocks; rows of one matrix and their blocks
    int64_t n_matrices;
    const char * x; int64_t x_row;          // bytes
    const float * xs; int64_t xs_row, xs_block; // elements; of codes
    int x_kind;
    char * y; int64_t y_row;                // bytes
    float * ys; int64_t ys_row, ys_block;   // of codes
    int y_kind;
    int ncols;                              // dense columns, or (token, slot) pairs
    uint32_t per_token, one_per;            // the activation row of a pair is pair / per_token; 2^32 / per_token, rounded down
    const char * ids; int64_t ids_s0, ids_s1; bool ids_i64; int n_used; // one matrix per pair
    const int32_t * pairs, * bounds;        // pairs sorted by matrix
    int ksplit, lds_cols, cus, tiles;
    uint32_t one_block;                     // 2^32 / KB, rounded up: exact for the items of a pass (below 2^32 / KB)
};

__device__ __forceinline__ float scale_at(const void * s, bool bf16, int64_t i) {
    return bf16 ? bf16_bits_to_f32(((const uint16_t *) s)[i]) : ((const float *) s)[i];
}

__device__ __forceinline__ int row_of_pair(const fp8_launch & p, uint32_t pair) {
    const uint32_t t = __umulhi(pair, p.one_per); // at most one too few
    return (int) (t + (pair - t * p.per_token >= p.per_token));
}

// results 4 q .. 4 q + 3 of 16 of one column; rows behind the matrix are left out
template <int KIND>
__device__ __forceinline__ void store4(const fp8_launch & p, int64_t y_index, int row, f32x4_t v) {
    char * const at = p.y + y_index * p.y_row + (int64_t) row * (KIND == BF16 ? 2 : 4);
    if (row + 4 <= p.nrows && ((uintptr_t) at & (KIND == BF16 ? 7 : 15)) == 0) {
        if (KIND == BF16) {
            *(u32x2_t *) at = u32x2_t{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
        } else {
            *(f32x4_t *) at = v;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (row + e < p.nrows) {
            if (KIND == BF16) {
                ((uint16_t *) at)[e] = (uint16_t) bf16_pair(v[e], 0.f);
            } else {
                ((float *) at)[e] = v[e];
            }
        }
    }
}

// rows of zeros for pairs whose id names no matrix: rows from .. from + n of the results
__device__ __forceinline__ void zero_row(const fp8_launch & p, int64_t pair, int from, int n, int i, int step) {
    n = min(n, p.nrows - from);
    for (; i < n; i += step) {
        const int r = from + i;
        if (p.y_kind == F32) {
            ((float *) (p.y + pair * p.y_row))[r] = 0.f;
        } else if (p.y_kind == BF16) {
            ((uint16_t *) (p.y + pair * p.y_row))[r] = 0;
        } else {
            (p.y + pair * p.y_row)[r] = 0;
            if (r % FP8_BLOCK == 0) {
                p.ys[pair * p.ys_row + r / FP8_BLOCK * p.ys_block] = FP8_SMALLEST / FP8_LARGEST;
            }
        }
    }
}

__device__ __forceinline__ float gated(float g, float u) { return silu(g) * u; }

// ---------------------------------------------------------------- few columns

constexpr int FEW_PARTS = 64; // blocks of K that a wavefront takes at most: their scales are one register's lanes

// One wavefront takes 16 rows of the matrix at a time (of each of the two where they are gated) and its part of K; up to 16 CT columns are the
// other operand, from LDS, where the block has put their codes first (those of BF16 and FP32 rows it makes itself).  A lane's two
// loads of a step are 16 bytes each of row lane % 16, so that four lanes have half a line and both loads a whole one; weights go
// from memory to the operand's registers, D steps ahead, from one 16 rows on to the next.  K in ksplit parts, summed through LDS in a fixed order.
// 512 x 2048, one column: 4.5 us, a launch and the latency of its loads.
// ONE: 16 rows to a block and at most four steps of them to a wavefront, all loaded at once: no register is kept for the next 16 rows.
template <int CT, bool GLU, int XKIND, int NW, bool ONE>
__global__ void __launch_bounds__(NW * 64, ONE ? 2 : CT * (GLU ? 2 : 1) == 1 ? 4 : CT * (GLU ? 2 : 1) == 2 ? 3 : 2) k_fp8_few(const fp8_launch p) {
    constexpr int NM = GLU ? 2 : 1, D = GLU && !ONE ? 2 : 4;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, m16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int KB = p.KB, pitch = KB * FP8_BLOCK + 16;
    float * const lds_scales = (float *) (lds + p.lds_cols * pitch); // [lds_cols][KB]
    f32x4_t * const red = (f32x4_t *) (lds + (p.lds_cols * (pitch + KB * 4) + 15) / 16 * 16);

    int64_t matrix = 0;
    int begin = 0, end = p.ncols;
    const int ksplit = ONE ? NW : p.ksplit, groups = NW / ksplit, kp = wave % ksplit, group = wave / ksplit;
    const int row_step = gridDim.x * groups * 16;
    if (p.ids) {
        const int t = blockIdx.y / p.n_used, i = blockIdx.y % p.n_used;
        const char * at = p.ids + t * p.ids_s1 + i * p.ids_s0;
        matrix = p.ids_i64 ? *(const int64_t *) at : *(const int32_t *) at;
        begin = blockIdx.y;
        end = begin + 1;
        if (matrix < 0 || matrix >= p.n_matrices) {
            zero_row(p, blockIdx.y, 0, p.nrows, blockIdx.x * NW * 64 + threadIdx.x, gridDim.x * NW * 64);
            return;
        }
    }
    const auto x_of = [&](int c) -> int64_t { return p.ids ? row_of_pair(p, c) : c; };

    const int s0 = KB * kp / ksplit, steps = KB * (kp + 1) / ksplit - s0; // (at most FEW_PARTS)
    const bool cut = p.K % FP8_BLOCK != 0 && s0 + steps == KB;
    // the last block's chunks behind the matrix's last column: the row's first instead, taken as zeros (the columns' are zeros in LDS)
    const int last = (KB - 1) * FP8_BLOCK + q * 16;
    const bool out0 = cut && last >= p.K, out1 = cut && last + 64 >= p.K;

    const int pass = p.lds_cols;
    const auto column_of = [&](int i) { return KB == 1 ? i : (int) __umulhi((uint32_t) i, p.one_block); }; // i / KB
    for (int c0 = p.ids ? begin : blockIdx.y * pass; c0 < end; c0 += p.ids ? 1 : gridDim.y * pass) {
        const int nc = min(end - c0, pass);
        u32x4_t w[D][NM][2];
        const uint8_t * at[NM]; // the 16 rows whose loads are under way
        uint32_t off = 0;
        float sw[NM], sw_next[NM];
        const auto at_rows = [&](int r0) { // rows behind the matrix repeat its last: not stored
            const int row = min(r0, p.nrows - 1);
            off = min(m16, p.nrows - 1 - row) * p.K + q * 16;
#pragma unroll
            for (int m = 0; m < NM; m++) {
                at[m] = (m ? p.up : p.w) + (matrix * p.nrows + row) * p.K + s0 * FP8_BLOCK;
                sw_next[m] = scale_at(m ? p.ups : p.ws, p.scales_bf16, (matrix * p.NB + row / FP8_BLOCK) * KB + s0 + min(lane, steps - 1));
            }
        };
        const auto load = [&](int i, int u) {
            uint32_t k0 = off, k1 = off + 64;
            if (cut && i == steps - 1) {
                k0 -= out0 ? last : 0;
                k1 -= out1 ? last + 64 : 0;
            }
#pragma unroll
            for (int m = 0; m < NM; m++) {
                // (an offset of a chunk behind the last column goes back to column 0: added in 64 bits)
                w[u][m][0] = *(const u32x4_t *) (at[m] + i * FP8_BLOCK + (int64_t) (int32_t) k0);
                w[u][m][1] = *(const u32x4_t *) (at[m] + i * FP8_BLOCK + (int64_t) (int32_t) k1);
            }
        };
        const int first_row = (blockIdx.x * groups + group) * 16;
        at_rows(first_row);
#pragma unroll
        for (int u = 0; u < D; u++) {
            if (u < steps) {
                load(u, u);
            }
        }
        // Codes and scales of the columns, eight lanes to a block of 128 (with 16 the quotients and the maximum across them were twice as
        // much work to a block: 19 columns of 2576 in 91 blocks 12.1 us), several blocks' loads under way.
        __syncthreads();
        constexpr int AHEAD = (XKIND == F32 ? 2 : 4) / (CT == 1 && !ONE ? 2 : 1), GROUPS = NW * 8;
        const int items = nc * KB;
        for (int base = 0; base < items; base += GROUPS * AHEAD) {
            u32x4_t raw[AHEAD][XKIND == F32 ? 4 : XKIND == BF16 ? 2 : 1];
            float scale[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                if (base + j * GROUPS >= items) {
                    break;
                }
                const int i = min(base + j * GROUPS + (int) (threadIdx.x >> 3), items - 1), c = column_of(i), b = i - c * KB, k = b * FP8_BLOCK + (threadIdx.x & 7) * 16;
                const int64_t r = x_of(c0 + c);
#pragma unroll
                for (u32x4_t & v : raw[j]) {
                    v = u32x4_t{};
                }
                if (k < p.K) {
                    const char * const src = p.x + r * p.x_row + (int64_t) k * (XKIND == BF16 ? 2 : XKIND == F32 ? 4 : 1);
#pragma unroll
                    for (int e = 0; e < (int) (sizeof(raw[j]) / 16); e++) {
                        raw[j][e] = *(const u32x4_t *) (src + e * 16);
                    }
                }
                if (XKIND == CODES) {
                    scale[j] = p.xs[r * p.xs_row + b * p.xs_block];
                }
            }
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                if (base + j * GROUPS >= items) {
                    break;
                }
                const int i = min(base + j * GROUPS + (int) (threadIdx.x >> 3), items - 1), c = column_of(i), b = i - c * KB, k = b * FP8_BLOCK + (threadIdx.x & 7) * 16;
                u32x4_t codes = raw[j][0]; // (the last item's by several where the items end: the same ones)
                if constexpr (XKIND != CODES) {
                    float v[2][8];
                    if constexpr (XKIND == BF16) {
                        bf16x8_to_f32(raw[j][0], v[0]);
                        bf16x8_to_f32(raw[j][XKIND == BF16], v[1]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            v[e >> 3][e & 7] = __uint_as_float(raw[j][e >> 2][e & 3]);
                        }
                    }
                    const fp8_scales s = fp8_scales_of(eight_max_dpp(fmaxf(most_of8(v[0]), most_of8(v[1]))));
                    const u32x2_t lo = fp8_pack8(v[0], s.inverse), hi = fp8_pack8(v[1], s.inverse);
                    codes = u32x4_t{lo[0], lo[1], hi[0], hi[1]};
                    scale[j] = s.scale;
                }
                *(u32x4_t *) (lds + c * pitch + k) = codes;
                if ((threadIdx.x & 7) == 0) {
                    lds_scales[c * KB + b] = scale[j];
                }
            }
        }
        __syncthreads();

        const char * x_at[CT];
        const float * sx_at[CT];
#pragma unroll
        for (int t = 0; t < CT; t++) { // (columns behind the last repeat it: not stored)
            const int c = min(t * 16 + m16, nc - 1);
            x_at[t] = lds + c * pitch + s0 * FP8_BLOCK + q * 16;
            sx_at[t] = lds_scales + c * KB + s0;
        }
        for (int r0 = first_row; r0 < p.nrows + group * 16; r0 += row_step) { // (the block's wavefronts make the same rounds)
#pragma unroll
            for (int m = 0; m < NM; m++) {
                sw[m] = sw_next[m];
            }
            f32x4_t acc[NM][CT] = {};
            const bool more = !ONE && r0 + row_step < p.nrows + group * 16;
            for (int base = 0; base < (ONE ? 1 : steps); base += D) {
#pragma unroll
                for (int u = 0; u < D; u++) {
                    const int i = base + u;
                    if (i >= steps) {
                        break;
                    }
                    if (cut && i == steps - 1) {
#pragma unroll
                        for (int m = 0; m < NM; m++) {
                            w[u][m][0] = out0 ? u32x4_t{} : w[u][m][0];
                            w[u][m][1] = out1 ? u32x4_t{} : w[u][m][1];
                        }
                    }
                    fp8_wide ww[NM];
#pragma unroll
                    for (int m = 0; m < NM; m++) {
                        ww[m] = fp8_widen(w[u][m][0], w[u][m][1]);
                    }
                    if (!ONE && i + D < steps) {
                        load(i + D, u);
                    }
#pragma unroll
                    for (int t = 0; t < CT; t++) {
                        const fp8_wide xw = fp8_widen(*(const u32x4_t *) (x_at[t] + i * FP8_BLOCK), *(const u32x4_t *) (x_at[t] + i * FP8_BLOCK + 64));
                        const float sx = sx_at[t][i];
#pragma unroll
                        for (int m = 0; m < NM; m++) {
                            const f32x4_t part = fp8_sum16(ww[m], xw);
                            const float both = __uint_as_float((uint32_t) __builtin_amdgcn_readlane((int) __float_as_uint(sw[m]), i)) * sx;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                acc[m][t][e] = fmaf(part[e], both, acc[m][t][e]);
                            }
                        }
                    }
                }
            }
            if (more) {
                at_rows(r0 + row_step);
#pragma unroll
                for (int u = 0; u < D; u++) {
                    if (u < steps) {
                        load(u, u);
                    }
                }
            }
            if (ksplit > 1) {
                __syncthreads();
#pragma unroll
                for (int m = 0; m < NM; m++) {
#pragma unroll
                    for (int t = 0; t < CT; t++) {
                        red[((wave * NM + m) * CT + t) * 64 + lane] = acc[m][t];
                    }
                }
                __syncthreads();
                if (kp != 0) {
                    continue;
                }
                for (int i = 1; i < ksplit; i++) {
#pragma unroll
                    for (int m = 0; m < NM; m++) {
#pragma unroll
                        for (int t = 0; t < CT; t++) {
                            acc[m][t] += red[(((wave + i) * NM + m) * CT + t) * 64 + lane];
                        }
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < CT; t++) {
                const int c = t * 16 + m16;
                if (c >= nc) {
                    continue;
                }
                f32x4_t v = acc[0][t];
                if (GLU) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        v[e] = gated(v[e], acc[NM - 1][t][e]);
                    }
                }
                if (p.y_kind == BF16) {
                    store4<BF16>(p, c0 + c, r0 + 4 * q, v);
                } else {
                    store4<F32>(p, c0 + c, r0 + 4 * q, v);
                }
            }
        }
    }
}

// The second products of a token's experts and their weighted sum in one launch, for few tokens (a launch of one token's slots and one of
// their sum: 2048 x 512, eight slots 5.5 + 4.0 us; this 6.4): a block takes 16 rows of a token's result, a wavefront the slots wave, wave + 8 ..,
// and the sum is made in the order of the slots, one fmaf each (bf16n_moe_combine's).  Hidden rows: FP32, made codes by the block.
__global__ void __launch_bounds__(512, 4) k_fp8_down(const fp8_launch p, const void * wts, bool wts_bf16) {
    constexpr int NW = 8, D = 4;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, m16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int KB = p.KB, slots = p.n_used, token = blockIdx.y, row0 = blockIdx.x * 16;
    const fp8_down_lds in = fp8_down_layout(slots, KB);
    const int pitch = in.pitch;
    float * const lds_scales = (float *) (lds + in.scales);  // [slots][KB]
    float * const res = (float *) (lds + in.results);        // [slots][16]
    const bool cut = p.K % FP8_BLOCK != 0;
    const int last = (KB - 1) * FP8_BLOCK + q * 16;
    const bool out0 = cut && last >= p.K, out1 = cut && last + 64 >= p.K;
    const int64_t row_off = (int64_t) min(m16, p.nrows - 1 - row0) * p.K + q * 16;

    u32x4_t w[D][2];
    float sw = 0.f;
    const uint8_t * at = p.w;
    const auto matrix_of = [&](int slot) -> int64_t {
        const char * id = p.ids + token * p.ids_s1 + slot * p.ids_s0;
        const int64_t m = p.ids_i64 ? *(const int64_t *) id : *(const int32_t *) id;
        return m >= 0 && m < p.n_matrices ? m : -1;
    };
    const auto load = [&](int s, int u) {
        const bool end = cut && s == KB - 1;
        const int64_t k = (int64_t) s * FP8_BLOCK;
        w[u][0] = *(const u32x4_t *) (at + row_off + (end && out0 ? -q * 16 : k));
        w[u][1] = *(const u32x4_t *) (at + row_off + (end && out1 ? -q * 16 : k + 64));
    };
    const auto begin = [&](int64_t matrix) {
        at = p.w + (matrix * p.nrows + row0) * p.K;
        sw = scale_at(p.ws, p.scales_bf16, (matrix * p.NB + row0 / FP8_BLOCK) * KB + min(lane, KB - 1));
#pragma unroll
        for (int u = 0; u < D; u++) {
            if (u < KB) {
                load(u, u);
            }
        }
    };
    int64_t matrix = wave < slots ? matrix_of(wave) : -1;
    if (matrix >= 0) {
        begin(matrix);
    }
    for (int i = threadIdx.x >> 4; i < slots * KB; i += NW * 4) {
        const int c = i / KB, b = i - c * KB, k = b * FP8_BLOCK + (threadIdx.x & 15) * 8;
        float v[8] = {};
        if (k < p.K) {
            const char * src = p.x + ((int64_t) token * slots + c) * p.x_row + (int64_t) k * 4;
            const f32x4_t lo = *(const f32x4_t *) src, hi = *(const f32x4_t *) (src + 16);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[e] = e < 4 ? lo[e & 3] : hi[e & 3];
            }
        }
        const fp8_scales s = fp8_scales_of(row_max_dpp(most_of8(v)));
        *(u32x2_t *) (lds + c * pitch + k) = fp8_pack8(v, s.inverse);
        if ((threadIdx.x & 15) == 0) {
            lds_scales[c * KB + b] = s.scale;
        }
    }
    __syncthreads();
    for (int slot = wave; slot < slots; slot += NW) {
        f32x4_t acc = {};
        if (matrix >= 0) {
            const char * const x_at = lds + slot * pitch + q * 16;
            for (int base = 0; base < KB; base += D) {
#pragma unroll
                for (int u = 0; u < D; u++) {
                    const int s = base + u;
                    if (s >= KB) {
                        break;
                    }
                    if (cut && s == KB - 1) {
                        w[u][0] = out0 ? u32x4_t{} : w[u][0];
                        w[u][1] = out1 ? u32x4_t{} : w[u][1];
                    }
                    const fp8_wide ww = fp8_widen(w[u][0], w[u][1]);
                    if (s + D < KB) {
                        load(s + D, u);
                    }
                    const fp8_wide xw = fp8_widen(*(const u32x4_t *) (x_at + s * FP8_BLOCK), *(const u32x4_t *) (x_at + s * FP8_BLOCK + 64));
                    const float both = __uint_as_float((uint32_t) __builtin_amdgcn_readlane((int) __float_as_uint(sw), s)) * lds_scales[slot * KB + s];
                    const f32x4_t part = fp8_sum16(ww, xw);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        acc[e] = fmaf(part[e], both, acc[e]);
                    }
                }
            }
        }
        if (m16 == 0) {
            *(f32x4_t *) (res + slot * 16 + 4 * q) = acc;
        }
        matrix = slot + NW < slots ? matrix_of(slot + NW) : -1;
        if (matrix >= 0) {
            begin(matrix);
        }
    }
    __syncthreads();
    const int r = row0 + threadIdx.x;
    if (threadIdx.x < 16 && r < p.nrows) {
        float acc = 0.f;
        for (int i = 0; i < slots; i++) {
            acc = fmaf(scale_at(wts, wts_bf16, (int64_t) token * slots + i), res[i * 16 + threadIdx.x], acc);
        }
        store_y(p.y + token * p.y_row, p.y_kind == BF16, r, acc);
    }
}

// ---------------------------------------------------------------- many columns

__device__ __align__(16) const uint32_t g_zeros[4] = {0, 0, 0, 0};

// rows of columns' codes that the threads copy at least, eight threads to a row
__host__ __device__ constexpr int many_x_rows(int cols, int threads) { return (cols * 8 + threads - 1) / threads * (threads / 8); }
// LDS of a step: the rows of both sides and the columns' scales (of 64 columns at least)
__host__ __device__ constexpr int many_stage(int a_rows, int cols, int threads) {
    return (a_rows + many_x_rows(cols, threads)) * FP8_BLOCK + (cols < 64 ? 64 : cols) * 4;
}

// vector memory operations under way: at most N, and no read of LDS
template <int N> __device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14); }
// a barrier that waits for nothing by itself (__syncthreads also waits for every load, those of later steps among them)
__device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// the sum over this lane and those below it
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int dpp_below(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xf, false); }
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_below<0x111, 0xf>(v); // row_shr 1, 2, 4, 8
    v = dpp_below<0x112, 0xf>(v);
    v = dpp_below<0x114, 0xf>(v);
    v = dpp_below<0x118, 0xf>(v);
    v = dpp_below<0x142, 0xa>(v); // row_bcast 15, 31
    return dpp_below<0x143, 0xc>(v);
}

constexpr int LIST_GROUP = 4;

// The columns of pass `pass` of all lists, `cols` to a pass: every wavefront looks for itself, eight lists to a lane, 512 at a time.  matrix: -1 if
// there are fewer passes.
struct list_pass { int matrix, begin, end; };
__device__ __forceinline__ list_pass find_pass(const int32_t * bounds, int n_matrices, int pass, int cols) {
    constexpr int PER = 8;
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int m0 = 0; m0 <= n_matrices; m0 += 64 * PER) { // (n_matrices: the pairs that name none)
        int b[PER + 1], mine = 0;
#pragma unroll
        for (int i = 0; i <= PER; i++) {
            b[i] = bounds[min(m0 + lane * PER + i, n_matrices + 1)];
        }
#pragma unroll
        for (int i = 0; i < PER; i++) {
            mine += (b[i + 1] - b[i] + cols - 1) / cols;
        }
        const int upto = before + wave_scan(mine);
        const uint64_t behind = __ballot(upto > pass);
        if (behind) {
            const int owner = __builtin_ctzll(behind);
            int left = pass - (upto - mine), matrix = 0, begin = 0, end = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int n = (b[i + 1] - b[i] + cols - 1) / cols;
                if (left >= 0 && left < n) {
                    matrix = m0 + lane * PER + i;
                    begin = b[i] + left * cols;
                    end = min(b[i + 1], begin + cols);
                }
                left -= n;
            }
            return {__builtin_amdgcn_readlane(matrix, owner), __builtin_amdgcn_readlane(begin, owner), __builtin_amdgcn_readlane(end, owner)};
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return {-1, 0, 0};
}

// WR x WC wavefronts, RT x CT results of 16 x 16 to each.  Codes of both sides go straight into LDS, S - 1 steps of 128 columns ahead:
// rows of 128 bytes, their eight places of 16 bytes exchanged by the row's low bits so that the operands' reads find every
// bank.  A step's products start from zero and are added to the results times their scales, those of a row of tiles while the next row's
// are under way.  BF16 results are summed by the instruction
// on the codes.  FP32 ones are summed from BF16 operands (fp8_sum16), and so are those that become codes with a scale, which a value
// 1.5e-5 off would put on the other side of a border now and then (0.0015 of the norm of 300 rows of 1408 that are 0.0003 off so).
// OUT codes: the results of ROWS = 128 rows leave as codes with a scale.
// Lists: a block to 64 columns of one matrix, every pass a block of its own.  Gate and up: the scales of the columns in registers, so that two blocks'
// stages are the whole of a CU's LDS (one block with 128 columns that took a list's passes in turn: 2048 tokens of 256 experts of 512 x 2048 190 us,
// 512 tokens 128; now 145 and 104).  Down, whose K is short: two row tiles to a block, the second's copies under the first's last products (2048 tokens,
// one / two / four: 110, 105, 107 with FP32 results, 98, 93, 102 with BF16 ones).
template <int WR, int WC, int RT, int CT, int S, bool GLU, bool LIST, int OUT>
__global__ void __launch_bounds__(WR * WC * 64, 2) k_fp8_many(const fp8_launch p) {
    constexpr bool WIDE = OUT != BF16, SX_REGS = LIST && GLU, TILES = LIST && !GLU;
    static_assert(!TILES || S == 2, "a step ahead");
    constexpr int NM = GLU ? 2 : 1, THREADS = WR * WC * 64, A_ROWS = WR * RT * 16, ROWS = A_ROWS / NM, COLS = WC * CT * 16, TM = RT / NM;
    constexpr int SCALES = (A_ROWS + many_x_rows(COLS, THREADS)) * FP8_BLOCK, STAGE = SX_REGS ? (A_ROWS + COLS) * FP8_BLOCK : many_stage(A_ROWS, COLS, THREADS), A_COPIES = A_ROWS * 8 / THREADS, B_COPIES = (COLS * 8 + THREADS - 1) / THREADS;
    static_assert(A_COPIES * THREADS == A_ROWS * 8, "whole copies");
    static_assert(FP8_BLOCK % (TM * 16) == 0, "a wavefront's rows have one scale");
    static_assert(OUT != CODES || ROWS == FP8_BLOCK, "a block of rows has one scale");
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, m16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % WR, wc = wave / WR;
    int64_t matrix = 0;
    int begin = 0, end = p.ncols, row_tile;
    if (LIST) {
        // An XCD takes every eighth block: LIST_GROUP passes in a row of the same rows are one XCD's, whose L2 then has the rows of a list's
        // later passes (gate and up of 2048 tokens of 256 experts 152 us without, 145 so; with 2, 8, 16 148, 146, 147).
        const int row_tiles = ((p.nrows + ROWS - 1) / ROWS + p.tiles - 1) / p.tiles;
        const int64_t id = (int64_t) blockIdx.y * gridDim.x + blockIdx.x, slot = id >> 3, item = slot / LIST_GROUP * 8 + (id & 7);
        row_tile = (int) (item % row_tiles) * p.tiles;
        const list_pass f = find_pass(p.bounds, (int) p.n_matrices, (int) (item / row_tiles * LIST_GROUP + slot % LIST_GROUP), COLS);
        if (f.matrix < 0) {
            return;
        }
        matrix = f.matrix;
        begin = f.begin;
        end = f.end;
    } else {
        // An XCD takes every eighth block, which is made a contiguous part of the tiles here: WIDEST column tiles of one row tile
        // after the other, more of them where they are the smaller, so that what runs there at a time shares few pieces of either side
        // (gated, BF16 results, us with four everywhere: 2048 x 2048, 128 columns 13.8 for 10.9; 1408 x 2048, 600 16.4 for 15.7).
        const int row_tiles = (p.nrows + ROWS - 1) / ROWS, col_tiles = (p.ncols + COLS - 1) / COLS;
        const int n = row_tiles * col_tiles, per = (n + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
        if ((int) (blockIdx.x >> 3) >= per || id >= n) {
            return;
        }
        constexpr int WIDEST = A_ROWS <= COLS ? 4 : A_ROWS <= 2 * COLS ? 6 : A_ROWS <= 4 * COLS ? 8 : A_ROWS <= 8 * COLS ? 12 : 24;
        const int group = id / (row_tiles * WIDEST), in = id - group * row_tiles * WIDEST, wide = min(WIDEST, col_tiles - group * WIDEST);
        row_tile = in / wide;
        begin = (group * WIDEST + in % wide) * COLS;
        end = min(end, begin + COLS);
    }
    const int row0 = row_tile * ROWS, KB = p.KB;
    const int n_tiles = TILES ? min(p.tiles, (p.nrows + ROWS - 1) / ROWS - row_tile) : 1, n_steps = n_tiles * KB;
    const bool cut = p.K % FP8_BLOCK != 0;

    // what this thread copies: a place of rows (threadIdx.x >> 3) + i * THREADS / 8, chunk by the row's low bits
    const int chunk = (threadIdx.x & 7) ^ ((threadIdx.x >> 3) & 7);
    uint32_t a_off[A_COPIES];
    const auto of_up = [&](int i) { return GLU && (i * (THREADS / 8) + wave * 8) / 16 % RT >= TM; };
#pragma unroll
    for (int i = 0; i < A_COPIES; i++) {
        const int r = i * (THREADS / 8) + (threadIdx.x >> 3), t = r / 16;
        a_off[i] = min((t / RT * TM + t % RT % TM) * 16 + r % 16, p.nrows - 1 - row0) * p.K + chunk * 16;
    }
    const int wave_row = row0 + wr * TM * 16;
    const int frag0 = m16 * FP8_BLOCK + ((q ^ (m16 & 7)) << 4), frag1 = frag0 ^ 64;
    const int a_frag = wr * RT * 16 * FP8_BLOCK, b_frag = A_ROWS * FP8_BLOCK + wc * 16 * FP8_BLOCK;

    if (LIST && matrix == p.n_matrices) {
        for (int c = begin; c < end; c++) {
            zero_row(p, p.pairs[c], row0, n_tiles * ROWS, threadIdx.x, THREADS);
        }
        return;
    }
    const uint8_t * const w_base = p.w + (matrix * p.nrows + row0) * p.K, * const up_base = p.up + (matrix * p.nrows + row0) * p.K;
    const int64_t scale_row = (matrix * p.NB + min(wave_row, p.nrows - 1) / FP8_BLOCK) * KB;
    const int c0 = begin, nc = end - begin;
    const auto x_of = [&](int i) -> int64_t { return LIST ? row_of_pair(p, p.pairs[c0 + min(i, nc - 1)]) : c0 + min(i, nc - 1); };
    const char * b_at[B_COPIES];
#pragma unroll
    for (int i = 0; i < B_COPIES; i++) {
        b_at[i] = p.x + x_of(i * (THREADS / 8) + (threadIdx.x >> 3)) * p.x_row + chunk * 16;
    }
    const float * const sx_at = p.xs + x_of(threadIdx.x % COLS) * p.xs_row;
    const float * sxr_at[CT];
    if constexpr (SX_REGS) {
#pragma unroll
        for (int c = 0; c < CT; c++) {
            sxr_at[c] = p.xs + x_of((c * WC + wc) * 16 + m16) * p.xs_row;
        }
    }
    f32x4_t acc[RT][CT] = {};
    const auto store = [&](auto columns, int tile) {
        if constexpr (OUT != CODES) {
#pragma unroll
            for (int c = 0; c < decltype(columns)::value; c++) {
                const int col = (c * WC + wc) * 16 + m16;
                if (col >= nc) {
                    continue;
                }
                const int64_t y = LIST ? p.pairs[c0 + col] : c0 + col;
#pragma unroll
                for (int t = 0; t < TM; t++) {
                    store4<OUT>(p, y, wave_row + tile * ROWS + t * 16 + 4 * q, acc[t][c]);
                }
            }
        }
    };
    // M: tiles of 16 columns to a wavefront, one loop for each number of them (with a branch around a tile's products the compiler puts
    // their sums behind the branches, where on some ways too few cycles pass between a product and the read of its result)
    const auto steps = [&](auto columns) {
        constexpr int M = decltype(columns)::value, BM = (M * WC * 16 * 8 + THREADS - 1) / THREADS, COPIES = A_COPIES + BM + (SX_REGS ? M : 1); // of a step
        float sx_next[SX_REGS ? M : 1];
        static_assert((S - 2) * COPIES < 64, "what the counter of loads can tell apart");
        int v_copy = 0, s_copy = 0; // what is copied next, of all steps and of the tile's
        int64_t tile_copy = 0;
        const auto copy = [&] {
            char * const to = lds + v_copy % S * STAGE + wave * 1024;
            const int s = s_copy;
            const int64_t k = s * FP8_BLOCK;
            const uint8_t * const wk = w_base + tile_copy + k, * const uk = up_base + k;
            if (cut && s == KB - 1) { // chunks behind the last column are zeros on both sides
                const bool none = s * FP8_BLOCK + chunk * 16 >= p.K;
#pragma unroll
                for (int i = 0; i < A_COPIES; i++) {
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *) (none ? (const uint8_t *) g_zeros : (of_up(i) ? uk : wk) + a_off[i]),
                                                     (__attribute__((address_space(3))) void *) (to + i * THREADS * 16), 16, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < BM; i++) {
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *) (none ? (const char *) g_zeros : b_at[i] + k),
                                                     (__attribute__((address_space(3))) void *) (to + A_ROWS * FP8_BLOCK + i * THREADS * 16), 16, 0, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < A_COPIES; i++) {
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *) ((of_up(i) ? uk : wk) + a_off[i]),
                                                     (__attribute__((address_space(3))) void *) (to + i * THREADS * 16), 16, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < BM; i++) {
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *) (b_at[i] + k),
                                                     (__attribute__((address_space(3))) void *) (to + A_ROWS * FP8_BLOCK + i * THREADS * 16), 16, 0, 0);
                }
            }
            // the columns' scales, 64 to a wavefront (the same ones by several where there are fewer)
            if constexpr (!SX_REGS) {
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *) (sx_at + s * p.xs_block),
                                                 (__attribute__((address_space(3))) void *) (lds + v_copy % S * STAGE + SCALES + wave * 64 % COLS * 4), 4, 0, 0);
            } else {
#pragma unroll
                for (int c = 0; c < M; c++) {
                    sx_next[c] = sxr_at[c][s * p.xs_block];
                }
            }
            v_copy++;
            s_copy++;
            if (TILES && s_copy == KB) {
                s_copy = 0;
                tile_copy += (int64_t) ROWS * p.K;
            }
        };
        // 64 steps' scales of the wavefront's rows, one to a lane; waited for here: a wait at their use, in the loop, would be one for every
        // copy under way
        float sw[NM];
        const auto load_scales = [&](int s) {
#pragma unroll
            for (int m = 0; m < NM; m++) {
                sw[m] = scale_at(m ? p.ups : p.ws, p.scales_bf16, scale_row + min(s + lane, n_steps - 1));
                asm volatile("" : "+v"(sw[m]));
            }
        };
#pragma unroll
        for (int s = 0; s < S - 1; s++) {
            if (s < n_steps) {
                copy();
            }
        }
        int s_tile = 0, tile = 0;
        for (int s64 = 0; s64 < n_steps; s64 += 64) {
            load_scales(s64);
            const int s_end = min(s64 + 64, n_steps);
            for (int s = s64; s < s_end; s++) {
                // this wavefront's copies of the step are in LDS; those of up to S - 2 later ones are under way
                if (S > 3 && s + 2 < n_steps) {
                    wait_loads<(S > 3 ? 2 : 0) * COPIES>();
                } else if (S > 2 && s + 1 < n_steps) {
                    wait_loads<(S > 2 ? 1 : 0) * COPIES>();
                } else {
                    wait_loads<0>();
                }
                float sx_now[M];
                if constexpr (SX_REGS) {
#pragma unroll
                    for (int c = 0; c < M; c++) {
                        asm volatile("" : "+v"(sx_next[c]));
                        sx_now[c] = sx_next[c];
                    }
                }
                meet(); // all of the block's are, and nothing reads the buffer of the step before any more
                if (v_copy < n_steps) {
                    copy();
                }
                const char * const at = lds + s % S * STAGE;
                float both[NM][M];
#pragma unroll
                for (int c = 0; c < M; c++) {
                    const float sx = SX_REGS ? sx_now[c] : *(const float *) (at + SCALES + ((c * WC + wc) * 16 + m16) * 4);
#pragma unroll
                    for (int m = 0; m < NM; m++) {
                        both[m][c] = __uint_as_float((uint32_t) __builtin_amdgcn_readlane((int) __float_as_uint(sw[m]), s - s64)) * sx;
                    }
                }
                u32x4_t b[M][2], a[WIDE ? RT : 2][2];
                fp8_wide bw[M];
#pragma unroll
                for (int c = 0; c < M; c++) {
                    b[c][0] = *(const u32x4_t *) (at + b_frag + c * WC * 16 * FP8_BLOCK + frag0);
                    b[c][1] = *(const u32x4_t *) (at + b_frag + c * WC * 16 * FP8_BLOCK + frag1);
                }
#pragma unroll
                for (int t = 0; t < (WIDE ? RT : 1); t++) {
                    a[t][0] = *(const u32x4_t *) (at + a_frag + t * 16 * FP8_BLOCK + frag0);
                    a[t][1] = *(const u32x4_t *) (at + a_frag + t * 16 * FP8_BLOCK + frag1);
                }
                if constexpr (WIDE) { // (else the compiler puts every read right ahead of its use: 300 columns of 1408 x 2048, gated, 16.2 us for 15.3)
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int c = 0; c < M; c++) {
                        bw[c] = fp8_widen(b[c][0], b[c][1]);
                    }
                }
                f32x4_t part[2][M];
#pragma unroll
                for (int t = 0; t <= RT; t++) {
                    fp8_wide aw;
                    if (t < RT) {
                        if (!WIDE && t + 1 < RT) {
                            a[(t + 1) & 1][0] = *(const u32x4_t *) (at + a_frag + (t + 1) * 16 * FP8_BLOCK + frag0);
                            a[(t + 1) & 1][1] = *(const u32x4_t *) (at + a_frag + (t + 1) * 16 * FP8_BLOCK + frag1);
                        }
                        if constexpr (WIDE) {
                            aw = fp8_widen(a[t][0], a[t][1]);
                        }
                    }
#pragma unroll
                    for (int c = 0; c < M; c++) {
                        if (t < RT) {
                            if constexpr (WIDE) {
                                part[t & 1][c] = fp8_sum16(aw, bw[c]);
                            } else {
                                part[t & 1][c] = fp8_sum8(a[t & 1][0], a[t & 1][1], b[c][0], b[c][1]);
                            }
                        }
                        if (t > 0) {
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                acc[t - 1][c][e] = fmaf(part[(t - 1) & 1][c][e], both[(t - 1) / TM][c], acc[t - 1][c][e]);
                            }
                        }
                    }
                }
                if constexpr (!WIDE) { // in this order: a product, the additions of one a row of tiles before
#pragma unroll
                    for (int t = 0; t < RT; t++) {
#pragma unroll
                        for (int c = 0; c < M; c++) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            if (t > 0) {
                                __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                            }
                            if (c == 0 && t + 1 < RT) {
                                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                            }
                        }
                    }
                }
                if (TILES && ++s_tile == KB) {
                    store(columns, tile);
#pragma unroll
                    for (int t = 0; t < RT; t++) {
#pragma unroll
                        for (int c = 0; c < M; c++) {
                            acc[t][c] = f32x4_t{};
                        }
                    }
                    s_tile = 0;
                    tile++;
                }
            }
        }
    };
    if constexpr (LIST) { // (the lowest number that has them all: one for the block)
        const int tiles = ((nc + 15) / 16 + WC - 1) / WC;
        static_assert(CT == 4 || CT == 2, "one loop each");
        if constexpr (CT == 4) {
            tiles == 1 ? steps(std::integral_constant<int, 1>{}) : tiles == 2 ? steps(std::integral_constant<int, 2>{})
            : tiles == 3 ? steps(std::integral_constant<int, 3>{}) : steps(std::integral_constant<int, 4>{});
        } else {
            tiles == 1 ? steps(std::integral_constant<int, 1>{}) : steps(std::integral_constant<int, 2>{});
        }
    } else {
        steps(std::integral_constant<int, CT>{});
    }
    if (GLU) {
#pragma unroll
        for (int t = 0; t < TM; t++) {
#pragma unroll
            for (int c = 0; c < CT; c++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    acc[t][c][e] = gated(acc[t][c][e], acc[RT - TM + t][c][e]);
                }
            }
        }
    }
    if constexpr (OUT == CODES) {
        float * const most = (float *) lds; // [WR][COLS]
        float mine[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) {
            float v = 0.f;
#pragma unroll
            for (int t = 0; t < TM; t++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v = fmaxf(v, wave_row + t * 16 + 4 * q + e < p.nrows ? fabsf(acc[t][c][e]) : 0.f);
                }
            }
            v = fmaxf(v, __shfl_xor(v, 16, 64));
            mine[c] = fmaxf(v, __shfl_xor(v, 32, 64));
        }
        __syncthreads();
        if (q == 0) {
#pragma unroll
            for (int c = 0; c < CT; c++) {
                most[wr * COLS + (c * WC + wc) * 16 + m16] = mine[c];
            }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const int col = (c * WC + wc) * 16 + m16;
            if (col >= nc) {
                continue;
            }
            float v = most[col];
#pragma unroll
            for (int i = 1; i < WR; i++) {
                v = fmaxf(v, most[i * COLS + col]);
            }
            const fp8_scales s = fp8_scales_of(v);
            const int64_t y = LIST ? p.pairs[c0 + col] : c0 + col;
            if (wr == 0 && q == 0) {
                p.ys[y * p.ys_row + row_tile * p.ys_block] = s.scale;
            }
#pragma unroll
            for (int t = 0; t < TM; t++) {
                const int r = wave_row + t * 16 + 4 * q;
                if (r < p.nrows) { // (rows are a multiple of 16)
                    *(uint32_t *) (p.y + y * p.y_row + r) = fp8_pack4(acc[t][c][0] * s.inverse, acc[t][c][1] * s.inverse, acc[t][c][2] * s.inverse, acc[t][c][3] * s.inverse);
                }
            }
        }
    } else if constexpr (!TILES) {
        store(std::integral_constant<int, CT>{}, 0);
    }
}

// ---------------------------------------------------------------- rows in 8 bits

// A block of 128 values to 16 lanes.
template <int KIND>
__global__ void __launch_bounds__(256) k_fp8_rows(const char * x, int64_t x_row, uint8_t * y, int64_t y_row, float * s, int64_t s_row, int64_t s_block, int64_t rows, int K) {
    const int KB = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    for (int64_t i = (int64_t) blockIdx.x * 16 + (threadIdx.x >> 4); i < rows * KB; i += (int64_t) gridDim.x * 16) {
        const int64_t r = i / KB;
        const int b = (int) (i - r * KB), k = b * FP8_BLOCK + (threadIdx.x & 15) * 8;
        float v[8] = {};
        if (k < K) {
            const char * src = x + r * x_row + (int64_t) k * (KIND == BF16 ? 2 : 4);
            if (KIND == BF16) {
                bf16x8_to_f32(*(const u32x4_t *) src, v);
            } else {
                const f32x4_t a = *(const f32x4_t *) src, d = *(const f32x4_t *) (src + 16);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    v[j] = j < 4 ? a[j & 3] : d[j & 3];
                }
            }
        }
        const fp8_scales q = fp8_scales_of(row_max_dpp(most_of8(v)));
        if (k < K) {
            *(u32x2_t *) (y + r * y_row + k) = fp8_pack8(v, q.inverse);
        }
        if ((threadIdx.x & 15) == 0) {
            s[r * s_row + b * s_block] = q.scale;
        }
    }
}

__device__ __forceinline__ u32x4_t to_bf16x8(const float (&v)[8]) {
    return u32x4_t{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
}

// The glue of a decode step (bf16n_add_rmsnorm) with its norm in 8 bits: a block to a token, C pieces of eight elements to a thread, 16 threads to
// a block of 128, eight slots' rows on the way at a time (one after the other: 333 tokens of 2576 with eight slots 10.9 us).  A row stays
// in registers between the sum of its squares and its codes.  Every sum and the norm are held in 64 bits and become
// FP32 once, ahead of the scales: a code is off by a whole step, a sixteenth of its value, wherever an error of a last place carries a value over the
// middle of two codes, which 32 bits did to one or two of 858 thousand (and were 8.9 us there for 9.3).
// 8192 tokens of 2048: 21.1 us, 118 MB at 5.6 TB/s (two inputs in turn; three 22.5); one token 2.4, the chain of its loads, sum and scale.
template <int C, bool SLOTS>
__global__ void __launch_bounds__(1024) k_add_rmsnorm_fp8(const add_norm_args p, uint8_t * y, int64_t y_row, float * s, int64_t s_row, int64_t s_block) {
    __shared__ double wave_sq[16];
    __shared__ float wsm[SLOTS ? 1024 : 1];
    const int64_t tok = blockIdx.x, base = tok * p.n;
    const int threads = blockDim.x;
    if (SLOTS) {
        for (int i = threadIdx.x; i < p.n_used; i += threads) {
            const int64_t at = tok * p.n_used + i;
            wsm[i] = p.wts_bf16 ? bf16_bits_to_f32(((const uint16_t *) p.wts)[at]) : ((const float *) p.wts)[at];
        }
        __syncthreads();
    }
    double v[C][8];
    double sq = 0;
    u32x4_t gamma[C];
#pragma unroll
    for (int j = 0; j < C; j++) {
        const int i0 = (j * threads + threadIdx.x) * 8;
        u32x4_t a = {}, b = {}, c = {};
        gamma[j] = u32x4_t{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u}; // ones
        double acc[8] = {};
        if (i0 < p.n) {
            a = *(const u32x4_t *) (p.a + base + i0);
            if (p.b) {
                b = *(const u32x4_t *) (p.b + base + i0);
            }
            if (p.c) {
                c = *(const u32x4_t *) (p.c + base + i0);
            }
            if (p.gamma) {
                gamma[j] = *(const u32x4_t *) (p.gamma + i0);
            }
            if (SLOTS) {
                const float * row = p.ys + (tok * p.n_used) * p.n + i0;
                constexpr int WAY = C == 1 ? 8 : 4; // (registers)
                for (int k0 = 0; k0 < p.n_used; k0 += WAY) {
                    f32x4_t lo[WAY], hi[WAY];
#pragma unroll
                    for (int k = 0; k < WAY; k++) { // (a slot past the last: the last row again, unused)
                        const float * at = row + (int64_t) min(k0 + k, p.n_used - 1) * p.n;
                        lo[k] = *(const f32x4_t *) at;
                        hi[k] = *(const f32x4_t *) (at + 4);
                    }
#pragma unroll
                    for (int k = 0; k < WAY; k++) {
                        if (k0 + k < p.n_used) {
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                acc[e] = fma((double) wsm[k0 + k], (double) (e < 4 ? lo[k][e & 3] : hi[k][e & 3]), acc[e]);
                            }
                        }
                    }
                }
            }
        }
        float fa[8], fb[8], fc[8];
        bf16x8_to_f32(a, fa);
        bf16x8_to_f32(b, fb);
        bf16x8_to_f32(c, fc);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[j][e] = (double) fa[e] + (double) fb[e];
        }
        if (p.c) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[j][e] += (double) fc[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (SLOTS) {
                v[j][e] += acc[e];
            }
            sq = fma(v[j][e], v[j][e], sq);
        }
    }
    sq = wave_sum64(sq);
    if ((threadIdx.x & 63) == 0) {
        wave_sq[threadIdx.x >> 6] = sq;
    }
    __syncthreads();
    double total = 0;
    for (int i = 0; i < threads >> 6; i++) {
        total += wave_sq[i];
    }
    const double scale = 1.0 / sqrt(total / (double) p.n + (double) p.eps);
#pragma unroll
    for (int j = 0; j < C; j++) {
        const int i0 = (j * threads + threadIdx.x) * 8;
        const bool in = i0 < p.n;
        float g[8], y32[8];
        if (in && p.y_sum) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y32[e] = (float) v[j][e];
                asm("" : "+v"(y32[e])); // (else the two roundings become one from 64 bits to BF16, six instructions an element: 8192 x 2048 1.2 us)
            }
            *(u32x4_t *) (p.y_sum + base + i0) = to_bf16x8(y32);
        }
        bf16x8_to_f32(gamma[j], g);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            y32[e] = (float) (v[j][e] * scale * (double) g[e]);
        }
        if (in && p.y_norm) {
            *(u32x4_t *) (p.y_norm + base + i0) = to_bf16x8(y32);
        }
        const fp8_scales q = fp8_scales_of(row_max_dpp(most_of8(y32)));
        if (in) {
            *(u32x2_t *) (y + tok * y_row + i0) = fp8_pack8(y32, q.inverse);
            if ((threadIdx.x & 15) == 0) {
                s[tok * s_row + i0 / FP8_BLOCK * s_block] = q.scale;
            }
        }
    }
}

// y[t] = sum over the slots of w[t, k] * ys[t, k] for rows in FP32, slots in order, one fmaf each; n a multiple of 8.  For results that are not at 16-byte
// places: k_moe_combine, which takes them too, has one element of a row to a thread (2048 tokens, eight slots of 2048: 58 us, this 40, 3.4 TB/s).
__global__ void __launch_bounds__(256) k_fp8_combine(const float * ys, const void * w, bool w_bf16, char * y, bool y_bf16, int n_used, int64_t n) {
    const int64_t t = blockIdx.y, i = ((int64_t) blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= n) {
        return;
    }
    float acc[8] = {};
    for (int k = 0; k < n_used; k++) {
        const int64_t s = t * n_used + k;
        const float wk = scale_at(w, w_bf16, s);
        const f32x4_t lo = __builtin_nontemporal_load((const f32x4_t *) (ys + s * n + i)), hi = __builtin_nontemporal_load((const f32x4_t *) (ys + s * n + i + 4));
#pragma unroll
        for (int e = 0; e < 8; e++) {
            acc[e] = fmaf(wk, e < 4 ? lo[e & 3] : hi[e & 3], acc[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        store_y(y + t * n * (y_bf16 ? 2 : 4), y_bf16, i + e, acc[e]);
    }
}

// ---------------------------------------------------------------- launches

fp8_launch launch_of(const fp8_product & a, int cus) {
    fp8_launch p = {};
    const bf16n_fp8_weight & w = *a.w;
    p.w = w.codes; p.ws = w.scales; p.scales_bf16 = w.scales_bf16 != 0;
    if (a.up) {
        p.up = a.up->codes; p.ups = a.up->scales;
    }
    p.K = (int) w.K; p.KB = (int) ((w.K + FP8_BLOCK - 1) / FP8_BLOCK);
    p.n_matrices = w.n_matrices;
    p.nrows = (int) (w.rows / w.n_matrices); p.NB = (p.nrows + FP8_BLOCK - 1) / FP8_BLOCK;
    p.x = (const char *) a.x.at; p.x_row = a.x.row; p.xs = a.x.scales; p.xs_row = a.x.scale_row; p.xs_block = a.x.scale_block; p.x_kind = a.x.kind;
    p.y = (char *) a.y.at; p.y_row = a.y.row; p.ys = a.y.scales; p.ys_row = a.y.scale_row; p.ys_block = a.y.scale_block; p.y_kind = a.y.kind;
    p.ncols = (int) a.n_cols;
    p.per_token = (uint32_t) a.per_token; p.one_per = (uint32_t) std::min<uint64_t>(~0u, (1ull << 32) / a.per_token);
    p.ids = (const char *) a.ids; p.ids_i64 = a.ids_i64; p.ids_s0 = a.ids_s0; p.ids_s1 = a.ids_s1; p.n_used = a.n_used;
    p.pairs = a.pairs; p.bounds = a.bounds;
    p.cus = cus;
    p.one_block = (uint32_t) (((1ull << 32) + p.KB - 1) / p.KB);
    return p;
}

constexpr size_t FEW_LDS = 160 * 1024 - 1024;

// a kernel instance's template arguments (bf16n_last_kernel)
std::string text_of(std::initializer_list<int> numbers) {
    std::string s;
    for (const int n : numbers) {
        s += (s.empty() ? "" : ", ") + std::to_string(n);
    }
    return s;
}

// without p: the LDS limit is raised
template <int CT, bool GLU, int XKIND, int NW, bool ONE>
void few_go(const fp8_launch * p, dim3 grid, size_t lds, hipStream_t stream) {
    const auto kernel = k_fp8_few<CT, GLU, XKIND, NW, ONE>;
    if (!p) {
        (void) hipFuncSetAttribute((const void *) kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int) FEW_LDS);
        return;
    }
    static const std::string text = text_of({CT, GLU, XKIND, NW, ONE});
    note_kernel("k_fp8_few", text.c_str(), 0);
    kernel<<<grid, NW * 64, lds, stream>>>(*p);
}

size_t few_lds(int cols, int KB, int ct, bool glu, int nw, int ksplit) {
    return ((size_t) cols * (KB * FP8_BLOCK + 16 + KB * 4) + 15) / 16 * 16 + (ksplit > 1 ? (size_t) nw * (glu ? 2 : 1) * ct * 1024 : 0);
}

enum { FEW_ONE, FEW_EIGHT, FEW_FOUR }; // all at once; eight wavefronts; four
// without p: every instance's limit is raised
void few_instance(const fp8_launch * p, int ct, bool glu, int shape, dim3 grid, size_t lds, hipStream_t stream) {
    const auto by_kind = [&](auto c, auto g, auto n, auto one) {
        constexpr int CT = decltype(c)::value, NW = decltype(n)::value;
        constexpr bool GLU = decltype(g)::value, ONE = decltype(one)::value;
        if (!p || p->x_kind == CODES) {
            few_go<CT, GLU, CODES, NW, ONE>(p, grid, lds, stream);
        }
        if (!p || p->x_kind == BF16) {
            few_go<CT, GLU, BF16, NW, ONE>(p, grid, lds, stream);
        }
        if (!p || p->x_kind == F32) {
            few_go<CT, GLU, F32, NW, ONE>(p, grid, lds, stream);
        }
    };
    const auto by_shape = [&](auto c, auto g) {
        if (!p || shape == FEW_ONE) {
            by_kind(c, g, std::integral_constant<int, 8>{}, std::true_type{});
        }
        if (!p || shape == FEW_EIGHT) {
            by_kind(c, g, std::integral_constant<int, 8>{}, std::false_type{});
        }
        if constexpr (decltype(c)::value == 1) { // (single pairs)
            if (!p || shape == FEW_FOUR) {
                by_kind(c, g, std::integral_constant<int, 4>{}, std::false_type{});
            }
        }
    };
    const auto by_ct = [&](auto g) {
        if (!p || ct == 1) {
            by_shape(std::integral_constant<int, 1>{}, g);
        }
        if (!p || ct == 2) {
            by_shape(std::integral_constant<int, 2>{}, g);
        }
    };
    if (!p || glu) {
        by_ct(std::true_type{});
    }
    if (!p || !glu) {
        by_ct(std::false_type{});
    }
}

// cols: columns of a pass; busy: matrices or passes that have columns; blocks: of them all, grid.y
void run_few(fp8_launch p, bool glu, int cols, int64_t busy, int y_blocks, int cus, hipStream_t stream) {
    const int64_t tiles = (p.nrows + 15) / 16 * busy;
    const int ct = cols <= 16 ? 1 : 2, nw = ct == 2 || tiles <= 4 * cus ? 8 : 4; // (four: single pairs, many of them)
    int ksplit = nw == 8 ? 8 : tiles <= 16 * cus ? 4 : 1;
    while (ksplit > 1 && p.KB < ksplit) {
        ksplit /= 2;
    }
    while ((p.KB + ksplit - 1) / ksplit > FEW_PARTS) {
        ksplit *= 2;
    }
    p.ksplit = ksplit;
    p.lds_cols = cols;
    const int rows = nw / ksplit * 16, n_blocks = (p.nrows + rows - 1) / rows;
    const size_t lds = few_lds(cols, p.KB, ct, glu, nw, ksplit);
    if (ksplit == 8 && tiles <= 2 * cus && p.KB <= 32) { // (else 512 x 2048, one column 6.7 us for 4.5; 1453 x 2576, 19 columns 10.2 for 8.4)
        few_instance(&p, ct, glu, FEW_ONE, dim3(n_blocks, y_blocks), lds, stream);
        return;
    }
    const int room = cus * (int) std::min<size_t>(nw == 8 ? 2 : 4, LDS_BYTES / lds);
    const int rounds = (int) std::max<int64_t>(1, std::min<int64_t>(8, (int64_t) n_blocks * busy / room));
    few_instance(&p, ct, glu, nw == 8 ? FEW_EIGHT : FEW_FOUR, dim3((n_blocks + rounds - 1) / rounds, y_blocks), lds, stream);
}

// columns of a pass of k_fp8_few: as many as are there, 32 at most, and what LDS holds
int few_pass(int64_t cols, int KB, bool glu) {
    int n = (int) std::min<int64_t>(cols, 32);
    while (n > 1 && few_lds(n, KB, n <= 16 ? 1 : 2, glu, 8, 8) > FEW_LDS) {
        n--;
    }
    return n;
}

template <int WR, int WC, int RT, int CT, int S, bool GLU, bool LIST, int OUT>
void many_go(const fp8_launch * p, hipStream_t stream) { // without p: its LDS limit is raised
    constexpr int ROWS = WR * RT * 16 / (GLU ? 2 : 1), COLS = WC * CT * 16, LDS = S * (LIST && GLU ? (WR * RT * 16 + COLS) * FP8_BLOCK : many_stage(WR * RT * 16, COLS, WR * WC * 64));
    static_assert((size_t) LDS <= LDS_BYTES, "fits");
    const auto kernel = k_fp8_many<WR, WC, RT, CT, S, GLU, LIST, OUT>;
    if (!p) {
        (void) hipFuncSetAttribute((const void *) kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        return;
    }
    const int row_tiles = (p->nrows + ROWS - 1) / ROWS, col_tiles = (p->ncols + COLS - 1) / COLS;
    fp8_launch q = *p;
    q.tiles = LIST && !GLU && p->nrows % ROWS == 0 ? 2 : 1;
    dim3 grid((unsigned) (((int64_t) row_tiles * col_tiles + 7) / 8 * 8));
    if (LIST) {
        const int64_t passes = p->n_matrices + 1 + p->ncols / COLS; // at most
        const int64_t items = (passes + LIST_GROUP - 1) / LIST_GROUP * ((row_tiles + q.tiles - 1) / q.tiles), blocks = (items + 7) / 8 * 8 * LIST_GROUP;
        grid.x = (unsigned) std::min<int64_t>(blocks, 1 << 20);
        grid.y = (unsigned) ((blocks + grid.x - 1) / grid.x);
    }
    static const std::string text = text_of({WR, WC, RT, CT, S, GLU, LIST, OUT});
    note_kernel("k_fp8_many", text.c_str(), 0);
    kernel<<<grid, WR * WC * 64, LDS, stream>>>(q);
}

template <int WR, int WC, int RT, int CT, int S, bool GLU, bool LIST>
void many_kinds(const fp8_launch * p, int y_kind, hipStream_t stream) {
    if constexpr (GLU) {
        if (!p || y_kind == CODES) {
            many_go<WR, WC, RT, CT, S, GLU, LIST, CODES>(p, stream);
        }
    }
    if (!p || y_kind == BF16) {
        many_go<WR, WC, RT, CT, S, GLU, LIST, BF16>(p, stream);
    }
    if (!p || y_kind == F32) {
        many_go<WR, WC, RT, CT, S, GLU, LIST, F32>(p, stream);
    }
}

// Tiles to choose from, and what a step of 128 columns of K takes, us: of one block to a CU, and of each where the CUs are full of them.  Here and in
// run_many: calls behind one another on two inputs in turn (on three 8192 x 2048 by 8192 columns, 152, takes 173: they pass the caches, and power holds the clock).
struct tile_of { int rows, cols; float alone, full; };
// the tile whose steps take least: those of one block or of the rounds that the tiles make
int best_tile(const tile_of * tiles, int n, const fp8_launch & p) {
    int best = 0;
    float least = 0;
    for (int i = 0; i < n; i++) {
        const int64_t blocks = (int64_t) ((p.nrows + tiles[i].rows - 1) / tiles[i].rows) * ((p.ncols + tiles[i].cols - 1) / tiles[i].cols);
        const float t = std::max(tiles[i].alone, (float) ((blocks + p.cus - 1) / p.cus) * tiles[i].full);
        if (i == 0 || t < least) {
            least = t;
            best = i;
        }
    }
    return best;
}

// without p: every instance's limit is raised
void run_many(const fp8_launch * p, bool glu, bool list, hipStream_t stream) {
    const int kind = p ? p->y_kind : 0;
#define MANY(WHEN, N, ...) if (!p || ((WHEN) && best == N)) { many_kinds<__VA_ARGS__>(p, kind, stream); }
#define MANY_ONE(WHEN, N, ...) if (!p || ((WHEN) && best == N)) { many_go<__VA_ARGS__>(p, stream); }
    int best = 0;
    if (p && list) {
        best = 0;
    } else if (p && glu && kind == CODES) { // ( us in this order: 1408 x 2048, 300 columns 34, 23, 17, 15; 2048 x 2048, 2048 columns 39, 47, 47, 67)
        const tile_of tiles[] = {{128, 128, 2.0f, 2.05f}, {128, 64, 1.4f, 1.45f}, {128, 32, 1.1f, 0.75f}, {128, 16, 0.85f, 0.54f}};
        best = best_tile(tiles, 4, *p);
    } else if (p && glu && p->ncols <= 16) { // (BF16 / FP32 results with 64 x 16 and 128 x 16: 12288 x 2048, 8 columns 10.8 / 11.4 us, 15.3 / 15.6; 65536 x 2048, 4 54.7 / 55.3, 51.3 / 47.7)
        best = (p->nrows + 63) / 64 <= 2 * p->cus ? 6 : 3;
    } else if (p && glu) {
        // (128 x 128, 64 x 64, 32 x 64, 128 x 16, us: BF16 results 1408 x 2048, 300 columns 22, 11.8, 9.9, 13.6; 2048 x 2048, 2048 24, 28, 33, 53; FP32 33, 15.6, 12.6, 15.4 and 38, 40, 46, 65)
        const tile_of bf16[] = {{128, 128, 1.2f, 1.45f}, {64, 64, 0.6f, 0.43f}, {32, 64, 0.47f, 0.26f}}, f32[] = {{128, 128, 2.0f, 2.2f}, {64, 64, 0.83f, 0.63f}, {32, 64, 0.62f, 0.38f}};
        const int of[] = {0, 5, 4};
        best = of[best_tile(kind == BF16 ? bf16 : f32, 3, *p)];
    } else if (p && p->ncols <= 16) {
        // (Us of 64 x 64 tiles, 128 x 16, 64 x 16, one column: BF16 results 20480 x 2048 11.0, 9.2, 9.9, 16384 x 8192 29, 27, 21; FP32 248320 x 2048 101, 86, 87, 16384 x 8192 43, 31, 26.)
        best = (p->nrows + 63) / 64 <= p->cus ? 9 : 8;
    } else if (p && kind == BF16) {
        // (5120 x 2048, us in this order: 128 columns 33, 16, 11, 9.1; 1024: 39, 23, 21, 22; 2048: 40, 36, 32, 41; 8192 x 2048, 8192: 152, 171, 189, 235;
        // the last two, 64 columns 9.4, 7.6; 150 10.0, 9.3; 300 11.4, 15.6)
        const tile_of tiles[] = {{256, 256, 2.0f, 2.0f}, {128, 128, 0.95f, 0.685f}, {128, 64, 0.62f, 0.387f}, {64, 64, 0.45f, 0.238f}, {32, 64, 0.33f, 0.22f}};
        best = best_tile(tiles, 5, *p);
    } else if (p) { // (5120 x 2048, us in this order: 64 columns 29, 15, 10.5; 2048: 65, 50, 56; 8192 x 2048, 8192: 264, 293, 336; the last two, 64 columns 11.1, 9.3; 150 11.6, 12.6)
        const tile_of tiles[] = {{256, 128, 2.0f, 2.05f}, {128, 64, 0.88f, 0.6f}, {64, 64, 0.62f, 0.33f}, {32, 64, 0.51f, 0.32f}};
        best = best_tile(tiles, 4, *p);
    }
    MANY(glu && list, 0, 4, 1, 4, 4, 2, true, true)
    MANY(!glu && list, 0, 2, 2, 4, 2, 2, false, true)
    MANY(glu && !list, 0, 4, 2, 4, 4, 2, true, false)
    MANY_ONE(glu && !list && kind == CODES, 1, 4, 2, 4, 2, 2, true, false, CODES)
    MANY_ONE(glu && !list && kind == CODES, 2, 4, 1, 4, 2, 2, true, false, CODES)
    MANY(glu && !list, 3, 4, 1, 4, 1, 2, true, false)
    MANY_ONE(glu && !list && kind == BF16, 4, 2, 2, 2, 2, 3, true, false, BF16)
    MANY_ONE(glu && !list && kind == F32, 4, 2, 2, 2, 2, 3, true, false, F32)
    MANY_ONE(glu && !list && kind == BF16, 5, 2, 2, 4, 2, 2, true, false, BF16)
    MANY_ONE(glu && !list && kind == F32, 5, 2, 2, 4, 2, 2, true, false, F32)
    MANY_ONE(glu && !list && kind == BF16, 6, 4, 1, 2, 1, 3, true, false, BF16)
    MANY_ONE(glu && !list && kind == F32, 6, 4, 1, 2, 1, 3, true, false, F32)
    MANY_ONE(!glu && !list && kind == BF16, 0, 2, 4, 8, 4, 2, false, false, BF16)
    MANY_ONE(!glu && !list && kind == BF16, 1, 2, 2, 4, 4, 2, false, false, BF16)
    MANY_ONE(!glu && !list && kind == BF16, 2, 2, 2, 4, 2, 2, false, false, BF16)
    MANY_ONE(!glu && !list && kind == BF16, 3, 2, 2, 2, 2, 3, false, false, BF16)
    MANY_ONE(!glu && !list && kind == BF16, 4, 2, 2, 1, 2, 4, false, false, BF16)
    MANY_ONE(!glu && !list && kind == BF16, 8, 4, 1, 2, 1, 3, false, false, BF16)
    MANY_ONE(!glu && !list && kind == BF16, 9, 4, 1, 1, 1, 4, false, false, BF16)
    MANY_ONE(!glu && !list && kind == F32, 0, 4, 2, 4, 4, 2, false, false, F32)
    MANY_ONE(!glu && !list && kind == F32, 1, 2, 2, 4, 2, 2, false, false, F32)
    MANY_ONE(!glu && !list && kind == F32, 2, 2, 2, 2, 2, 2, false, false, F32)
    MANY_ONE(!glu && !list && kind == F32, 3, 2, 2, 1, 2, 4, false, false, F32)
    MANY_ONE(!glu && !list && kind == F32, 8, 4, 1, 2, 1, 3, false, false, F32)
    MANY_ONE(!glu && !list && kind == F32, 9, 4, 1, 1, 1, 4, false, false, F32)
#undef MANY
#undef MANY_ONE
}


// Whether the blocks of the kernel for few columns turn rows that are not codes into them, each for itself, rather than a launch ahead of it:
// 12 cycles of a block's CU for a block of 128 against 3 us (2576 columns of K: 19 columns 400 blocks, 32 670)
bool converts(int KB, int64_t cols) { return KB * cols <= 512; }

// Whether the kernel for few columns takes them: single pairs, and matrices of so few times 16 rows, times 16 columns, that two of these at most come to a CU.  Us of it /
// of tiles, results in BF16: 4096 x 2048, 1 column 4.8 / 9.0, 32 6.9 / 7.4; 5120 x 2048, 16 6.8 / 9.1, 20 9.7 / 7.4; 12288 x 2048, 1 11.5 / 9.7; 248320 x 2048, 1 101 / 90, 32 164 / 102;
// 1408 x 2048, 64 6.3 / 7.5, 100 10.8 / 7.5; 4096 x 8192, 32 20 / 28, 8192 x 8192, 20 32 / 28.  Where K is short tiles are level (512 x 512, 1 4.7 / 4.4), and 17 columns and more theirs
// (32 5.3 / 4.5).
constexpr int FEW_UNITS = 512;
int64_t few_limit(const bf16n_fp8_weight & w) { // the most columns of a dense product that it takes
    const int KB = (int) ((w.K + FP8_BLOCK - 1) / FP8_BLOCK);
    const int64_t n = FEW_UNITS / std::max<int64_t>(1, (w.rows + 15) / 16) * few_pass(16, KB, true);
    return KB >= 8 ? n : std::min<int64_t>(n, 16);
}
bool few(const bf16n_fp8_weight & w, int64_t n_cols, bool listed, bool by_ids) { return by_ids || (!listed && n_cols <= few_limit(w)); }
size_t aligned(size_t n) { return (n + 255) / 256 * 256; }
size_t codes_bytes(int64_t rows, int64_t K) { return aligned(rows * K) + aligned(rows * ((K + FP8_BLOCK - 1) / FP8_BLOCK) * 4); }

} // namespace

void fp8_init() {
    (void) hipFuncSetAttribute((const void *) k_fp8_down, hipFuncAttributeMaxDynamicSharedMemorySize, (int) FEW_LDS);
    few_instance(nullptr, 0, false, 0, dim3(), 0, nullptr);
    run_many(nullptr, false, false, nullptr);
}

void launch_fp8_rows(const bf16n_fp8_rows & x, const bf16n_fp8_rows & y, int64_t rows, int64_t K, int cus, hipStream_t stream) {
    const int64_t items = rows * ((K + FP8_BLOCK - 1) / FP8_BLOCK);
    const unsigned grid = (unsigned) std::min<int64_t>((items + 15) / 16, (int64_t) cus * 64);
    (x.kind == BF16 ? k_fp8_rows<BF16> : k_fp8_rows<F32>)<<<grid, 256, 0, stream>>>((const char *) x.at, x.row, (uint8_t *) y.at, y.row, y.scales, y.scale_row, y.scale_block, rows, (int) K);
}

void launch_add_rmsnorm_fp8(const add_norm_args & a, const bf16n_fp8_rows & y, int n_tok, hipStream_t stream) {
    const int pieces = (int) ((a.n + 7) / 8), threads = std::min(1024, (pieces + 63) / 64 * 64);
    (a.ys ? (pieces <= 1024 ? k_add_rmsnorm_fp8<1, true> : k_add_rmsnorm_fp8<2, true>) : (pieces <= 1024 ? k_add_rmsnorm_fp8<1, false> : k_add_rmsnorm_fp8<2, false>))<<<n_tok, threads, 0, stream>>>(a, (uint8_t *) y.at, y.row, y.scales, y.scale_row, y.scale_block);
}

// whether rows of activations become codes in a launch of their own
static bool in_launch(const bf16n_fp8_weight & w, int x_kind, int64_t n_cols, bool listed, bool by_ids) {
    const int KB = (int) ((w.K + FP8_BLOCK - 1) / FP8_BLOCK);
    return x_kind != CODES && !(few(w, n_cols, listed, by_ids) && converts(KB, by_ids ? 1 : std::min<int64_t>(n_cols, 32)));
}

uint64_t fp8_workspace_bytes(const bf16n_fp8_weight & w, bool glu, int x_kind, int y_kind, int64_t x_rows, int64_t n_cols, bool listed, bool by_ids) {
    if (n_cols == 0) { // (the sizes of a pass and their number are for columns that there are)
        return 0;
    }
    const bool f = few(w, n_cols, listed, by_ids);
    uint64_t n = 0;
    if (in_launch(w, x_kind, n_cols, listed, by_ids)) {
        n += codes_bytes(x_rows, w.K);
    }
    if (y_kind == CODES && f) {
        n += aligned(n_cols * (w.rows / w.n_matrices) * 4);
    }
    return n;
}

uint64_t fp8_workspace_upto(const bf16n_fp8_weight & w, bool glu, int x_kind, int y_kind, int64_t x_rows, int64_t n_cols, bool listed, bool by_ids) {
    const uint64_t n = fp8_workspace_bytes(w, glu, x_kind, y_kind, x_rows, n_cols, listed, by_ids);
    const int64_t most = few_limit(w); // (both kernels' workspaces grow with the columns)
    return listed || by_ids || n_cols <= most ? n : std::max(n, fp8_workspace_bytes(w, glu, x_kind, y_kind, most, most, false, false));
}

void launch_fp8_product(const fp8_product & a, void * workspace, int cus, hipStream_t stream) {
    const bool glu = a.up != nullptr, listed = a.pairs != nullptr, by_ids = a.ids != nullptr;
    const bool f = few(*a.w, a.n_cols, listed, by_ids);
    fp8_launch p = launch_of(a, cus);
    char * ws = (char *) workspace;
    if (in_launch(*a.w, p.x_kind, a.n_cols, listed, by_ids)) {
        const bf16n_fp8_rows codes = {ws, (float *) (ws + aligned(a.x_rows * a.w->K)), a.w->K, 1, a.x_rows, CODES, 0};
        launch_fp8_rows(a.x, codes, a.x_rows, a.w->K, cus, stream);
        p.x = ws; p.x_row = a.w->K; p.xs = codes.scales; p.xs_row = 1; p.xs_block = a.x_rows; p.x_kind = CODES;
        ws += codes_bytes(a.x_rows, a.w->K);
    }
    if (!f) {
        run_many(&p, glu, listed, stream);
        return;
    }
    bf16n_fp8_rows plain = {};
    if (p.y_kind == CODES) {
        plain = {ws, nullptr, (int64_t) p.nrows * 4, 0, 0, F32, 0};
        p.y = ws; p.y_row = plain.row; p.y_kind = F32;
    }
    if (by_ids) {
        run_few(p, glu, 1, a.n_cols, (int) a.n_cols, cus, stream);
    } else {
        const int pass = few_pass(a.n_cols, p.KB, glu), passes = (int) ((a.n_cols + pass - 1) / pass);
        run_few(p, glu, pass, passes, passes, cus, stream);
    }
    if (plain.at) {
        launch_fp8_rows(plain, a.y, a.n_cols, p.nrows, cus, stream);
    }
}

bool fp8_down_fits(const bf16n_fp8_weight & down, int n_used) {
    const int KB = (int) ((down.K + FP8_BLOCK - 1) / FP8_BLOCK);
    return KB <= FEW_PARTS && fp8_down_layout(n_used, KB).bytes <= (int) FEW_LDS; // (n_used below 1024)
}
void launch_fp8_down(const fp8_product & a, const void * wts, bool wts_bf16, int n_tok, int cus, hipStream_t stream) {
    const fp8_launch p = launch_of(a, cus);
    note_kernel("k_fp8_down", nullptr, 0);
    k_fp8_down<<<dim3((p.nrows + 15) / 16, n_tok), 512, fp8_down_layout(p.n_used, p.KB).bytes, stream>>>(p, wts, wts_bf16);
}

void launch_fp8_combine(const float * ys, const void * w, bool w_bf16, void * y, bool y_bf16, int n_tok, int n_used, int64_t n, hipStream_t stream) {
    k_fp8_combine<<<dim3((unsigned) ((n / 8 + 255) / 256), (unsigned) n_tok), 256, 0, stream>>>(ys, w, w_bf16, (char *) y, y_bf16, n_used, n);
}

} // namespace dev
} // namespace bf16n
