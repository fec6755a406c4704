// Products with 4-bit weights and group scales (gfx950).
#include "dev_int4.h"
#include "launchers.h"

#include <algorithm>
#include <string>

namespace bf16n {
namespace dev {

namespace {

struct i4_launch {
    i4_matrix w, up;
    int K;                                  // columns, a multiple of 32
    int group_log2, n_groups;
    int nrows;                              // rows of one matrix
    const char * x; int64_t x_tok, x_slot;  // bytes; a list's pair takes activation row pair (per_slot) or pair / n_used
    char * y; int64_t y_tok, y_slot;        // bytes
    bool y_bf16;
    int ncols, n_used;                      // columns (dense) or (token, slot) pairs
    int x_per_slot;
    const char * ids; int64_t ids_s0, ids_s1; bool ids_i64;  // one matrix per (token, slot)
    int64_t n_matrices;
    const int32_t * pairs, * bounds;        // pairs sorted by matrix
    int cols_per_pass, ksplit;
};

constexpr int I4_STEP = 128; // columns that a wavefront takes at a time: 32 to a lane of each quarter

// pitch of a row of activations in LDS, in elements: whole steps, and 16 bytes more so that the 16 rows of an operand lie in
// different banks
__host__ __device__ inline int i4_pitch(int K) { return (K + I4_STEP - 1) / I4_STEP * I4_STEP + 8; }

// The columns of a launch's block, shared by the two kernels for few columns: which matrix, where a column's activations and results are.
struct i4_columns {
    const i4_launch & p;
    int64_t matrix = 0, x_one = 0, y_one = 0;
    int begin = 0, end;
    bool named = true; // false: the ids name no matrix
    __device__ i4_columns(const i4_launch & p) : p(p), end(p.ncols) {
        if (p.ids) {
            const int t = blockIdx.y / p.n_used, i = blockIdx.y % p.n_used;
            const char * at = p.ids + t * p.ids_s1 + i * p.ids_s0;
            matrix = p.ids_i64 ? *(const int64_t *) at : *(const int32_t *) at;
            named = matrix >= 0 && matrix < p.n_matrices;
            x_one = t * p.x_tok + (i % p.x_per_slot) * p.x_slot;
            y_one = t * p.y_tok + i * p.y_slot;
            end = 1;
        } else if (p.bounds) {
            matrix = blockIdx.y;
            begin = p.bounds[matrix];
            end = p.bounds[matrix + 1];
            named = matrix < p.n_matrices; // behind the last one: pairs that name none
        }
    }
    __device__ int64_t y_of(int c) const { return p.pairs ? p.pairs[c] * p.y_slot : y_one + c * p.y_tok; }
    __device__ int64_t x_of(int c) const {
        if (p.pairs) {
            const int pair = p.pairs[c];
            return p.x_per_slot > 1 ? pair * p.x_slot : pair / p.n_used * p.x_tok;
        }
        return x_one + c * p.x_tok;
    }
    __device__ void zero() const { // no such matrix: rows of zeros
        for (int c = begin + blockIdx.z; c < end; c += gridDim.z) {
            for (int r = blockIdx.x * blockDim.x + threadIdx.x; r < p.nrows; r += gridDim.x * blockDim.x) {
                store_y(p.y + y_of(c), p.y_bf16, r, 0.f);
            }
        }
    }
};

// Few columns.  One wavefront takes 16 rows of the matrix (of each of the two where they are gated) and 256 columns of it at
// a time: a lane's 32 bytes are 64 codes of row lane % 16 (four lanes have 128 bytes of a row, a whole
// line), turned into eight operands of v_mfma_f32_16x16x32_bf16 whose other
// operand is the activations, from LDS; result: lane = row of the matrix, register = activation row (so that a scale
// is one value to a lane).  FP32 activations are three BF16 rows each (rows 4 t .. 4 t + 2 of the 16: one lane's registers).
// The sums of the activations over a group, which the zero points need, are taken once, on the way into LDS.
// A step's registers take the codes of the step U later as soon as its operands are made.
// Wavefronts of a block share the rows (ksplit parts of K each, summed through LDS in a fixed order) or take other rows.
// Bound by HBM where the matrix is large: 248320 x 2048, one token, 5.2 TB/s.
template <int NT, int NM, int GM, bool GLU, bool XF32, bool ZEROS, int NW>
__global__ void __launch_bounds__(NW * 64, NT * NM > 2 ? 2 : 4) k_i4_few(const i4_launch p) {
    constexpr int U = NM == 1 ? 2 : 1;                  // pairs of steps whose codes are loaded ahead
    constexpr int NG = GM == 0 ? 1 : GM == 1 ? 2 : 4;   // groups in a step of 128 columns (128 and more columns, 64, 32)
    constexpr int CPT = XF32 ? 4 : 16;                  // columns in a tile of 16 activation rows
    constexpr int NA = XF32 ? 1 : 4;                    // results of a lane in a tile
    constexpr int TILE_ROWS = 16 * (GLU ? 1 : NM);
    extern __shared__ __align__(16) char lds[];
    uint16_t * const xs = (uint16_t *) lds;
    const int lane = threadIdx.x & 63, m16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int K = p.K, pitch = i4_pitch(K), x_rows = p.cols_per_pass * (XF32 ? 3 : 1);
    const int steps = (K + I4_STEP - 1) / I4_STEP;
    float * const xsum = (float *) (xs + x_rows * pitch);          // [steps * NG][NT * CPT]
    int64_t * const y_off = (int64_t *) (xsum + steps * NG * NT * CPT); // [NT * CPT]
    float * const red = (float *) (y_off + NT * CPT);

    const i4_columns cols(p);
    if (!cols.named) {
        cols.zero();
        return;
    }
    const int64_t matrix = cols.matrix;
    const int c_begin = cols.begin, c_end = cols.end;

    const int row_groups = NW / p.ksplit, kp = wave % p.ksplit;
    const int pairs = (steps + 1) / 2, s0 = pairs * kp / p.ksplit, s1 = pairs * (kp + 1) / p.ksplit;
    const int n_chunks = (s1 - s0 + U - 1) / U;
    const int block_rows = row_groups * TILE_ROWS;
    const int first_row = blockIdx.x * block_rows + wave / p.ksplit * TILE_ROWS, row_step = gridDim.x * block_rows;
    // rows beyond the columns repeat the last: their results are dropped
    int x_at[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int c = min(t * CPT + (XF32 ? m16 >> 2 : m16), p.cols_per_pass - 1);
        x_at[t] = (XF32 ? c * 3 + min(m16 & 3, 2) : c) * pitch + (GM == 0 ? (q & 1) * 64 + (q >> 1) * 32 : q * 8);
    }
    // a last pair that is cut short: lanes behind the last column read the columns before it, against activations of zero
    const int at_last = (pairs - 1) * 2 * I4_STEP + q * 64, tail[2] = {at_last < K ? 0 : q * 32, at_last + 32 < K ? 0 : q * 32 + 16};
    const uint32_t f16[2] = {p.w.f16 ? ~0u : 0u, p.up.f16 ? ~0u : 0u};

    for (int c0 = c_begin + blockIdx.z * p.cols_per_pass; c0 < c_end; c0 += gridDim.z * p.cols_per_pass) {
        const int nc = min(c_end - c0, p.cols_per_pass);

        u32x4_t code[U * NM * 2];
        // where the loads are: a tile's place is the same for all lanes, a lane's offset in it the same for all tiles but one that
        // the matrix ends in, whose lanes beyond repeat its last row
        const uint8_t * codes[NM];
        int code_off[NM];
        const auto at_tile = [&](int r0) {
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const i4_matrix & w = GLU && m ? p.up : p.w;
                const int r = min(r0 + (GLU ? 0 : 16 * m), p.nrows - 1);
                const int64_t base = matrix * p.nrows + r;
                codes[m] = w.codes + base * (K / 2);
                code_off[m] = min(m16, p.nrows - 1 - r) * (K / 2) + q * 32;
            }
        };
        const auto load = [&](int s, int u) {
#pragma unroll
            for (int m = 0; m < NM; m++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    code[(u * NM + m) * 2 + h] = *(const u32x4_t *) (codes[m] + s * I4_STEP + h * 16 + (code_off[m] - (s == pairs - 1 ? tail[h] : 0)));
                }
            }
        };
        // Scales and zero points come by blocks of 16 groups, four of its row to a lane of each quarter, a block ahead; a step takes
        // them from the quarter that has its group.  (A load of one scale by every lane for every 128 columns: 248320 x 2048, one token, 72 us where this takes 55.)
        uint64_t sc[NM], sc_next[NM];
        uint32_t ze[NM], ze_next[NM];
        const auto block_of = [&](int s) { return (s * 2 * I4_STEP >> p.group_log2) >> 4; };
        const auto first_of = [&](int block, int quarter) { return max(min(block * 16 + quarter * 4, p.n_groups - 4), 0); };
        const auto load_block = [&](int r0, int block) {
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const i4_matrix & w = GLU && m ? p.up : p.w;
                const int r = min(r0 + (GLU ? 0 : 16 * m), p.nrows - 1);
                const int64_t base = (matrix * p.nrows + r) * p.n_groups;
                const int at = min(m16, p.nrows - 1 - r) * p.n_groups + first_of(block, q);
                if (p.n_groups >= 4) {
                    sc_next[m] = *(const u64_at_2 *) (w.scales + base + at);
                    if (ZEROS) {
                        ze_next[m] = *(const u32_at_1 *) (w.zeros + base + at);
                    }
                } else {
                    const int i1 = min(1, p.n_groups - 1), i2 = min(2, p.n_groups - 1);
                    sc_next[m] = w.scales[base + at] | (uint32_t) w.scales[base + at + i1] << 16 | (uint64_t) w.scales[base + at + i2] << 32;
                    if (ZEROS) {
                        ze_next[m] = w.zeros[base + at] | w.zeros[base + at + i1] << 8 | w.zeros[base + at + i2] << 16;
                    }
                }
            }
        };
        at_tile(first_row);
        load_block(first_row, block_of(s0));
#pragma unroll
        for (int u = 0; u < U; u++) {
            load(min(s0 + u, s1 - 1), u);
        }

        // Activations into LDS, in the operands' order, zeros behind the last column of the matrix, and their groups' sums: a
        // wavefront takes 512 columns of a row at a time and has AHEAD such pieces on the way.  (One after the other cost a latency
        // each: 16 tokens of 5120 x 2048 in this kernel 11.9 us, now 10.8.)
        constexpr int AHEAD = XF32 ? 2 : 4;
        const int octs = (pitch - 8) / 8; // a multiple of 16: a row of 16 lanes has 128 columns of one activation row
        const int per_row = (octs + 63) / 64, pieces = p.cols_per_pass * per_row;
        __syncthreads();
        for (int first = wave; first < pieces; first += NW * AHEAD) {
            f32x4_t va[AHEAD], vb[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                const int i = first + k * NW, c = i / per_row, o = (i - c * per_row) * 64 + lane;
                va[k] = vb[k] = f32x4_t{};
                if (i < pieces && c < nc && o * 8 < K) {
                    const char * src = p.x + cols.x_of(c0 + c) + o * (XF32 ? 32 : 16);
                    va[k] = *(const f32x4_t *) src;
                    if (XF32) {
                        vb[k] = *(const f32x4_t *) (src + 16);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                const int i = first + k * NW, c = i / per_row, o = (i - c * per_row) * 64 + lane;
                float sum = 0.f;
                if (i < pieces && o < octs) { // (rows of 16 lanes are in or out as a whole)
                    if constexpr (XF32) {
                        uint32_t parts[3][8];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const float v = j < 4 ? va[k][j & 3] : vb[k][j & 3];
                            f32_parts(v, parts[0][j], parts[1][j], parts[2][j]);
                            sum += v;
                        }
#pragma unroll
                        for (int h = 0; h < 3; h++) {
                            const uint32_t * e = parts[h];
                            *(u32x4_t *) (xs + (c * 3 + h) * pitch + o * 8) =
                                u32x4_t{e[0] | e[2] << 16, e[4] | e[6] << 16, e[1] | e[3] << 16, e[5] | e[7] << 16};
                        }
                    } else {
                        const u32x4_t v = __builtin_bit_cast(u32x4_t, va[k]);
                        *(u32x4_t *) (xs + c * pitch + o * 8) = i4_order(v);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            sum += __uint_as_float(v[j] << 16) + __uint_as_float(v[j] & 0xFFFF0000u);
                        }
                    }
                }
                sum = dpp_add<0xB1, 0xf>(sum); // over 4, 8 or 16 lanes: 32, 64 or 128 columns
                sum = dpp_add<0x4E, 0xf>(sum);
                if (GM < 2) {
                    sum = dpp_add<0x141, 0xf>(sum);
                }
                if (GM < 1) {
                    sum = dpp_add<0x140, 0xf>(sum);
                }
                constexpr int OG = 16 / NG;
                if (i < pieces && o < octs && o % OG == 0) {
                    xsum[o / OG * (NT * CPT) + c] = sum;
                }
            }
        }
        if (threadIdx.x < nc) {
            y_off[threadIdx.x] = cols.y_of(c0 + threadIdx.x);
        }
        __syncthreads();

        int parity = 0;
        const f32x4_t none = {};
        for (int r0 = first_row; r0 < p.nrows + wave / p.ksplit * TILE_ROWS; r0 += row_step) { // (the block's wavefronts make the same rounds)
            float acc[NM * NT][NA];
#pragma unroll
            for (int t = 0; t < NM * NT; t++) {
#pragma unroll
                for (int e = 0; e < NA; e++) {
                    acc[t][e] = 0.f;
                }
            }
            for (int chunk = 0; chunk < n_chunks; chunk++) {
                int ahead = s0 + (chunk + 1) * U;
                if (chunk + 1 == n_chunks) {
                    at_tile(r0 + row_step); // behind the matrix: its last row, for nothing
                    ahead = s0;
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int s = s0 + chunk * U + u;
                    if (s < s1) {
                        const int block = block_of(s);
                        if (s == s0 || block != block_of(s - 1)) {
#pragma unroll
                            for (int m = 0; m < NM; m++) {
                                sc[m] = sc_next[m];
                                ze[m] = ze_next[m];
                            }
                            const bool more = block < block_of(s1 - 1);
                            load_block(more ? r0 : r0 + row_step, more ? block + 1 : block_of(s0));
                        }
                        // the words of the two steps: lanes of the upper half wave give theirs of the first for the lower half's of the second
                        u32x4_t d[2][NM];
#pragma unroll
                        for (int m = 0; m < NM; m++) {
                            const u32x4_t & a = code[(u * NM + m) * 2], & b = code[(u * NM + m) * 2 + 1];
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const auto r = __builtin_amdgcn_permlane32_swap(a[j], b[j], false, false);
                                d[0][m][j] = r[0];
                                d[1][m][j] = r[1];
                            }
                        }
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            if (h && s * 2 + 1 == steps) {
                                break;
                            }
                            float sv[NM * NG], zv[NM * NG];
#pragma unroll
                            for (int m = 0; m < NM; m++) {
                                if (GM) {
                                    d[h][m] = i4_transpose(d[h][m]); // (quarter 1 has the third 32 columns here, quarter 2 the second)
                                    const uint32_t v = d[h][m][1];
                                    d[h][m][1] = d[h][m][2];
                                    d[h][m][2] = v;
                                }
#pragma unroll
                                for (int g = 0; g < NG; g++) {
                                    const int gi = min((s * 2 + h) * I4_STEP + g * (I4_STEP / NG) >> p.group_log2, p.n_groups - 1);
                                    const int quarter = (gi >> 2) & 3, i = gi - first_of(block, quarter), from = (quarter * 16 + m16) * 4;
                                    const uint32_t v = __builtin_amdgcn_ds_bpermute(from, (uint32_t) (i & 2 ? sc[m] >> 32 : sc[m]));
                                    sv[m * NG + g] = i4_scale(v >> (i & 1) * 16 & 0xFFFFu, f16[GLU && m]);
                                    zv[m * NG + g] = ZEROS ? (float) ((uint32_t) __builtin_amdgcn_ds_bpermute(from, ze[m]) >> i * 8 & 0xFFu) : 8.f;
                                }
                            }
#pragma unroll
                            for (int g = 0; g < NG; g++) {
                                f32x4_t part[NM * NT];
#pragma unroll
                                for (int j = g * 4 / NG; j < (g + 1) * 4 / NG; j++) {
                                    const bool first = j == g * 4 / NG;
                                    bf16x8_t wf[NM];
#pragma unroll
                                    for (int m = 0; m < NM; m++) {
                                        wf[m] = i4_operand(d[h][m][j]);
                                    }
#pragma unroll
                                    for (int t = 0; t < NT; t++) {
                                        const bf16x8_t xf = __builtin_bit_cast(bf16x8_t, *(const u32x4_t *) (xs + x_at[t] + (s * 2 + h) * I4_STEP + (GM == 0 ? j * 8 : j * 32)));
#pragma unroll
                                        for (int m = 0; m < NM; m++) {
                                            part[m * NT + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, wf[m], first ? none : part[m * NT + t], 0, 0, 0);
                                        }
                                    }
                                }
#pragma unroll
                                for (int t = 0; t < NT; t++) {
                                    const float * at = xsum + ((s * 2 + h) * NG + g) * (NT * CPT) + t * CPT + q * NA;
                                    float x[NA];
                                    if constexpr (XF32) {
                                        x[0] = at[0];
                                    } else {
                                        *(f32x4_t *) x = *(const f32x4_t *) at;
                                    }
#pragma unroll
                                    for (int m = 0; m < NM; m++) {
                                        const f32x4_t & pt = part[m * NT + t];
#pragma unroll
                                        for (int e = 0; e < NA; e++) {
                                            const float sum = XF32 ? pt[0] + (pt[1] + pt[2]) : pt[e];
                                            acc[m * NT + t][e] = fmaf(sv[m * NG + g], fmaf(-zv[m * NG + g], x[e], sum), acc[m * NT + t][e]);
                                        }
                                    }
                                }
                            }
                        }
                    }
                    load(min(ahead + u, s1 - 1), u);
                }
            }
            if (p.ksplit > 1) {
                float * const buf = red + parity * (NW * 64 * NA * NM * NT);
                parity ^= 1; // the next tile's sums go elsewhere: the barrier in between is one that the readers of this one pass
#pragma unroll
                for (int i = 0; i < NM * NT; i++) {
#pragma unroll
                    for (int e = 0; e < NA; e++) {
                        buf[((wave * NM * NT + i) * NA + e) * 64 + lane] = acc[i][e];
                    }
                }
                __syncthreads();
                if (kp != 0) {
                    continue;
                }
                for (int k = 1; k < p.ksplit; k++) {
#pragma unroll
                    for (int i = 0; i < NM * NT; i++) {
#pragma unroll
                        for (int e = 0; e < NA; e++) {
                            acc[i][e] += buf[(((wave + k) * NM * NT + i) * NA + e) * 64 + lane];
                        }
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
                for (int e = 0; e < NA; e++) {
                    const int c = t * CPT + q * NA + e;
                    if (c < nc) {
                        char * const y = p.y + y_off[c];
#pragma unroll
                        for (int m = 0; m < (GLU ? 1 : NM); m++) {
                            const int r = r0 + 16 * m + m16;
                            if (r < p.nrows) {
                                store_y(y, p.y_bf16, r, GLU ? silu(acc[t][e]) * acc[(GLU ? NT : 0) + t][e] : acc[m * NT + t][e]);
                            }
                        }
                    }
                }
            }
        }
    }
}

// Few columns of a matrix whose rows are few as well: nothing is shared through LDS but the sums of the parts of K.  A
// wavefront loads its codes, scales and activations, these as the operand's lanes hold them, at once, one latency in
// all; the groups' sums of the activations come from products with ones.
// 512 x 2048, one token: 4.1 us in a graph, 5.8 with the activations through LDS; 1453 x 2560, gated, groups of 32, 11 tokens 7.8 / 14.5.  Bound by that latency.
template <int NT, int GM, bool GLU, bool XF32, bool ZEROS>
__global__ void __launch_bounds__(512, 2) k_i4_small(const i4_launch p) {
    constexpr int NW = 8, NM = GLU ? 2 : 1, NG = GM == 0 ? 1 : GM == 1 ? 2 : 4, CPT = XF32 ? 4 : 16, NA = XF32 ? 1 : 4;
    __shared__ float red[NW * NM * NT * NA * 64];
    const int lane = threadIdx.x & 63, m16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const i4_columns cols(p);
    if (!cols.named) {
        cols.zero();
        return;
    }
    const int K = p.K, steps = (K + I4_STEP - 1) / I4_STEP, n_pairs = (steps + 1) / 2, kp = wave % p.ksplit;
    const int row_groups = NW / p.ksplit, r0 = (blockIdx.x * row_groups + wave / p.ksplit) * 16;
    const int first = min(r0, p.nrows - 1), row = min(m16, p.nrows - 1 - first); // rows beyond the matrix repeat its last: dropped
    const int64_t base = cols.matrix * p.nrows + first;
    const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, u32x4_t{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
    const f32x4_t none = {};
    for (int c0 = cols.begin + blockIdx.z * p.cols_per_pass; c0 < cols.end; c0 += gridDim.z * p.cols_per_pass) {
        const int nc = min(cols.end - c0, p.cols_per_pass);
        const char * x_at[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            x_at[t] = p.x + cols.x_of(c0 + min(t * CPT + (XF32 ? m16 >> 2 : m16), nc - 1));
        }
        float acc[NM * NT][NA];
#pragma unroll
        for (int i = 0; i < NM * NT; i++) {
#pragma unroll
            for (int e = 0; e < NA; e++) {
                acc[i][e] = 0.f;
            }
        }
        for (int s = kp; s < n_pairs; s += p.ksplit) {
            u32x4_t code[NM][2];
            uint64_t sc[NM][NG == 4 ? 2 : 1], ze[NM]; // scales, 16 bits each, and zero points of the 2 NG groups
            const int g0 = s * 2 * I4_STEP >> p.group_log2;
            const bool whole = p.group_log2 <= 7 && g0 + 2 * NG <= p.n_groups;
            const int at = s * 2 * I4_STEP + q * 64; // lanes behind the last column read columns before it, against activations of zero
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const i4_matrix & w = GLU && m ? p.up : p.w;
                const uint8_t * from = w.codes + base * (K / 2) + row * (K / 2);
                code[m][0] = *(const u32x4_t *) (from + (at < K ? at : 0) / 2);
                code[m][1] = *(const u32x4_t *) (from + (at + 32 < K ? at + 32 : 0) / 2);
                const uint16_t * sat = w.scales + base * p.n_groups + row * p.n_groups;
                const uint8_t * zat = w.zeros + base * p.n_groups + row * p.n_groups;
                ze[m] = 0;
                if (whole) {
                    if (NG == 1) {
                        sc[m][0] = *(const u32_at_2 *) (sat + g0);
                    } else {
                        sc[m][0] = *(const u64_at_2 *) (sat + g0);
                        sc[m][NG == 4 ? 1 : 0] = *(const u64_at_2 *) (sat + g0 + (NG == 4 ? 4 : 0));
                    }
                    if (ZEROS) {
                        ze[m] = NG == 1 ? *(const u16_at_1 *) (zat + g0) : NG == 2 ? *(const u32_at_1 *) (zat + g0) : *(const u64_at_1 *) (zat + g0);
                    }
                } else {
                    sc[m][0] = sc[m][NG == 4 ? 1 : 0] = 0;
#pragma unroll
                    for (int g = 0; g < 2 * NG; g++) {
                        const int gi = min((s * 2 * I4_STEP + g * (I4_STEP / NG)) >> p.group_log2, p.n_groups - 1);
                        sc[m][g / 4] |= (uint64_t) sat[gi] << g % 4 * 16;
                        ze[m] |= ZEROS ? (uint64_t) zat[gi] << g * 8 : 0;
                    }
                }
            }
            bf16x8_t xf[NT][8];
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int h = i / 4, j = i % 4;
                    const int col = (s * 2 + h) * I4_STEP + (GM == 0 ? (q & 1) * 64 + (q >> 1) * 32 + j * 8 : j * 32 + q * 8);
                    u32x4_t v = {};
                    if constexpr (XF32) {
                        f32x4_t a = {}, b = {};
                        if (col < K) {
                            a = *(const f32x4_t *) (x_at[t] + col * 4);
                            b = *(const f32x4_t *) (x_at[t] + col * 4 + 16);
                        }
                        uint32_t e[8];
#pragma unroll
                        for (int l = 0; l < 8; l++) { // this lane's part of the three
                            uint32_t f0, f1, f2;
                            f32_parts(l < 4 ? a[l & 3] : b[l & 3], f0, f1, f2);
                            e[l] = (m16 & 3) == 0 ? f0 : (m16 & 3) == 1 ? f1 : f2;
                        }
                        v = u32x4_t{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
                    } else if (col < K) {
                        v = *(const u32x4_t *) (x_at[t] + col * 2);
                    }
                    xf[t][i] = __builtin_bit_cast(bf16x8_t, v);
                }
            }
            u32x4_t d[2][NM];
#pragma unroll
            for (int m = 0; m < NM; m++) {
#pragma unroll
                for (int j = 0; j < 4; j++) { // as in k_i4_few
                    const auto r = __builtin_amdgcn_permlane32_swap(code[m][0][j], code[m][1][j], false, false);
                    d[0][m][j] = r[0];
                    d[1][m][j] = r[1];
                }
                if (GM) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const u32x4_t e = i4_transpose(d[h][m]);
                        d[h][m] = u32x4_t{e[0], e[2], e[1], e[3]};
                    }
                }
            }
#pragma unroll
            for (int g = 0; g < 2 * NG; g++) {
                f32x4_t part[NM * NT], xsum[NT];
                constexpr int J = 4 / NG;
#pragma unroll
                for (int j = 0; j < J; j++) {
                    const int i = g * J + j;
                    bf16x8_t wf[NM];
#pragma unroll
                    for (int m = 0; m < NM; m++) {
                        wf[m] = i4_operand_in_order(d[i / 4][m][i % 4]);
                    }
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        xsum[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[t][i], ones, j ? xsum[t] : none, 0, 0, 0);
#pragma unroll
                        for (int m = 0; m < NM; m++) {
                            part[m * NT + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[t][i], wf[m], j ? part[m * NT + t] : none, 0, 0, 0);
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < NM; m++) {
                    const float sv = i4_scale((uint32_t) (sc[m][g / 4] >> g % 4 * 16) & 0xFFFFu, (GLU && m ? p.up : p.w).f16 ? ~0u : 0u);
                    const float zv = ZEROS ? (float) ((uint32_t) (ze[m] >> g * 8) & 0xFFu) : 8.f;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const f32x4_t & a = part[m * NT + t], & b = xsum[t];
#pragma unroll
                        for (int e = 0; e < NA; e++) {
                            const float sum = XF32 ? a[0] + (a[1] + a[2]) : a[e], x = XF32 ? b[0] + (b[1] + b[2]) : b[e];
                            acc[m * NT + t][e] = fmaf(sv, fmaf(-zv, x, sum), acc[m * NT + t][e]);
                        }
                    }
                }
            }
        }
        if (p.ksplit > 1) {
            __syncthreads(); // (the last pass's sums have been read)
#pragma unroll
            for (int i = 0; i < NM * NT; i++) {
#pragma unroll
                for (int e = 0; e < NA; e++) {
                    red[((wave * NM * NT + i) * NA + e) * 64 + lane] = acc[i][e];
                }
            }
            __syncthreads();
            if (kp != 0) {
                continue;
            }
            for (int k = 1; k < p.ksplit; k++) {
#pragma unroll
                for (int i = 0; i < NM * NT; i++) {
#pragma unroll
                    for (int e = 0; e < NA; e++) {
                        acc[i][e] += red[(((wave + k) * NM * NT + i) * NA + e) * 64 + lane];
                    }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int e = 0; e < NA; e++) {
                const int c = t * CPT + q * NA + e;
                if (c < nc && r0 + m16 < p.nrows) {
                    store_y(p.y + cols.y_of(c0 + c), p.y_bf16, r0 + m16, GLU ? silu(acc[t][e]) * acc[(GLU ? NT : 0) + t][e] : acc[t][e]);
                }
            }
        }
    }
}

// ---------------------------------------------------------------- many columns
//
// The zero points' part of a product,  - sum_g s[r, g] z[r, g] X[t, g]  with X the sum of the activations over group g (of 128
// columns where it is larger), is a product of its own over the groups.  Both factors are cut into three BF16 parts that add
// up to them, so that it runs on the matrix cores as well: eight columns for a group, X1 X2 X1 X3 X2 X1 X3 X2 against
// Z1 Z1 Z2 Z1 Z2 Z3 Z2 Z3, instead of four FMAs per result tile and group.  A third part is below 2^-14 of its number, so what is left
// out, X3 Z3, is below 2^-28 of the product.

// X of every activation row, in parts: one thread to 32 columns.  For lists of columns by matrix the last block counts the pieces of
// `cols` columns of every matrix (and of the pairs that name none) instead and lists them: (matrix, first column, columns), how many in table[0].
__global__ void __launch_bounds__(256) k_i4_sums(const char * x, int64_t x_row, int K, int group, int64_t n_rows, u32x4_t * sums, int64_t sums_row,
                                                 const int32_t * bounds, int n_matrices, int cols, int4 * table) {
    if (bounds && blockIdx.x == gridDim.x - 1) {
        __shared__ int of_wave[4];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        int before = 0;
        for (int b = 0; b <= n_matrices; b += 256) {
            const int m = b + threadIdx.x;
            const int from = m <= n_matrices ? bounds[m] : 0, to = m <= n_matrices ? bounds[m + 1] : 0, n = (to - from + cols - 1) / cols;
            int upto = n;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(upto, o, 64);
                upto += lane >= o ? v : 0;
            }
            if (lane == 63) {
                of_wave[wave] = upto;
            }
            __syncthreads();
            int at = before + upto - n;
            for (int w = 0; w < 4; w++) {
                at += w < wave ? of_wave[w] : 0;
                before += of_wave[w];
            }
            for (int k = 0; k < n; k++) {
                table[1 + at + k] = int4{m, from + k * cols, min(cols, to - from - k * cols), 0};
            }
            __syncthreads();
        }
        if (threadIdx.x == 0) {
            table[0] = int4{before, 0, 0, 0};
        }
        return;
    }
    const int per = group / 32;                               // threads to a group: 1, 2 or 4
    const int64_t segs = (K / 32 + per - 1) / per * per;
    const int64_t i = (int64_t) blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t row = i / segs, seg = i % segs;
    float v = 0.f;
    if (row < n_rows && seg < K / 32) {
        const u32x4_t * at = (const u32x4_t *) (x + row * x_row + seg * 64);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const u32x4_t d = at[j];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v += __uint_as_float(d[e] << 16) + __uint_as_float(d[e] & 0xFFFF0000u);
            }
        }
    }
    if (per > 1) {
        v += __shfl_xor(v, 1, 64);
    }
    if (per > 2) {
        v += __shfl_xor(v, 2, 64);
    }
    if (row < n_rows && seg % per == 0) {
        uint32_t a, b, c;
        f32_parts(v, a, b, c);
        sums[row * sums_row + seg / per] = u32x4_t{a | b << 16, a | c << 16, b | a << 16, c | b << 16};
    }
}

struct i4_many {
    i4_matrix w, up;
    int K, nrows;
    int group_log2, n_groups;
    const char * x; int64_t x_row;          // bytes
    char * y; int64_t y_row;                // bytes
    bool y_bf16;
    const u32x4_t * sums; int sums_row;     // groups of a row, of sum_group_log2 columns
    int sum_group_log2;
    int ncols;
    const int32_t * pairs, * bounds;        // lists of columns by matrix, or null
    const int4 * table;                     // and their pieces
    int n_matrices;
    uint32_t per_token, one_used;           // pairs to a row of activations, and 2^32 over them
    int row_tiles, col_tiles;               // dense: the grid
};

// A block takes WM * MT * 16 columns and WN * NT * 16 rows (half of them of either matrix where they are gated) and 128 columns of K
// at a time: the activations' piece and the codes go straight into LDS a step ahead (two buffers, 16-byte places exchanged by the row's
// low bits so that the operands' reads find every bank); a wavefront turns its own codes into operands, which serve MT tiles.  Every product over a group starts from zero and is added to the result times its scale.
// Bound by the vector instructions (nine for eight codes and tile of rows, four for a tile of results and group), the products and the
// reads of LDS, which take turns more than they overlap: 8192 tokens of 8192 x 2048 take 332 us, 830 TFLOP/s, 2048 of 5120 x 2048 64, 670.
// (Of the 332 us without the additions 294 remained, without the conversions 309, without three of four products 234.)  Making the next
// operands under this step's products, with a step's copies spread over it, came to the same times.
template <int WM, int WN, int MT, int NT, int GM, bool GLU, bool LIST>
__global__ void __launch_bounds__(WM * WN * 64, LIST ? 3 : 2) k_i4_many(const i4_many p) {
    constexpr int THREADS = WM * WN * 64, COLS = WM * MT * 16, ROWS = WN * NT * 16 / (GLU ? 2 : 1);
    constexpr int NG = GM == 0 ? 1 : GM == 1 ? 2 : 4, LOADS = COLS * 16 / THREADS;
    static_assert(THREADS == 256 && LOADS * THREADS == COLS * 16, "a thread copies the same place of rows 16 apart");
    constexpr int CODE_BYTES = WN * NT * 1024, COPIES = WN * NT / 4; // codes of a step; a wavefront copies those of COPIES tiles of rows
    static_assert(COPIES * 4 == WN * NT, "four wavefronts");
    extern __shared__ __align__(16) char lds[]; // two pieces of activations, two of codes, for lists the places of the results
    constexpr int CODES = 2 * COLS * 256;
    int64_t * const y_at = (int64_t *) (lds + CODES + 2 * CODE_BYTES);
    const int lane = threadIdx.x & 63, m16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM;

    // the block's rows and columns
    int64_t matrix = 0;
    int c0, nc, row_tile;
    if constexpr (LIST) {
        // An XCD takes every eighth block, which is made a contiguous part of (piece, row tile) here: the row tiles of a piece read
        // its activations from one L2.
        const int n = p.table[0].x * p.row_tiles, per = (n + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
        if ((int) (blockIdx.x >> 3) >= per || id >= n) {
            return;
        }
        const int4 piece = p.table[1 + id / p.row_tiles];
        const int m = piece.x;
        matrix = m;
        row_tile = id % p.row_tiles;
        c0 = piece.y;
        nc = piece.z;
        if (m == p.n_matrices) { // zeros for the pairs that name none
            const int from = row_tile * ROWS, rows = min(ROWS, p.nrows - from);
            for (int i = threadIdx.x; i < nc * ROWS; i += THREADS) {
                if (i % ROWS < rows) {
                    store_y(p.y + p.pairs[c0 + i / ROWS] * p.y_row, p.y_bf16, from + i % ROWS, 0.f);
                }
            }
            return;
        }
    } else {
        // An XCD takes every eighth block, which is made a contiguous part of the tiles here: four column tiles of one row tile
        // after the other, so that what runs there at a time shares few pieces of activations (four times a row tile's bytes).
        // 8192 x 2048, 8192 tokens: 332 us where all column tiles of a row tile side by side take 373.
        const int n = p.row_tiles * p.col_tiles, per = (n + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
        if (id >= n) {
            return;
        }
        const int group = id / (p.row_tiles * 4), in = id - group * p.row_tiles * 4, wide = min(4, p.col_tiles - group * 4);
        row_tile = in / wide;
        c0 = (group * 4 + in % wide) * COLS;
        nc = min(COLS, p.ncols - c0);
    }
    const auto x_row_of = [&](int i) { // the activation row behind column i; columns that are not there repeat the last
        const int c = c0 + min(i, nc - 1);
        if constexpr (!LIST) {
            return c;
        } else { // a pair's token: by the reciprocal, rounded down, which is at most one too few
            const uint32_t pair = p.pairs[c], token = __umulhi(pair, p.one_used);
            return (int) (token + (pair - token * p.per_token >= p.per_token));
        }
    };
    if (LIST && threadIdx.x < nc) {
        y_at[threadIdx.x] = p.pairs[c0 + threadIdx.x] * p.y_row; // (read behind the barriers of the steps)
    }

    const int row0 = row_tile * ROWS;
    const int S = (int) ((p.K + I4_STEP - 1) / I4_STEP), E = (p.sums_row + 15) / 16;
    const int place = threadIdx.x & 15, octet = place ^ (threadIdx.x >> 4); // what this thread copies: places of rows (threadIdx.x >> 4) + 16 i
    // (rows of the activations start below 2^32 bytes, the launch sees to it; octets behind the last column repeat one before it: the codes
    // are zeros there)
    uint32_t x_off[LOADS], x_at[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        x_at[i] = x_row_of(i * 16 + (threadIdx.x >> 4));
        x_off[i] = x_at[i] * (uint32_t) p.x_row + octet * 16;
    }
    const bool cut = p.K % I4_STEP != 0; // the last step is cut short
    const auto copy_sums = [&](int step, int buf) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            if (i * 16 >= nc) {
                break;
            }
            const int64_t r = x_at[i];
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *) (p.sums + r * p.sums_row + min(step * 16 + octet, p.sums_row - 1)),
                                             (__attribute__((address_space(3))) void *) (lds + buf * (COLS * 256) + wave * 1024 + i * 4096), 16, 0, 0);
        }
    };
    const auto copy = [&](int s, int buf) {
        const char * const from = p.x + s * (I4_STEP * 2);
        if (cut && s == S - 1 && s * I4_STEP + octet * 8 >= p.K) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                x_off[i] -= octet * 16;
            }
        }
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            if (i * 16 < nc) { // (places of rows 16 i ..)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *) (from + x_off[i]),
                                                 (__attribute__((address_space(3))) void *) (lds + buf * (COLS * 256) + wave * 1024 + i * 4096), 16, 0, 0);
            }
        }
    };
    // a lane's row of tile n as an offset from the wavefront's first
    const int wave_row = (int) min(row0 + wn * (GLU ? NT / 2 : NT) * 16, p.nrows - 1);
    const int64_t wave_at = matrix * p.nrows + wave_row;
    int row_off[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        row_off[n] = min((GLU ? n % (NT / 2) : n) * 16 + m16, (int) p.nrows - 1 - wave_row);
    }
    const auto of = [&](int n) -> const i4_matrix & { return GLU && n >= NT / 2 ? p.up : p.w; };
    // the codes of a step: a wavefront copies tiles of rows wave, wave + 4 .., four lanes to a row; places exchanged by the row's bits
    uint32_t code_off[COPIES];
    const uint8_t * code_at[COPIES];
    const int chunk = (lane & 3) ^ (lane >> 4);
#pragma unroll
    for (int i = 0; i < COPIES; i++) {
        const int t = i * 4 + wave, n = t % NT, r = row0 + (t / NT * (GLU ? NT / 2 : NT) + (GLU ? n % (NT / 2) : n)) * 16, first = min(r, p.nrows - 1);
        code_at[i] = of(n).codes + (matrix * p.nrows + first) * (p.K / 2);
        code_off[i] = min(lane >> 2, p.nrows - 1 - first) * (p.K / 2) + chunk * 16;
    }
    const auto copy_codes = [&](int s, int buf) {
        if (cut && s == S - 1 && s * I4_STEP + chunk * 32 >= p.K) {
#pragma unroll
            for (int i = 0; i < COPIES; i++) {
                code_off[i] -= chunk * 16;
            }
        }
#pragma unroll
        for (int i = 0; i < COPIES; i++) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *) (code_at[i] + s * (I4_STEP / 2) + code_off[i]),
                                             (__attribute__((address_space(3))) void *) (lds + CODES + buf * CODE_BYTES + i * 4096 + wave * 1024), 16, 0, 0);
        }
    };
    // scales by blocks of 16 groups, four of its row to a lane of each quarter, a block ahead
    uint64_t sc[NT], sc_next[NT];
    const auto block_of = [&](int s) { return (s * I4_STEP >> p.group_log2) >> 4; };
    const auto first_of = [&](int block, int quarter) { return max(min(block * 16 + quarter * 4, p.n_groups - 4), 0); };
    const auto load_block = [&](int block) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const uint16_t * from = of(n).scales + wave_at * p.n_groups + (uint32_t) (row_off[n] * p.n_groups + first_of(block, q));
            if (p.n_groups >= 4) {
                sc_next[n] = *(const u64_at_2 *) from;
            } else {
                sc_next[n] = from[0] | (uint32_t) from[min(1, p.n_groups - 1)] << 16 | (uint64_t) from[min(2, p.n_groups - 1)] << 32;
            }
        }
    };

    f32x4_t acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            acc[m][n] = f32x4_t{};
        }
    }
    const f32x4_t none = {};
    const auto arrived = [] {
        __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0): this wavefront's copies are in LDS
        __syncthreads();                    // all of them are, and nothing reads the other buffer any more
    };
    // column tiles m * WM + wm are this wavefront's: those that the columns reach are spread over all
    const int mt = ((nc + 15) / 16 - wm + WM - 1) / WM;
    const int tiles = (wm * 16 + m16) * 256;
    const auto operand = [&](int at, int m) { return __builtin_bit_cast(bf16x8_t, *(const u32x4_t *) (lds + at + m * (WM * 4096))); };

    if (E == 1) { // (a longer row's first step comes with the last sums)
        copy_codes(0, 1);
        load_block(0);
    }
    uint32_t zs[4][NT], zz[4][NT]; // scales and zero points of the groups of a step, ahead of the wait
    const auto load_zeros = [&](int step) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (step * 16 + j * 4 >= p.sums_row) {
                break;
            }
            const int gi = min((step * 16 + j * 4 + q) >> (p.group_log2 - p.sum_group_log2), p.n_groups - 1);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint32_t at = row_off[n] * p.n_groups + gi;
                zs[j][n] = (of(n).scales + wave_at * p.n_groups)[at];
                zz[j][n] = of(n).zeros ? (of(n).zeros + wave_at * p.n_groups)[at] : 8u;
            }
        }
    };
    load_zeros(0);
    copy_sums(0, 0);
    if (E == 1) {
        copy(0, 1);
    }
    for (int step = 0; step < E; step++) { // the zero points' part: groups step * 16 ..
        const int buf = step & 1;
        arrived();
        if (step + 1 < E) {
            copy_sums(step + 1, buf ^ 1);
        } else if (E > 1) {
            copy(0, buf ^ 1);
            copy_codes(0, buf ^ 1);
            load_block(0);
        }
        const int left = p.sums_row - step * 16;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j * 4 >= left) {
                break;
            }
            bf16x8_t zf[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float sz = -i4_scale(zs[j][n], of(n).f16 ? ~0u : 0u) * (float) zz[j][n];
                uint32_t a, b, c;
                f32_parts(j * 4 + q < left ? sz : 0.f, a, b, c);
                zf[n] = __builtin_bit_cast(bf16x8_t, u32x4_t{a | a << 16, b | a << 16, b | c << 16, b | c << 16});
            }
#pragma unroll
            for (int m = 0; m < MT; m++) {
                if (LIST && m >= mt) {
                    break;
                }
                const bf16x8_t xf = operand(tiles + buf * (COLS * 256) + ((j * 4 + q) ^ m16) * 16, m);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, zf[n], acc[m][n], 0, 0, 0);
                }
            }
        }
        if (step + 1 < E) {
            load_zeros(step + 1);
        }
    }
    int buf = E & 1;
    int at[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        at[j] = tiles + buf * (COLS * 256) + ((GM == 0 ? q * 4 + j : j * 4 + q) ^ m16) * 16;
    }
    const auto steps = [&](auto tiles_of_columns) {
        constexpr int M = decltype(tiles_of_columns)::value;
        for (int s = 0; s < S; s++) {
            arrived();
            if (s + 1 < S) {
                copy(s + 1, buf ^ 1);
                copy_codes(s + 1, buf ^ 1);
            }
            const int block = block_of(s);
            if (s == 0 || block != block_of(s - 1)) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    sc[n] = sc_next[n];
                }
                if (block < block_of(S - 1)) {
                    load_block(block + 1);
                }
            }
            u32x4_t code[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                code[n] = *(const u32x4_t *) (lds + CODES + buf * CODE_BYTES + (wn * NT + n) * 1024 + m16 * 64 + (q ^ (m16 >> 2)) * 16);
            }
            bf16x8_t wf[NT][4], xs[2][4];
            float sv[NT * NG];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                xs[0][j] = operand(at[j], 0);
            }
            if (cut && s == S - 1 && s * I4_STEP + q * 32 >= p.K) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    code[n] = u32x4_t{};
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const u32x4_t d = GM ? i4_transpose(code[n]) : code[n];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    wf[n][j] = i4_operand_in_order(d[j]);
                }
#pragma unroll
                for (int i = 0; i < NG; i++) {
                    const int g = min((s * I4_STEP + i * (I4_STEP / NG)) >> p.group_log2, p.n_groups - 1);
                    const int quarter = (g >> 2) & 3, e = g - first_of(block, quarter);
                    const uint32_t v = __builtin_amdgcn_ds_bpermute((quarter * 16 + m16) * 4, (uint32_t) (e & 2 ? sc[n] >> 32 : sc[n]));
                    sv[n * NG + i] = i4_scale(v >> (e & 1) * 16 & 0xFFFFu, of(n).f16 ? ~0u : 0u);
                }
            }
            // a tile's products over a group are added up while the matrix cores work on the next ones
            f32x4_t part[2][NT];
#pragma unroll
            for (int u = 0; u <= M * NG; u++) {
                const int m = u / NG, i = u % NG;
                constexpr int J = 4 / NG;
                const bool live = u < M * NG && (!LIST || GM || m < mt);
                if (live) {
                    if (i == 0 && m + 1 < M) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            xs[(m + 1) & 1][j] = operand(at[j], m + 1);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < J; j++) {
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            part[u & 1][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xs[m & 1][i * J + j], wf[n][i * J + j], j ? part[u & 1][n] : none, 0, 0, 0);
                        }
                    }
                }
                if (u > 0) {
                    const int pm = (u - 1) / NG, pi = (u - 1) % NG;
#pragma unroll
                    for (int n = 0; n < NT; n++) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            acc[pm][n][e] = fmaf(sv[n * NG + pi], part[(u - 1) & 1][n][e], acc[pm][n][e]);
                        }
                    }
                }
                if (!live) {
                    break;
                }
                __builtin_amdgcn_sched_barrier(0); // (else the operands of all tiles are read first, and the registers spill)
            }
            const int flip = buf ? -COLS * 256 : COLS * 256;
            buf ^= 1;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                at[j] += flip;
            }
        }
    };
    const auto write = [&](auto tiles_of_columns, auto type) {
        constexpr int M = decltype(tiles_of_columns)::value;
        using T = decltype(type);
        const int r = row0 + wn * (GLU ? NT / 2 : NT) * 16 + m16;
        char * const y_lane = p.y + (int64_t) r * sizeof(T);
#pragma unroll
        for (int m = 0; m < M; m++) {
            if (LIST && m >= mt) {
                break;
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int c = (m * WM + wm) * 16 + q * 4 + e;
                if (c < nc) {
                    T * const y = (T *) (y_lane + (LIST ? y_at[c] : (c0 + c) * p.y_row));
#pragma unroll
                    for (int n = 0; n < (GLU ? NT / 2 : NT); n++) {
                        if (r + n * 16 < p.nrows) {
                            const float v = GLU ? silu(acc[m][n][e]) * acc[m][n + (GLU ? NT / 2 : 0)][e] : acc[m][n][e];
                            if constexpr (sizeof(T) == 2) {
                                y[n * 16] = __builtin_bit_cast(uint16_t, (__bf16) v);
                            } else {
                                y[n * 16] = v;
                            }
                        }
                    }
                }
            }
        }
    };
    const auto run = [&](auto tiles_of_columns) {
        steps(tiles_of_columns);
        if (p.y_bf16) {
            write(tiles_of_columns, uint16_t{});
        } else {
            write(tiles_of_columns, float{});
        }
    };
    // Lists: where a step is within a group, its loop ends at the last tile that has columns.  With smaller groups the branches cost so many
    // registers that two blocks are on a CU where three could be: there two tiles or all four, the columns that are not there along
    // with the others and then left out.  256 experts, 2048 tokens, groups of 64 337 -> 298 us, 32 424 -> 373; 700 tokens, 64 199 -> 171; but groups
    // of 128, 2048 tokens 258 -> 266.  (With the branches held to three blocks: groups of 64 295
    // and, 700 tokens, 177; groups of 32 1303, the registers spill.)
    if (LIST && GM && mt <= 2) {
        run(std::integral_constant<int, 2>());
    } else {
        run(std::integral_constant<int, MT>());
    }
}

// ---------------------------------------------------------------- pairs by matrix

// Every (token, slot) pair under the matrix that its id names, in ascending order, and behind them the pairs whose id
// names none: block e lists the pairs of id e (block n_matrices the others) behind those of the ids below it, which it counts
// itself.  A wavefront takes a contiguous part of the ids and reads it twice, four ids to a lane at a time where they lie in a row
// (VECTOR).  Bound by latency: the ids are in L2.
template <typename ID, bool VECTOR>
__global__ void __launch_bounds__(1024) k_i4_route(const char * ids, int64_t s0, int64_t s1, int n_matrices, int n_pairs, int n_used,
                                                   int32_t * pairs, int32_t * bounds) {
    constexpr int V = VECTOR ? 4 : 1, ROUND = 64 * V;
    typedef ID vec_t __attribute__((ext_vector_type(4)));
    __shared__ int below_w[16], mine_w[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int e = blockIdx.x;
    const int per = ((n_pairs + waves - 1) / waves + ROUND - 1) / ROUND * ROUND;
    const int lo = min(wave * per, n_pairs), hi = min(lo + per, n_pairs);
    // a pair's matrix: n_matrices for ids that name none, -1 behind the last pair
    const auto load = [&](int i, int (&v)[V]) {
        ID at[V];
        if (VECTOR && i + V <= n_pairs) {
            const vec_t four = *(const vec_t *) (ids + (int64_t) i * sizeof(ID));
#pragma unroll
            for (int j = 0; j < V; j++) {
                at[j] = four[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const int p = min(i + j, n_pairs - 1);
                at[j] = VECTOR ? ((const ID *) ids)[p] : *(const ID *) (ids + p / n_used * s1 + p % n_used * s0);
            }
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
            v[j] = i + j >= hi ? -1 : at[j] >= 0 && at[j] < n_matrices ? (int) at[j] : n_matrices;
        }
    };
    int below = 0, mine = 0;
#pragma unroll 4
    for (int b = lo; b < hi; b += ROUND) {
        int v[V];
        load(b + lane * V, v);
#pragma unroll
        for (int j = 0; j < V; j++) {
            below += __popcll(__ballot((unsigned) v[j] < (unsigned) e));
            mine += __popcll(__ballot(v[j] == e));
        }
    }
    if (lane == 0) {
        below_w[wave] = below;
        mine_w[wave] = mine;
    }
    __syncthreads();
    int start = 0, total = 0;
    for (int i = 0; i < waves; i++) {
        start += below_w[i] + (i < wave ? mine_w[i] : 0);
        total += below_w[i] + mine_w[i];
    }
    if (threadIdx.x == 0) {
        bounds[e] = start;
        if (e == n_matrices) {
            bounds[e + 1] = total;
        }
    }
    if (mine == 0) {
        return;
    }
#pragma unroll 4
    for (int b = lo; b < hi; b += ROUND) {
        int v[V];
        load(b + lane * V, v);
        int at = start;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const uint64_t who = __ballot(v[j] == e);
            at += __popcll(who & ((1ull << lane) - 1)); // lanes below: all of their ids come first
            start += __popcll(who);
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
            if (v[j] == e) {
                pairs[at++] = b + lane * V + j;
            }
        }
    }
}

// ---------------------------------------------------------------- dispatch

// LDS of k_i4_few: activations, their groups' sums, the results' places, and two buffers for the parts of K
size_t few_lds(int K, int cols, bool f32, int nt, int nm, int groups_per_step, int ksplit) {
    const size_t steps = (size_t) (K + I4_STEP - 1) / I4_STEP, per_tile = f32 ? 4 : 16;
    return (size_t) cols * (f32 ? 3 : 1) * i4_pitch(K) * 2 + steps * groups_per_step * nt * per_tile * 4 + nt * per_tile * 8
           + (ksplit > 1 ? (size_t) 2 * 8 * 64 * 4 * (f32 ? 1 : 4) * nm * nt : 0);
}

constexpr size_t I4_FEW_LDS = 160 * 1024 - 1024;

// a kernel instance's template arguments as a profiler prints them (bf16n_last_kernel)
std::string text_of(std::initializer_list<int> numbers, std::initializer_list<bool> flags, const char * last = "") {
    std::string s;
    for (const int n : numbers) {
        s += (s.empty() ? "" : ", ") + std::to_string(n);
    }
    for (const bool f : flags) {
        s += f ? ", true" : ", false";
    }
    return s + last;
}

struct few_plan { int nt, grid_y, grid_z, cus; hipStream_t stream; bool raise_limits, small; };

template <int NT, int GM, bool GLU, bool XF32, bool ZEROS>
void launch_few(const i4_launch & p, const few_plan & f) {
    constexpr int NW = 8, NM = GLU ? 2 : 1;
    const auto kernel = k_i4_few<NT, NM, GM, GLU, XF32, ZEROS, NW>;
    if (f.raise_limits) {
        (void) hipFuncSetAttribute((const void *) kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int) I4_FEW_LDS);
        return;
    }
    const int block_rows = NW / p.ksplit * 16;
    const int n_blocks = (p.nrows + block_rows - 1) / block_rows;
    if (f.small) {
        static const std::string text = text_of({NT, GM}, {GLU, XF32, ZEROS});
        note_kernel("k_i4_small", text.c_str(), 0);
        k_i4_small<NT, GM, GLU, XF32, ZEROS><<<dim3(n_blocks, f.grid_y, f.grid_z), NW * 64, 0, f.stream>>>(p);
        return;
    }
    const size_t lds = few_lds(p.K, p.cols_per_pass, XF32, NT, NM, GM == 0 ? 1 : GM == 1 ? 2 : 4, p.ksplit);
    // one matrix: as many blocks as the device holds, each with its share of the rows; more matrices: a block to a piece of rows, or to as
    // many as give a wavefront eight pairs of steps (77 tokens, 2048 x 512 of 256 experts: 66 us with two, 45 with eight)
    const int room = f.cus * (int) std::min<size_t>(2, LDS_BYTES / lds), steps = (p.K + I4_STEP - 1) / I4_STEP;
    const int rounds = f.grid_y == 1 ? (n_blocks + room - 1) / room : std::max(1, std::min<int>(16 * p.ksplit / steps, (int64_t) n_blocks * f.grid_y / (4 * f.cus)));
    static const std::string text = text_of({NT, NM, GM}, {GLU, XF32, ZEROS}, ", 8");
    static_assert(NW == 8, "in the text");
    note_kernel("k_i4_few", text.c_str(), 0);
    kernel<<<dim3((n_blocks + rounds - 1) / rounds, f.grid_y, f.grid_z), NW * 64, lds, f.stream>>>(p);
}

template <int GM, bool ZEROS>
void pick_few(const i4_launch & p, bool glu, bool f32, const few_plan & f) {
    if (glu) {
        f32 ? launch_few<1, GM, true, true, ZEROS>(p, f) : f.nt == 1 ? launch_few<1, GM, true, false, ZEROS>(p, f) : launch_few<2, GM, true, false, ZEROS>(p, f);
    } else {
        f32 ? launch_few<1, GM, false, true, ZEROS>(p, f) : f.nt == 1 ? launch_few<1, GM, false, false, ZEROS>(p, f) : launch_few<2, GM, false, false, ZEROS>(p, f);
    }
}

void pick_few(const i4_launch & p, bool glu, bool f32, int gm, bool zeros, const few_plan & f) {
    zeros ? (gm == 0 ? pick_few<0, true> : gm == 1 ? pick_few<1, true> : pick_few<2, true>)(p, glu, f32, f)
          : (gm == 0 ? pick_few<0, false> : gm == 1 ? pick_few<1, false> : pick_few<2, false>)(p, glu, f32, f);
}

void init_few() {
    for (int i = 0; i < 48; i++) { // every instance
        const i4_launch none = {};
        const few_plan f = {(i & 1) + 1, 0, 0, 0, nullptr, true, false};
        if ((i & 24) != 24) {
            pick_few(none, i & 2, i & 4, i >> 3 & 3, i & 32, f);
        }
    }
}

// LDS of k_i4_many: two pieces of activations and of codes, for lists the places of the results
constexpr size_t many_lds(int cols, int rows, bool list) { return (size_t) 2 * cols * 256 + 2 * rows * 64 + (list ? cols * 8 : 0); }

// an instance of k_i4_many over WM * MT * 16 columns and WN * NT * 16 rows; without p: its LDS limit is raised
template <int WM, int WN, int MT, int NT, int GM, bool LIST>
void launch_many(const i4_many * p, bool glu, unsigned blocks, hipStream_t stream) {
    constexpr int LDS = (int) many_lds(WM * MT * 16, WN * NT * 16, LIST);
    const auto kernel = glu ? k_i4_many<WM, WN, MT, NT, GM, true, LIST> : k_i4_many<WM, WN, MT, NT, GM, false, LIST>;
    if (p) {
        static const std::string text[2] = {text_of({WM, WN, MT, NT, GM}, {false, LIST}), text_of({WM, WN, MT, NT, GM}, {true, LIST})};
        note_kernel("k_i4_many", text[glu].c_str(), 0);
        kernel<<<blocks, 256, LDS, stream>>>(*p);
    } else {
        (void) hipFuncSetAttribute((const void *) kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    }
}

template <int GM> void init_many() {
    for (const bool glu : {false, true}) {
        launch_many<2, 2, 4, 4, GM, false>(nullptr, glu, 0, nullptr);
        launch_many<1, 4, 4, 2, GM, false>(nullptr, glu, 0, nullptr);
        launch_many<1, 4, 4, 2, GM, true>(nullptr, glu, 0, nullptr);
    }
}

template <int GM>
void pick_many(i4_many & p, bool glu, int cols, hipStream_t stream) {
    const bool list = p.bounds != nullptr;
    const int rows = 128 / (glu ? 2 : 1);
    p.row_tiles = (p.nrows + rows - 1) / rows;
    p.col_tiles = (p.ncols + cols - 1) / cols;
    // lists: no more pieces than full ones and one cut short to a matrix
    const int64_t pieces = list ? std::min<int64_t>(p.ncols, p.ncols / cols + p.n_matrices + 1) : p.col_tiles;
    const unsigned n = (unsigned) ((pieces * p.row_tiles + 7) / 8 * 8);
    list ? launch_many<1, 4, 4, 2, GM, true>(&p, glu, n, stream)
         : cols == 128 ? launch_many<2, 2, 4, 4, GM, false>(&p, glu, n, stream) : launch_many<1, 4, 4, 2, GM, false>(&p, glu, n, stream);
}

i4_matrix matrix_of(const bf16n_int4_weight & w) { return {w.codes, (const uint16_t *) w.scales, w.zeros, w.scales_f16 != 0}; }

i4_launch launch_of(const bf16n_int4_weight & w, const bf16n_int4_weight * up, int64_t nrows) {
    i4_launch p = {};
    p.w = matrix_of(w);
    p.up = matrix_of(up ? *up : w);
    p.K = (int) w.K;
    p.group_log2 = 31 - __builtin_clz((unsigned) w.group);
    p.n_groups = (int) ((w.K + w.group - 1) / w.group);
    p.nrows = (int) nrows;
    return p;
}

// the sums of the activations' groups, and the products of many columns
void run_many(const bf16n_int4_weight & w, const bf16n_int4_weight * up, i4_many & p, int64_t x_rows, void * workspace, int cols, hipStream_t stream) {
    p.w = matrix_of(w);
    p.up = matrix_of(up ? *up : w);
    p.K = (int) w.K;
    p.group_log2 = 31 - __builtin_clz((unsigned) w.group);
    p.n_groups = (int) ((w.K + w.group - 1) / w.group);
    p.sum_group_log2 = std::min(p.group_log2, 7);
    const int group = 1 << p.sum_group_log2, per = group / 32;
    p.sums = (const u32x4_t *) workspace;
    p.sums_row = (int) ((w.K + group - 1) / group);
    const int64_t threads = x_rows * ((w.K / 32 + per - 1) / per * per);
    int4 * const table = (int4 *) ((u32x4_t *) workspace + x_rows * p.sums_row);
    p.table = table;
    k_i4_sums<<<(unsigned) ((threads + 255) / 256 + (p.bounds ? 1 : 0)), 256, 0, stream>>>(p.x, p.x_row, p.K, group, x_rows, (u32x4_t *) workspace, p.sums_row,
                                                                                         p.bounds, p.n_matrices, cols, table);
    (p.group_log2 >= 7 ? pick_many<0> : p.group_log2 == 6 ? pick_many<1> : pick_many<2>)(p, up != nullptr, cols, stream);
}

void run_few(i4_launch & p, bool glu, bool f32, bool zeros, int max_cols, int64_t matrices, int grid_y, int cus, hipStream_t stream) {
    const int steps = (p.K + I4_STEP - 1) / I4_STEP;
    const int gm = p.group_log2 >= 7 ? 0 : p.group_log2 == 6 ? 1 : 2;
    // parts of K: as many as make two wavefronts for every SIMD of the device out of the tiles of 16 rows
    const int64_t tiles = (p.nrows + 15) / 16 * matrices;
    int ksplit = 1;
    while (ksplit < 8 && ksplit * 4 <= steps + 1 && tiles * ksplit < 8 * cus) {
        ksplit *= 2;
    }
    const auto fits = [&](int cols, int nt) { return few_lds(p.K, cols, f32, nt, glu ? 2 : 1, 1 << gm, ksplit) <= I4_FEW_LDS; };
    const int nt = !f32 && max_cols > 16 && fits(32, 2) ? 2 : 1;
    p.cols_per_pass = std::min(max_cols, f32 ? 4 : 16 * nt);
    while (!fits(p.cols_per_pass, nt)) {
        p.cols_per_pass--;
    }
    p.ksplit = ksplit;
    const int passes = p.bounds || p.ids ? 1 : std::min(65535, (max_cols + p.cols_per_pass - 1) / p.cols_per_pass);
    // the kernel without activations in LDS: up to two tiles of rows for a CU (one with FP32 activations, whose lanes part them
    // themselves).  us, with it / without, BF16, 16 tokens: 5120 x 2048 9.4 / 10.8, 10240 x 2048 14.5 / 11.7; FP32, three: 8192 x 2048 12.7 / 8.7
    const bool small = tiles <= (f32 ? 1 : 2) * cus;
    pick_few(p, glu, f32, gm, zeros, {nt, grid_y, passes, cus, stream, false, small});
}

} // namespace

void int4_init() {
    init_few();
    init_many<0>();
    init_many<1>();
    init_many<2>();
}

// sums of the activations' groups, and the pieces of lists (at most one of a matrix cut short, one of the pairs without a matrix)
int64_t int4_workspace_bytes(const bf16n_int4_weight & w, int64_t x_rows, int64_t n_pairs, int n_matrices) {
    const int group = std::min(w.group, I4_STEP);
    return x_rows * ((w.K + group - 1) / group) * 16 + (n_pairs ? (n_pairs / 64 + n_matrices + 3) * 16 : 0);
}

void launch_int4_mmv(const bf16n_int4_weight & w, const bf16n_int4_weight * up, const bf16n_mmv_args & a, bool ids_i64, void * workspace,
                     uint64_t workspace_bytes, int cus, hipStream_t stream) {
    // Many columns where one pass of 32 is not all and the matrix has rows enough: its kernel takes 1.1 us a step however few its
    // blocks are (one and a half to a CU add nothing), a pass of 32 columns over 16 rows costs 1 / 800 of that on a whole device.
    // us, many / few: 5120 x 2048, 64 tokens 24.1 / 18.6, 200 25.3 / 50; 233 x 5440, 125 50 / 9.4; 512 x 2048, 512 24.1 / 15.0, 2048 25.7 / 49;
    // 20000 x 2048, 64 24.6 / 36.8
    const int64_t units = (a.nrows + 15) / 16 * ((a.ncols + 31) / 32), blocks = (a.nrows + 127) / 128 * ((a.ncols + 63) / 64);
    const int64_t rounds = std::max<int64_t>(1, 2 * blocks / (3 * cus)), steps = (w.K + I4_STEP - 1) / I4_STEP;
    if (!a.ids && a.x_bf16 && a.ncols > 32 && units > 800 * rounds + 2200 / steps && a.x_tok >= 0 && a.ncols * a.x_tok < (int64_t) 1 << 32 && (int64_t) workspace_bytes >= int4_workspace_bytes(w, a.ncols, 0, 0)) {
        i4_many p = {};
        p.x = (const char *) a.x; p.x_row = a.x_tok;
        p.y = (char *) a.y; p.y_row = a.y_tok; p.y_bf16 = a.y_bf16 != 0;
        p.nrows = (int) a.nrows;
        p.ncols = a.ncols;
        p.n_matrices = 1;
        // tiles of 128 x 128 (two blocks to a CU) where they make two rounds, of 128 x 64 (three) below: 5120 x 2048, 2048 tokens, 640
        // tiles, 77.7 / 69.3 us, 4096 x 2048, 4096 tokens, 1024 tiles, 94.0 / 98.9
        const int64_t tiles = ((a.nrows + 127) / 128) * ((a.ncols + 127) / 128);
        run_many(w, up, p, a.ncols, workspace, tiles >= 4 * cus ? 128 : 64, stream);
        return;
    }
    i4_launch p = launch_of(w, up, a.nrows);
    p.x = (const char *) a.x; p.x_tok = a.x_tok; p.x_slot = a.x_slot;
    p.y = (char *) a.y; p.y_tok = a.y_tok; p.y_slot = a.y_slot; p.y_bf16 = a.y_bf16 != 0;
    p.ncols = a.ncols;
    p.n_used = a.ids ? a.n_used : 1;
    p.x_per_slot = a.x_per_slot > 0 ? a.x_per_slot : 1;
    p.ids = (const char *) a.ids; p.ids_s0 = a.ids_s0; p.ids_s1 = a.ids_s1; p.ids_i64 = ids_i64;
    p.n_matrices = a.ids ? w.rows / a.rows_per_matrix : 1;
    if (a.ids) {
        run_few(p, up != nullptr, !a.x_bf16, w.zeros != nullptr, 1, a.ncols, a.ncols, cus, stream);
    } else {
        run_few(p, up != nullptr, !a.x_bf16, w.zeros != nullptr, a.ncols, 1, 1, cus, stream);
    }
}

void launch_int4_route(const void * ids, bool i64, int64_t s0, int64_t s1, int n_matrices, int n_tok, int n_used, int32_t * pairs, int32_t * bounds,
                       hipStream_t stream) {
    const int n = n_tok * n_used;
    const int threads = n <= 256 ? 256 : 1024;
    const bool row = s0 == (i64 ? 8 : 4) && (s1 == s0 * n_used || n_tok == 1) && (uintptr_t) ids % (4 * s0) == 0;
    (i64 ? row ? k_i4_route<int64_t, true> : k_i4_route<int64_t, false> : row ? k_i4_route<int32_t, true> : k_i4_route<int32_t, false>)
        <<<n_matrices + 1, threads, 0, stream>>>((const char *) ids, s0, s1, n_matrices, n, n_used, pairs, bounds);
}

void launch_int4_mm_ids(const bf16n_int4_weight & w, const bf16n_int4_weight * up, const void * x, int64_t x_row, bool per_slot, const int32_t * pairs,
                        const int32_t * bounds, void * y, bool y_bf16, int64_t y_row, int n_matrices, int n_tok, int n_used, void * workspace, uint64_t workspace_bytes,
                        int cus, hipStream_t stream) {
    const int64_t x_rows = per_slot ? (int64_t) n_tok * n_used : n_tok;
    const int64_t n_pairs = (int64_t) n_tok * n_used;
    // many columns from 12 pairs to a matrix on.  256 experts, top-8, us with them / without: 300 tokens 135 / 131, 400 140 / 150, 512 149 / 177
    if (n_pairs > 12 * (int64_t) n_matrices && x_row >= 0 && x_rows * x_row < (int64_t) 1 << 31 && (int64_t) workspace_bytes >= int4_workspace_bytes(w, x_rows, n_pairs, n_matrices)) {
        i4_many p = {};
        p.x = (const char *) x; p.x_row = x_row * 2;
        p.y = (char *) y; p.y_row = y_row * (y_bf16 ? 2 : 4); p.y_bf16 = y_bf16;
        p.nrows = (int) (w.rows / n_matrices);
        p.ncols = (int) n_pairs;
        p.pairs = pairs; p.bounds = bounds;
        p.n_matrices = n_matrices;
        p.per_token = per_slot ? 1 : n_used; p.one_used = (uint32_t) std::min<uint64_t>(~0u, (1ull << 32) / p.per_token);
        run_many(w, up, p, x_rows, workspace, 64, stream);
        return;
    }
    i4_launch p = launch_of(w, up, w.rows / n_matrices);
    p.x = (const char *) x;
    p.x_tok = p.x_slot = x_row * 2;
    p.x_per_slot = per_slot ? 2 : 1;
    p.y = (char *) y;
    p.y_slot = y_row * (y_bf16 ? 2 : 4);
    p.y_tok = p.y_slot * n_used;
    p.y_bf16 = y_bf16;
    p.ncols = n_tok * n_used;
    p.n_used = n_used;
    p.pairs = pairs; p.bounds = bounds;
    p.n_matrices = n_matrices;
    const int even = (p.ncols + n_matrices - 1) / n_matrices;
    const int cols = std::min(p.ncols, even <= 2 ? 4 : even <= 5 ? 8 : 16); // room for twice an even share
    run_few(p, up != nullptr, false, w.zeros != nullptr, cols, std::min<int64_t>(n_matrices, p.ncols), n_matrices + 1, cus, stream);
}

} // namespace dev
} // namespace bf16n
