// Products with 4-bit weights and group scales (gfx950).
#include "dev_int4.h"
#include "launchers.h"

#include <algorithm>

namespace bf16n {
namespace dev {

namespace {

struct i4_launch {
    i4_matrix w, up;
    int64_t K;                              // columns, a multiple of 32
    int group_log2, n_groups;
    int64_t nrows;                          // rows of one matrix that are multiplied
    const char * x; int64_t x_tok, x_slot;  // bytes
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
__host__ __device__ inline int64_t i4_pitch(int64_t K) { return (K + I4_STEP - 1) / I4_STEP * I4_STEP + 8; }

// Few columns.  One wavefront takes 16 rows of the matrix (of each of the two where they are gated) and 128 columns of it at
// a time: a lane's 16 bytes are 32 codes of row lane % 16, turned into four operands of v_mfma_f32_16x16x32_bf16 whose other
// operand is the activations, from LDS; result: lane = row of the matrix, register = activation row (so that a scale
// is one value to a lane).  FP32 activations are three BF16 rows each (rows 4 t .. 4 t + 2 of the 16: one lane's registers).
// The sums of the activations over a group, which the zero points need, come from one more product with ones.
// Wavefronts of a block share the rows (ksplit parts of K each, summed through LDS in a fixed order) or take other rows.
// Bound by HBM where the matrix is large.
template <int NT, int NM, int GM, bool GLU, bool XF32, int NW>
__global__ void __launch_bounds__(NW * 64) k_i4_few(const i4_launch p) {
    constexpr int U = NM == 1 ? 4 : 2;                  // steps whose codes are loaded ahead
    constexpr int NG = GM == 0 ? 1 : GM == 1 ? 2 : 4;   // groups in a step (128 and more columns, 64, 32)
    constexpr int CPT = XF32 ? 4 : 16;                  // columns in a tile of 16 activation rows
    extern __shared__ __align__(16) char lds[];
    uint16_t * const xs = (uint16_t *) lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m16 = lane & 15, q = lane >> 4;
    const int64_t K = p.K, pitch = i4_pitch(K);
    float * const red = (float *) (lds + (size_t) p.cols_per_pass * (XF32 ? 3 : 1) * pitch * 2);

    // which matrix, and its columns
    int64_t matrix = 0;
    int c_begin = 0, c_end = p.ncols;
    bool named = true;
    if (p.ids) {
        const int t = blockIdx.y / p.n_used, i = blockIdx.y % p.n_used;
        const char * at = p.ids + t * p.ids_s1 + i * p.ids_s0;
        matrix = p.ids_i64 ? *(const int64_t *) at : *(const int32_t *) at;
        named = matrix >= 0 && matrix < p.n_matrices;
        matrix = named ? matrix : 0;
        c_begin = blockIdx.y;
        c_end = c_begin + 1;
    } else if (p.bounds) {
        matrix = blockIdx.y;
        c_begin = p.bounds[matrix];
        c_end = p.bounds[matrix + 1];
        named = matrix < p.n_matrices; // behind the last one: pairs that name none
        matrix = named ? matrix : 0;
    }
    const int64_t row_base = matrix * p.nrows;
    const int row_groups = NW / p.ksplit, kp = wave % p.ksplit;
    constexpr int TILE_ROWS = 16 * (GLU ? 1 : NM);
    const int64_t n_blocks = (p.nrows + (int64_t) row_groups * TILE_ROWS - 1) / (row_groups * TILE_ROWS);
    const auto column = [&](int c, bool slot_of_x) -> int64_t { // byte offset of column c's activations or results
        int t = c, i = 0;
        if (p.pairs) {
            const int pair = p.pairs[c];
            t = pair / p.n_used;
            i = pair % p.n_used;
        } else if (p.ids) {
            t = c / p.n_used;
            i = c % p.n_used;
        }
        return slot_of_x ? t * p.x_tok + (i % p.x_per_slot) * p.x_slot : t * p.y_tok + i * p.y_slot;
    };
    if (!named) { // no such matrix: a row of zeros
        for (int c = c_begin + blockIdx.z; c < c_end; c += gridDim.z) {
            for (int64_t r = blockIdx.x * (int64_t) blockDim.x + threadIdx.x; r < p.nrows; r += (int64_t) gridDim.x * blockDim.x) {
                store_y(p.y + column(c, false), p.y_bf16, r, 0.f);
            }
        }
        return;
    }

    const int steps = (int) ((K + I4_STEP - 1) / I4_STEP);
    const int s0 = steps * kp / p.ksplit, s1 = steps * (kp + 1) / p.ksplit;
    const int n_chunks = (s1 - s0 + U - 1) / U;
    int x_row = m16 < p.cols_per_pass ? m16 : p.cols_per_pass - 1; // rows beyond the columns repeat the last: their results are dropped
    if (XF32) {
        const int t = m16 >> 2, part = m16 & 3;
        x_row = (t < p.cols_per_pass ? t : p.cols_per_pass - 1) * 3 + (part < 3 ? part : 2);
    }

    for (int c0 = c_begin + blockIdx.z * p.cols_per_pass; c0 < c_end; c0 += gridDim.z * p.cols_per_pass) {
        const int nc = min(c_end - c0, p.cols_per_pass);
        // activations into LDS, in the operands' order, zeros behind the last column of the matrix
        const int octs = (int) ((pitch - 8) / 8);
        __syncthreads();
        for (int i = threadIdx.x; i < p.cols_per_pass * octs; i += NW * 64) {
            const int c = i / octs, o = i % octs;
            const bool in = c < nc && o * 8 < K;
            const char * src = p.x + column(c0 + (c < nc ? c : 0), true);
            if constexpr (XF32) {
                f32x4_t a = {}, b = {};
                if (in) {
                    a = *(const f32x4_t *) (src + o * 32);
                    b = *(const f32x4_t *) (src + o * 32 + 16);
                }
                uint32_t parts[3][8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    f32_parts(j < 4 ? a[j & 3] : b[j & 3], parts[0][j], parts[1][j], parts[2][j]);
                }
#pragma unroll
                for (int h = 0; h < 3; h++) {
                    const uint32_t * e = parts[h];
                    *(u32x4_t *) (xs + (c * 3 + h) * pitch + o * 8) =
                        u32x4_t{e[0] | e[2] << 16, e[4] | e[6] << 16, e[1] | e[3] << 16, e[5] | e[7] << 16};
                }
            } else {
                u32x4_t v = {};
                if (in) {
                    v = *(const u32x4_t *) (src + o * 16);
                }
                *(u32x4_t *) (xs + c * pitch + o * 8) = i4_order(v);
            }
        }
        __syncthreads();

        // the codes, scales and zero points of U steps of a tile of rows
        u32x4_t code_a[U * NM], code_b[U * NM];
        uint32_t sc_a[U * NM * NG], sc_b[U * NM * NG], ze_a[U * NM * NG], ze_b[U * NM * NG];
        const auto load = [&](int64_t tile, int chunk, u32x4_t * code, uint32_t * sc, uint32_t * ze) {
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const i4_matrix & w = GLU && m ? p.up : p.w;
                const int64_t r = min(tile * TILE_ROWS + (GLU ? 0 : 16 * m) + m16, p.nrows - 1) + row_base;
                const uint8_t * row = w.codes + r * (K / 2);
                const uint16_t * srow = w.scales + r * p.n_groups;
                const uint8_t * zrow = w.zeros ? w.zeros + r * p.n_groups : nullptr;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int s = min(s0 + chunk * U + u, s1 - 1);
                    const int64_t at = (int64_t) s * I4_STEP + q * 32;
                    code[u * NM + m] = *(const u32x4_t *) (row + (at < K ? at : 0) / 2);
#pragma unroll
                    for (int g = 0; g < NG; g++) {
                        const int gi = min((int) (((int64_t) s * I4_STEP + g * (I4_STEP / NG)) >> p.group_log2), p.n_groups - 1);
                        sc[(u * NM + m) * NG + g] = srow[gi];
                        ze[(u * NM + m) * NG + g] = zrow ? zrow[gi] : 8u;
                    }
                }
            }
        };
        f32x4_t acc[NM * NT];
        int parity = 0;
        const auto compute = [&](int64_t tile, int chunk, const u32x4_t * code, const uint32_t * sc, const uint32_t * ze) {
            if (chunk == 0) {
#pragma unroll
                for (int i = 0; i < NM * NT; i++) {
                    acc[i] = f32x4_t{};
                }
            }
            const f32x4_t none = {};
            const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, u32x4_t{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int s = s0 + chunk * U + u;
                if (s >= s1) {
                    break;
                }
                u32x4_t d[NM];
#pragma unroll
                for (int m = 0; m < NM; m++) {
                    d[m] = GM == 0 ? code[u * NM + m] : i4_transpose(code[u * NM + m]);
                }
                const uint16_t * xat = xs + x_row * pitch + s * I4_STEP + (GM == 0 ? q * 32 : q * 8);
                f32x4_t part[NM * NT], xsum[NT];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    bf16x8_t wf[NM];
#pragma unroll
                    for (int m = 0; m < NM; m++) {
                        wf[m] = i4_operand(d[m][j]);
                    }
                    constexpr int J0 = 4 / NG; // operands of a group
                    const bool first = j % J0 == 0;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        // a second tile of activation rows lies CPT columns on
                        const uint16_t * xt = xat + (t ? (int64_t) (min(x_row + t * CPT * (XF32 ? 3 : 1), p.cols_per_pass * (XF32 ? 3 : 1) - 1) - x_row) * pitch : 0);
                        const bf16x8_t xf = __builtin_bit_cast(bf16x8_t, *(const u32x4_t *) (xt + (GM == 0 ? j * 8 : j * 32)));
                        xsum[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, ones, first ? none : xsum[t], 0, 0, 0);
#pragma unroll
                        for (int m = 0; m < NM; m++) {
                            part[m * NT + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, wf[m], first ? none : part[m * NT + t], 0, 0, 0);
                        }
                    }
                    if (j % J0 == J0 - 1) {
                        const int g = j / J0;
#pragma unroll
                        for (int m = 0; m < NM; m++) {
                            const float sv = i4_scale(sc[(u * NM + m) * NG + g], (GLU && m ? p.up : p.w).f16);
                            const float zv = (float) ze[(u * NM + m) * NG + g];
#pragma unroll
                            for (int t = 0; t < NT; t++) {
#pragma unroll
                                for (int i = 0; i < (XF32 ? 3 : 4); i++) {
                                    acc[m * NT + t][i] = fmaf(sv, fmaf(-zv, xsum[t][i], part[m * NT + t][i]), acc[m * NT + t][i]);
                                }
                            }
                        }
                    }
                }
            }
            if (chunk != n_chunks - 1) {
                return;
            }
            if (p.ksplit > 1) {
                float * const buf = red + (size_t) parity * NW * 64 * 4 * NM * NT;
                parity ^= 1; // the next tile's sums go elsewhere: the barrier in between is one that the readers of this one pass
#pragma unroll
                for (int i = 0; i < NM * NT; i++) {
                    *(f32x4_t *) (buf + ((wave * NM * NT + i) * 64 + lane) * 4) = acc[i];
                }
                __syncthreads();
                if (kp != 0) {
                    return;
                }
                for (int k = 1; k < p.ksplit; k++) {
#pragma unroll
                    for (int i = 0; i < NM * NT; i++) {
                        acc[i] += *(const f32x4_t *) (buf + (((wave + k) * NM * NT + i) * 64 + lane) * 4);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
                for (int i = 0; i < (XF32 ? 1 : 4); i++) {
                    const int c = t * CPT + (XF32 ? q : q * 4 + i);
                    if (c < nc) {
                        char * const y = p.y + column(c0 + c, false);
                        const auto value = [&](int m) {
                            const f32x4_t & a = acc[m * NT + t];
                            return XF32 ? a[0] + (a[1] + a[2]) : a[i];
                        };
                        if constexpr (GLU) {
                            const int64_t r = tile * TILE_ROWS + m16;
                            if (r < p.nrows) {
                                store_y(y, p.y_bf16, r, silu(value(0)) * value(1));
                            }
                        } else {
#pragma unroll
                            for (int m = 0; m < NM; m++) {
                                const int64_t r = tile * TILE_ROWS + 16 * m + m16;
                                if (r < p.nrows) {
                                    store_y(y, p.y_bf16, r, value(m));
                                }
                            }
                        }
                    }
                }
            }
        };

        // the block's tiles, one chunk of steps after the other, the next one's loads ahead of this one's products
        const int64_t mine = (n_blocks - blockIdx.x + gridDim.x - 1) / gridDim.x;
        const int64_t total = mine * n_chunks;
        int64_t lt = 0, ct = 0;
        int lc = 0, cc = 0;
        const auto tile_of = [&](int64_t i) { return (blockIdx.x + i * gridDim.x) * row_groups + wave / p.ksplit; };
        const auto next = [&](int64_t & t, int & c) {
            if (++c == n_chunks) {
                c = 0;
                t++;
            }
        };
        if (total > 0) {
            load(tile_of(0), 0, code_a, sc_a, ze_a);
        }
        for (int64_t it = 0; it < total; it += 2) {
            next(lt, lc);
            if (it + 1 < total) {
                load(tile_of(lt), lc, code_b, sc_b, ze_b);
            }
            compute(tile_of(ct), cc, code_a, sc_a, ze_a);
            next(ct, cc);
            if (it + 1 < total) {
                next(lt, lc);
                if (it + 2 < total) {
                    load(tile_of(lt), lc, code_a, sc_a, ze_a);
                }
                compute(tile_of(ct), cc, code_b, sc_b, ze_b);
                next(ct, cc);
            }
        }
    }
}

// ---------------------------------------------------------------- pairs by matrix

// Every (token, slot) pair under the matrix that its id names, in ascending order, and behind them the pairs whose id
// names none: block e lists the pairs of id e (block n_matrices the others) behind those of the ids below it, which it counts
// itself.  A wavefront takes a contiguous part of the ids and reads it twice.  Bound by latency: the ids are in L2.
__global__ void __launch_bounds__(1024) k_i4_route(const char * ids, int64_t s0, int64_t s1, bool i64, int n_matrices, int n_pairs, int n_used,
                                                   int32_t * pairs, int32_t * bounds) {
    __shared__ int below_w[16], mine_w[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int64_t e = blockIdx.x;
    const int per = ((n_pairs + waves - 1) / waves + 63) / 64 * 64;
    const int lo = min(wave * per, n_pairs), hi = min(lo + per, n_pairs);
    const auto id_of = [&](int i) -> int64_t {
        const char * at = ids + (i / n_used) * s1 + (i % n_used) * s0;
        const int64_t v = i64 ? *(const int64_t *) at : *(const int32_t *) at;
        return v >= 0 && v < n_matrices ? v : n_matrices;
    };
    int below = 0, mine = 0;
#pragma unroll 4
    for (int b = lo; b < hi; b += 64) {
        const int64_t v = b + lane < hi ? id_of(b + lane) : INT64_MAX;
        below += __popcll(__ballot(v < e));
        mine += __popcll(__ballot(v == e));
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
    for (int b = lo; b < hi; b += 64) {
        const bool in = b + lane < hi && id_of(b + lane) == e;
        const uint64_t at = __ballot(in);
        if (in) {
            pairs[start + __popcll(at & ((1ull << lane) - 1))] = b + lane;
        }
        start += __popcll(at);
    }
}

// ---------------------------------------------------------------- dispatch

template <int NT, int NM, int GM, bool GLU, bool XF32>
void launch_few(const i4_launch & p, int grid_y, int grid_z, int cus, hipStream_t stream) {
    constexpr int NW = 8;
    const int64_t row_groups = NW / p.ksplit, tile_rows = 16 * (GLU ? 1 : NM);
    const int64_t n_blocks = (p.nrows + row_groups * tile_rows - 1) / (row_groups * tile_rows);
    const size_t lds = (size_t) p.cols_per_pass * (XF32 ? 3 : 1) * i4_pitch(p.K) * 2 + (p.ksplit > 1 ? 2 * NW * 64 * 16 * NM * NT : 0);
    const int64_t per_cu = std::max<int64_t>(1, std::min<int64_t>(2, (int64_t) (LDS_BYTES / std::max<size_t>(lds, 1))));
    const int64_t room = std::max<int64_t>(1, cus * per_cu / std::max(1, std::min(grid_y, 1 << 20)));
    const int64_t rounds = (n_blocks + room - 1) / room;
    const dim3 grid((unsigned) ((n_blocks + rounds - 1) / rounds), grid_y, grid_z);
    k_i4_few<NT, NM, GM, GLU, XF32, NW><<<grid, NW * 64, lds, stream>>>(p);
}

template <int GM>
void pick_few(const i4_launch & p, bool glu, bool f32, int nt, int grid_y, int grid_z, int cus, hipStream_t stream) {
    if (glu) {
        f32 ? launch_few<1, 2, GM, true, true>(p, grid_y, grid_z, cus, stream)
            : nt == 1 ? launch_few<1, 2, GM, true, false>(p, grid_y, grid_z, cus, stream) : launch_few<2, 2, GM, true, false>(p, grid_y, grid_z, cus, stream);
    } else {
        f32 ? launch_few<1, 1, GM, false, true>(p, grid_y, grid_z, cus, stream)
            : nt == 1 ? launch_few<1, 1, GM, false, false>(p, grid_y, grid_z, cus, stream) : launch_few<2, 1, GM, false, false>(p, grid_y, grid_z, cus, stream);
    }
}

constexpr size_t I4_FEW_LDS = 160 * 1024 - 1024;

template <int GM> void init_few() {
    const auto raise = [](const void * f) { (void) hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int) I4_FEW_LDS); };
    raise((const void *) k_i4_few<1, 2, GM, true, true, 8>);
    raise((const void *) k_i4_few<1, 2, GM, true, false, 8>);
    raise((const void *) k_i4_few<2, 2, GM, true, false, 8>);
    raise((const void *) k_i4_few<1, 1, GM, false, true, 8>);
    raise((const void *) k_i4_few<1, 1, GM, false, false, 8>);
    raise((const void *) k_i4_few<2, 1, GM, false, false, 8>);
}

i4_matrix matrix_of(const bf16n_int4_weight & w) { return {w.codes, (const uint16_t *) w.scales, w.zeros, w.scales_f16 != 0}; }

i4_launch launch_of(const bf16n_int4_weight & w, const bf16n_int4_weight * up, int64_t nrows) {
    i4_launch p = {};
    p.w = matrix_of(w);
    p.up = matrix_of(up ? *up : w);
    p.K = w.K;
    p.group_log2 = 31 - __builtin_clz((unsigned) w.group);
    p.n_groups = (int) ((w.K + w.group - 1) / w.group);
    p.nrows = nrows;
    return p;
}

void run_few(i4_launch & p, bool glu, bool f32, int max_cols, int64_t matrices, int grid_y, int cus, hipStream_t stream) {
    const int64_t pitch = i4_pitch(p.K) * 2 * (f32 ? 3 : 1);
    const int steps = (int) ((p.K + I4_STEP - 1) / I4_STEP);
    const int nm = glu ? 2 : 1;
    int nt = !f32 && max_cols > 16 ? 2 : 1;
    // parts of K: as many as make two wavefronts for every SIMD of the device out of the tiles of 16 rows
    const int64_t tiles = (p.nrows + 15) / 16 * matrices;
    int ksplit = 1;
    while (ksplit < 8 && ksplit * 2 <= steps && tiles * ksplit < 8 * cus) {
        ksplit *= 2;
    }
    const auto red = [&](int tiles_of_cols) { return ksplit > 1 ? (int64_t) 2 * 8 * 64 * 16 * nm * tiles_of_cols : 0; };
    if (nt == 2 && 32 * pitch + red(2) > (int64_t) I4_FEW_LDS) {
        nt = 1;
    }
    const int64_t fit = ((int64_t) I4_FEW_LDS - red(nt)) / pitch;
    p.cols_per_pass = (int) std::min<int64_t>({max_cols, f32 ? 4 : 16 * nt, fit});
    p.ksplit = ksplit;
    const int passes = p.bounds ? 1 : p.ids ? 1 : (max_cols + p.cols_per_pass - 1) / p.cols_per_pass;
    const int gm = p.group_log2 >= 7 ? 0 : p.group_log2 == 6 ? 1 : 2;
    (gm == 0 ? pick_few<0> : gm == 1 ? pick_few<1> : pick_few<2>)(p, glu, f32, nt, grid_y, passes, cus, stream);
}

} // namespace

void int4_init() {
    init_few<0>();
    init_few<1>();
    init_few<2>();
}

void launch_int4_mmv(const bf16n_int4_weight & w, const bf16n_int4_weight * up, const bf16n_mmv_args & a, bool ids_i64, int cus, hipStream_t stream) {
    i4_launch p = launch_of(w, up, a.nrows);
    p.x = (const char *) a.x; p.x_tok = a.x_tok; p.x_slot = a.x_slot;
    p.y = (char *) a.y; p.y_tok = a.y_tok; p.y_slot = a.y_slot; p.y_bf16 = a.y_bf16 != 0;
    p.ncols = a.ncols;
    p.n_used = a.ids ? a.n_used : 1;
    p.x_per_slot = a.x_per_slot > 0 ? a.x_per_slot : 1;
    p.ids = (const char *) a.ids; p.ids_s0 = a.ids_s0; p.ids_s1 = a.ids_s1; p.ids_i64 = ids_i64;
    p.n_matrices = a.ids ? w.rows / a.rows_per_matrix : 1;
    if (a.ids) {
        run_few(p, up != nullptr, !a.x_bf16, 1, a.ncols, a.ncols, cus, stream);
    } else {
        run_few(p, up != nullptr, !a.x_bf16, a.ncols, 1, 1, cus, stream);
    }
}

void launch_int4_route(const void * ids, bool i64, int64_t s0, int64_t s1, int n_matrices, int n_tok, int n_used, int32_t * pairs, int32_t * bounds,
                       hipStream_t stream) {
    const int n = n_tok * n_used;
    const int threads = n <= 256 ? 256 : 1024;
    k_i4_route<<<n_matrices + 1, threads, 0, stream>>>((const char *) ids, s0, s1, i64, n_matrices, n, n_used, pairs, bounds);
}

void launch_int4_mm_ids(const bf16n_int4_weight & w, const bf16n_int4_weight * up, const void * x, int64_t x_row, bool per_slot, const int32_t * pairs,
                        const int32_t * bounds, void * y, bool y_bf16, int64_t y_row, int n_matrices, int n_tok, int n_used, int cus, hipStream_t stream) {
    i4_launch p = launch_of(w, up, w.rows / n_matrices);
    p.x = (const char *) x;
    p.x_tok = x_row * 2 * (per_slot ? n_used : 1);
    p.x_slot = x_row * 2;
    p.x_per_slot = per_slot ? n_used : 1;
    p.y = (char *) y;
    p.y_slot = y_row * (y_bf16 ? 2 : 4);
    p.y_tok = p.y_slot * n_used;
    p.y_bf16 = y_bf16;
    p.ncols = n_tok * n_used;
    p.n_used = n_used;
    p.pairs = pairs; p.bounds = bounds;
    p.n_matrices = n_matrices;
    const int64_t even = (p.ncols + n_matrices - 1) / n_matrices;
    run_few(p, up != nullptr, false, (int) std::min<int64_t>(p.ncols, std::max<int64_t>(16, even + even / 2)), std::min<int64_t>(n_matrices, p.ncols),
            n_matrices + 1, cus, stream);
}

} // namespace dev
} // namespace bf16n
