// Matrices orthogonalised by Newton-Schulz products: with X = M / (|M| + eps) (|M| the Frobenius norm, X with the
// shorter side s as rows and the longer l as columns), `steps` times
//   G = X X^T,  B = b G + c G G,  X = a X + B X,
// after which X's singular values lie near 1 (each went through x (a + b x^2 + c x^4)).
//
// Precision. The polynomial raises small singular values by up to a each step (485 times in five), and with them
// whatever error the products have: in 16-bit products it would be a tenth of the result. So every matrix is held as
// the sum of two float16 values, hi + lo, within 2^-23 of it, and a product is hi hi + (hi lo + lo hi) on the matrix
// cores, added in float32 (the splitting of single-precision products that Ootomo and Yokota published in 2022): as near
// to the definition as float32 products, at three times the cost of one float16 product instead of the sixteen that the
// matrix cores' float32 rate is below it. Of at most 64 rows, where the matrix cores are not what counts, lo lo (2^-25 of
// a product as a rule, of one sign in G's diagonal) is added too; of at most 8 rows all is in 64 bits. Off by, of the
// result's norm: 1024 x 4096 1.5e-6 (the same steps in float32: 4.1e-6 with the library's products, 1.4e-6 on the host);
// 64 x 576 of normal values 1.4e-6 (1.7e-6 and 1.4e-6; without lo lo 1.8e-6).
// Values are held 2^12 times as large, which keeps hi out of float16's subnormals and lo's steps below 2^-36; float16 ends
// at 16 times that, so a polynomial must keep X below 3.5, G's largest root, and b x^2 + c x^4, B's, below 15.9.
//
// Layout. A matrix lies in memory with both sides padded to whole tiles. Behind the last value there are zeros up to
// the next multiple of 64; beyond it, in the padding to 128, a small tile leaves what was there, which only reaches rows and
// columns that are padding themselves: no product reads that far along k. A row's 32 neighbouring values are 64 bytes of
// hi and 64 of lo, so that one step of a product reads a cache line of each row. Every product is of the form A B^T
// with rows of both read along k: X is kept as X and as X^T. Symmetric products form the tiles on and below the
// diagonal and write them to both places.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <numeric>
#include <vector>

#include "common.h"
#include "hand_over.h"
#include "typed.h"
#include "wave.h"

namespace mfh {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int THREADS = 256;
constexpr int K_STEP = 32;          // values of a row in one step: 128 bytes, hi and lo
constexpr int ROW_STEP = 2 * K_STEP;  // halves
constexpr int LARGE = 128, SMALL = 64;  // sides of a workgroup's tile
constexpr int SCALE_LOG = 12;
constexpr float SCALE = 1 << SCALE_LOG, UNSCALE = 1.0f / SCALE;
constexpr int GROUP = 30;  // matrices of a launch: their descriptors travel in its arguments
constexpr int XCD_COUNT = 8;
constexpr std::int64_t PARTS_BYTES = 48 << 20;  // workspace of split tiles' sums

// out = alpha A B^T + beta add, or the caller's matrix in its type.
struct Product {
    const _Float16* a;  // rows of A and of B
    const _Float16* b;
    const _Float16* add_t;  // optional, transposed (a symmetric one is its own)
    _Float16* out;          // optional
    _Float16* out_t;        // optional, transposed
    void* final;
    std::int64_t final_stride;
    float* parts;        // where the steps of a tile are split over workgroups: their sums,
    unsigned* arrived;   // and how many have come, a tile
    float alpha, beta;
    int ksteps, m_tiles, n_tiles;  // what holds values, in steps and in tiles of its own side
    int k_padded, m_padded, n_padded;  // the sides as they lie in memory
    int whole, splits;  // tiles of one workgroup each, and the parts of each tile behind them
    int rows, cols;                // of the caller's matrix, the shorter side as rows
    bool over_longer, symmetric, small, tall;  // the sums' side; tall: the caller's matrix is the transposed result
};

struct ProductGroup {
    Product p[GROUP];
    int first_unit[GROUP + 1];
    int round;  // the first units, which are dealt to the dies in runs
};
static_assert(sizeof(ProductGroup) <= 4096, "descriptors must fit the kernel arguments");

// Rows lie in LDS 128 bytes apart, half of its 64 banks, their eight 16-byte parts in the order part ^ key: a 16-byte read
// is served 16 lanes at a time, of neighbouring rows or, as the hardware pairs them, of four groups of four, and the
// key gives those of one parity other parts.
__device__ __forceinline__ int key_of(int row) { return row >> 1 & 7; }

// One step of a tile's rows on their way through registers to LDS, 16 bytes a lane. (Loads straight to LDS would spare
// the registers, but the compiler lets no LDS read pass one that is under way.)
template <int SIDE>
struct StagedRows {
    static constexpr int EACH = SIDE / 8 / (THREADS / 64);  // instructions of a wave, 8 rows each
    half8 v[EACH];

    __device__ __forceinline__ void load(const _Float16* __restrict__ lane_rows, std::int64_t pitch, int step) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) v[i] = *reinterpret_cast<const half8*>(lane_rows + i * 8 * pitch + step * ROW_STEP);
    }
    __device__ __forceinline__ void store(_Float16* lds) const {
        const int lane = threadIdx.x & 63, row = threadIdx.x / 64 * EACH * 8 + lane / 8;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            *reinterpret_cast<half8*>(lds + (row + i * 8) * ROW_STEP + ((lane & 7) ^ key_of(row + i * 8)) * 8) = v[i];
    }
    // This lane's first part of the tile's rows.
    static __device__ __forceinline__ const _Float16* lane_rows(const _Float16* rows, std::int64_t pitch) {
        const int lane = threadIdx.x & 63;
        return rows + (threadIdx.x / 64 * EACH * 8 + lane / 8) * pitch + (lane & 7) * 8;
    }
};

// The lane's 8 values of a 32 x 16 operand at LDS row `row` (its own lane % 32 included): part p of hi, or of lo.
__device__ __forceinline__ half8 operand(const _Float16* lds, int row, int part) {
    return *reinterpret_cast<const half8*>(lds + row * ROW_STEP + (part ^ key_of(row)) * 8);
}

// One term of a product of two pieces, hi and lo: hi hi, added to `sum`, or hi lo, lo hi or lo lo, added to `cross`. These are
// 2^-11 of hi hi: on their own they are added without a rounding of the whole sum each. With one sum for all three the
// result's error was half as large again (4096 x 4096: 2.3e-6 of it for 1.3e-6, 1024 x 4096: 2.2e-6 for 1.5e-6), in
// no less time.
__device__ __forceinline__ void add_term(int term, const half8 (&x)[2], const half8 (&y)[2], float16v& sum, float16v& cross) {
    float16v& to = term == 0 ? sum : cross;
    to = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[term / 2], y[term % 2], to, 0, 0, 0);
}

// A wave's scratch in LDS: 32 rows of a matrix as they lie in memory, 64 bytes of hi and 64 of lo each, their eight
// 16-byte parts stored as the operands' are; or 32 x 33 floats. Through it the lanes read and write whole lines of
// memory: straight from the registers, where a lane has four neighbours of one column, a line took 8 stores of 8
// bytes, or 64 of two.
constexpr int SCRATCH = 32 * 33 * 2;  // halves

__device__ __forceinline__ _Float16* scratch_at(_Float16* scratch, int row, int value, int low) {
    return scratch + row * ROW_STEP + ((value / 8 + 4 * low) ^ key_of(row)) * 8 + value % 8;
}

// Part lane % 8 of rows lane / 8 + 8 r: of the scratch, or of the 32 x 32 piece at `at` of a matrix.
__device__ __forceinline__ half8* scratch_part(_Float16* scratch, int r) {
    const int lane = threadIdx.x & 63, row = 8 * r + lane / 8;
    return reinterpret_cast<half8*>(scratch + row * ROW_STEP + ((lane & 7) ^ key_of(row)) * 8);
}
template <typename Half>
__device__ __forceinline__ Half* piece_part(Half* matrix, int row0, int col0, std::int64_t pitch, int r) {
    const int lane = threadIdx.x & 63;
    return matrix + (row0 + 8 * r + lane / 8) * pitch + col0 / K_STEP * ROW_STEP + (lane & 7) * 8;
}

__device__ __forceinline__ void write_scratch(_Float16* scratch, _Float16* matrix, int row0, int col0, std::int64_t pitch) {
    wave_order();
#pragma unroll
    for (int r = 0; r < 4; ++r) *reinterpret_cast<half8*>(piece_part(matrix, row0, col0, pitch, r)) = *scratch_part(scratch, r);
    wave_order();
}

template <typename T, typename P>
__device__ __forceinline__ void write_final(const P& p, const float (&v)[16], int i0, int j0, _Float16* scratch) {
    const int lane = threadIdx.x & 63;
    T* out = static_cast<T*>(p.final);
    if (!p.tall) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int i = i0 + e / 4 * 8 + lane / 32 * 4 + e % 4, j = j0 + (lane & 31);
            if (i < p.rows && j < p.cols) out[i * p.final_stride + j] = static_cast<T>(v[e]);
        }
        return;
    }
    float* tile = reinterpret_cast<float*>(scratch);
#pragma unroll
    for (int e = 0; e < 16; ++e) tile[(lane & 31) * 33 + e / 4 * 8 + lane / 32 * 4 + e % 4] = v[e];
    wave_order();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int row = e * 2 + lane / 32, i = i0 + (lane & 31), j = j0 + row;
        if (i < p.rows && j < p.cols) out[j * p.final_stride + i] = static_cast<T>(tile[row * 33 + (lane & 31)]);
    }
    wave_order();
}

// A wave's pieces of 32 x 32 from (i0, j0) on. A lane has column lane % 32 of a piece and its rows 8 q + 4 (lane / 32)
// + 0 .. 3.
template <int PIECES, typename T>
__device__ __forceinline__ void write_pieces(const Product& p, const float16v (&sum)[PIECES][PIECES], int i_first, int j_first,
                                             bool mirrored, _Float16* scratch) {
    const int lane = threadIdx.x & 63, column = lane & 31, high = lane / 32;
    const std::int64_t pitch = p.n_padded * 2, pitch_t = p.m_padded * 2;
    const float alpha = p.alpha * UNSCALE;
    half8 add[PIECES][PIECES][4];
    if (p.add_t) {
#pragma unroll
        for (int pi = 0; pi < PIECES; ++pi)
#pragma unroll
            for (int pj = 0; pj < PIECES; ++pj)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    add[pi][pj][r] = *reinterpret_cast<const half8*>(piece_part(p.add_t, j_first + 32 * pj, i_first + 32 * pi, pitch_t, r));
    }
#pragma unroll
    for (int pi = 0; pi < PIECES; ++pi)
#pragma unroll
        for (int pj = 0; pj < PIECES; ++pj) {
            const int i0 = i_first + 32 * pi, j0 = j_first + 32 * pj;
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = sum[pi][pj][e] * alpha;
            if (p.add_t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) *scratch_part(scratch, r) = add[pi][pj][r];
                wave_order();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const half4 hi = *reinterpret_cast<const half4*>(scratch_at(scratch, column, 8 * q + 4 * high, 0));
                    const half4 lo = *reinterpret_cast<const half4*>(scratch_at(scratch, column, 8 * q + 4 * high, 1));
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[4 * q + k] += p.beta * (static_cast<float>(hi[k]) + static_cast<float>(lo[k]));
                }
                wave_order();
            }
            if (p.final) {
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] *= UNSCALE;
                write_final<T>(p, v, i0, j0, scratch);
                continue;
            }
            half4 hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                hi[e / 4][e % 4] = static_cast<_Float16>(v[e]);
                lo[e / 4][e % 4] = static_cast<_Float16>(v[e] - static_cast<float>(hi[e / 4][e % 4]));
            }
            if (p.out_t) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    *reinterpret_cast<half4*>(scratch_at(scratch, column, 8 * q + 4 * high, 0)) = hi[q];
                    *reinterpret_cast<half4*>(scratch_at(scratch, column, 8 * q + 4 * high, 1)) = lo[q];
                }
                write_scratch(scratch, p.out_t, j0, i0, pitch_t);
            }
            if (mirrored) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int row = e / 4 * 8 + 4 * high + e % 4;
                    *scratch_at(scratch, row, column, 0) = hi[e / 4][e % 4];
                    *scratch_at(scratch, row, column, 1) = lo[e / 4][e % 4];
                }
                write_scratch(scratch, p.out, i0, j0, pitch);
            }
        }
}

// The sums of a tile's parts, in their order, by the workgroup that comes last; false for the others.
template <int SUMS, typename P>
__device__ __forceinline__ bool join_parts(const P& p, int tile, int part, float (&sum)[SUMS]) {
    __shared__ unsigned last;
    static_assert(SUMS % 2 == 0, "two sums a store");
    using Two = unsigned long long;
    Two* parts = reinterpret_cast<Two*>(p.parts) + static_cast<std::int64_t>(tile) * p.splits * (SUMS / 2) * THREADS + threadIdx.x;
#pragma unroll
    for (int i = 0; i < SUMS / 2; ++i) {
        const float two[2] = {sum[2 * i], sum[2 * i + 1]};
        hand_over(parts + (static_cast<std::int64_t>(part) * (SUMS / 2) + i) * THREADS, __builtin_bit_cast(Two, two));
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the sums are where every die sees them
    __syncthreads();
    if (threadIdx.x == 0) {
        last = __hip_atomic_fetch_add(p.arrived + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == static_cast<unsigned>(p.splits);
        if (last) hand_over(p.arrived + tile, 0u);
    }
    __syncthreads();
    if (!last) return false;
#pragma unroll
    for (int i = 0; i < SUMS; ++i) sum[i] = 0.0f;
    constexpr int TOGETHER = 64 / SUMS > 1 ? 64 / SUMS : 2;  // parts whose sums are on their way at once
    for (int first = 0; first < p.splits; first += TOGETHER) {
        Two two[TOGETHER][SUMS / 2];
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k) {
            if (first + k >= p.splits) break;
            const Two* from = parts + static_cast<std::int64_t>(first + k) * (SUMS / 2) * THREADS;
#pragma unroll
            for (int i = 0; i < SUMS / 2; ++i) two[k][i] = handed_over(from + i * THREADS);
        }
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k) {
            if (first + k >= p.splits) break;
#pragma unroll
            for (int i = 0; i < SUMS / 2; ++i) {
                sum[2 * i] += __uint_as_float(static_cast<unsigned>(two[k][i]));
                sum[2 * i + 1] += __uint_as_float(static_cast<unsigned>(two[k][i] >> 32));
            }
        }
    }
    return true;
}

// One SIDE x SIDE tile, or the steps of one part of it, by four waves of SIDE / 2 x SIDE / 2. Two steps lie in LDS, a
// step has two halves of 16 k. While one half is multiplied the other's operands are read from LDS and the next step's
// rows are stored there, in the place of the step before, which all waves have read: one barrier a step. 4096 x 4096:
// B X 385 us, 1.07 PFLOP/s of float16 products (a float16 product of 8192^3 by the library: 1.22), the matrix cores
// 65 % busy at the 1.7 GHz that the card then runs at.
template <int SIDE, typename T>
__device__ __forceinline__ void tile_product(const Product& p, int tile_i, int tile_j, int tile, int part, int parts, _Float16* lds) {
    constexpr int PIECES = SIDE / 64, STAGE = SIDE * ROW_STEP;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wave_i = wave / 2 * (SIDE / 2), wave_j = wave % 2 * (SIDE / 2);
    const std::int64_t pitch = p.k_padded * 2;
    const _Float16* a = p.a + static_cast<std::int64_t>(tile_i) * SIDE * pitch;
    const _Float16* b = p.b + static_cast<std::int64_t>(tile_j) * SIDE * pitch;
    const int begin = static_cast<int>(static_cast<long long>(p.ksteps) * part / parts);
    const int end = static_cast<int>(static_cast<long long>(p.ksteps) * (part + 1) / parts);
    float16v sum[PIECES][PIECES] = {}, cross[PIECES][PIECES] = {};
    const bool few = p.rows <= SMALL;  // products with lo lo
    struct Operands {
        half8 x[PIECES][2], y[PIECES][2];  // hi and lo
    };
    // AHEAD steps are in registers, or on their way there.
    constexpr int AHEAD = SIDE == SMALL ? 2 : 1;  // as many as leave four small tiles or two large ones a CU
    StagedRows<SIDE> rows_a[AHEAD], rows_b[AHEAD];
    const _Float16 *lane_a = StagedRows<SIDE>::lane_rows(a, pitch), *lane_b = StagedRows<SIDE>::lane_rows(b, pitch);
    const auto load = [&](int place, int step) {  // beyond the last step, that one again
        rows_a[place].load(lane_a, pitch, min(step, end - 1));
        rows_b[place].load(lane_b, pitch, min(step, end - 1));
    };
    const auto store = [&](int place, int step) {
        _Float16* to = lds + ((step - begin) & 1) * 2 * STAGE;
        rows_a[place].store(to);
        rows_b[place].store(to + STAGE);
    };
    const auto read = [&](int step, int half) {
        const _Float16* at = lds + ((step - begin) & 1) * 2 * STAGE;
        Operands o;
#pragma unroll
        for (int piece = 0; piece < PIECES; ++piece)
#pragma unroll
            for (int low = 0; low < 2; ++low) {
                o.x[piece][low] = operand(at, wave_i + piece * 32 + (lane & 31), low * 4 + half * 2 + lane / 32);
                o.y[piece][low] = operand(at + STAGE, wave_j + piece * 32 + (lane & 31), low * 4 + half * 2 + lane / 32);
            }
        return o;
    };
    const auto multiply = [&](const Operands& o) {
#pragma unroll
        for (int term = 0; term < 4; ++term) {
            if (term == 3 && (SIDE != SMALL || !few)) break;
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
                for (int j = 0; j < PIECES; ++j) add_term(term, o.x[i], o.y[j], sum[i][j], cross[i][j]);
        }
    };
    load(0, begin);
    store(0, begin);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) load(k, begin + 1 + k);
    __syncthreads();
    Operands first = read(begin, 0);
    for (int base = begin; base < end; base += AHEAD) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int step = base + k;
            if (step >= end) break;
            const Operands second = read(step, 1);
            store(k, step + 1);  // where the step before this one was, which all waves have read
            load(k, step + 1 + AHEAD);
            // The compiler would sink the reads to their uses, and wait for each there.
            __builtin_amdgcn_sched_barrier(0);
            multiply(first);
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
            first = read(step + 1, 0);
            __builtin_amdgcn_sched_barrier(0);
            multiply(second);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __syncthreads();  // LDS is free
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int j = 0; j < PIECES; ++j) sum[i][j] += cross[i][j];
    if (parts > 1) {
        float flat[PIECES * PIECES * 16];
#pragma unroll
        for (int e = 0; e < PIECES * PIECES * 16; ++e) flat[e] = sum[e / 16 / PIECES][e / 16 % PIECES][e % 16];
        if (!join_parts(p, tile - p.whole, part, flat)) return;
#pragma unroll
        for (int e = 0; e < PIECES * PIECES * 16; ++e) sum[e / 16 / PIECES][e / 16 % PIECES][e % 16] = flat[e];
    }
    write_pieces<PIECES, T>(p, sum, tile_i * SIDE + wave_i, tile_j * SIDE + wave_j, p.out && (!p.symmetric || tile_i != tile_j),
                            lds + wave * SCRATCH);
}

// LARGEST: the side of the launch's largest tiles, for which LDS is held.
template <int LARGEST, typename T>
__global__ __launch_bounds__(THREADS, 2) void product_kernel(ProductGroup group) {
    __shared__ __align__(1024) _Float16 lds[4 * LARGEST * ROW_STEP];
    // Neighbouring units of the first round go to the same die: workgroups are dealt to the dies in turn.
    int unit = blockIdx.x;
    if (unit < group.round) {
        const int die = unit % XCD_COUNT, share = group.round / XCD_COUNT, more = group.round % XCD_COUNT;
        unit = die * share + min(die, more) + unit / XCD_COUNT;
    }
    int item = 0;
    while (unit >= group.first_unit[item + 1]) ++item;
    const Product& p = group.p[item];
    const int within = unit - group.first_unit[item], beyond = within - p.whole;
    const int t = beyond < 0 ? within : p.whole + beyond / p.splits, part = beyond < 0 ? 0 : beyond % p.splits;
    const int parts = beyond < 0 ? 1 : p.splits;
    int i, j;
    if (p.symmetric) {  // the tiles on and below the diagonal, row by row
        i = static_cast<int>((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
        while (i * (i + 1) / 2 > t) --i;
        while ((i + 1) * (i + 2) / 2 <= t) ++i;
        j = t - i * (i + 1) / 2;
    } else {  // columns of eight tiles, so that a die's tiles share rows of both operands
        const int width = 8 * p.n_tiles, first = t / width * 8, rows = min(8, p.m_tiles - first), place = t % width;
        i = first + place % rows, j = place / rows;
    }
    if (LARGEST == SMALL || p.small) tile_product<SMALL, T>(p, i, j, t, part, parts, lds);
    else tile_product<LARGEST, T>(p, i, j, t, part, parts, lds);
}

// ---- before the products ----------------------------------------------------------------------
struct Source {
    const void* in;
    std::int64_t stride;
    _Float16* same;     // the split matrix as the caller has it, and transposed
    _Float16* across;
    double* squares;    // sums of squares, one a workgroup of squares_kernel
    int rows, cols, padded_rows, padded_cols;
    FastDiv columns;
};

struct SourceGroup {
    Source s[GROUP];
    int first_block[GROUP + 1];
    int square_blocks[GROUP];
    float eps;
};
static_assert(sizeof(SourceGroup) <= 4096, "descriptors must fit the kernel arguments");

constexpr int SQUARES_EACH = 16384;  // elements of a workgroup, while they are at most SQUARES_BLOCKS
constexpr int SQUARES_BLOCKS = 256;

template <typename Group>
__device__ __forceinline__ int item_of(const Group& group, unsigned block) {
    int item = 0;
    while (block >= static_cast<unsigned>(group.first_block[item + 1])) ++item;
    return item;
}

__device__ __forceinline__ double wave_total(double v) {
    for (int o = 32; o > 0; o /= 2) v += __shfl_xor(v, o);
    return v;
}

// The squares are added in 64 bits: no float32 overflows them.
template <typename T>
__global__ __launch_bounds__(THREADS) void squares_kernel(SourceGroup group) {
    __shared__ double parts[THREADS / 64];
    const int item = item_of(group, blockIdx.x), block = blockIdx.x - group.first_block[item], blocks = group.square_blocks[item];
    const Source& s = group.s[item];
    const T* in = static_cast<const T*>(s.in);
    const long long count = static_cast<long long>(s.rows) * s.cols, each = (count + blocks - 1) / blocks;
    const long long begin = block * each, end = min(begin + each, count);
    double sum = 0.0;
#pragma unroll 8
    for (long long at = begin + threadIdx.x; at < end; at += THREADS) {
        int column;
        const int row = s.columns.divmod(static_cast<int>(at), column);
        const double v = static_cast<float>(in[row * s.stride + column]);
        sum += v * v;
    }
    sum = wave_total(sum);
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0) s.squares[block] = parts[0] + parts[1] + parts[2] + parts[3];
}

// 64 x 64 values of a matrix, scaled, split and written in both orientations, with zeros in the padding.
template <typename T>
__global__ __launch_bounds__(THREADS) void split_kernel(SourceGroup group) {
    __shared__ float tile[64][65];
    __shared__ double factor;  // products in 64 bits: of the smallest norms it lies beyond float32
    const int item = item_of(group, blockIdx.x), tid = threadIdx.x;
    const Source& s = group.s[item];
    if (tid < 64) {
        double sum = 0.0;
        for (int i = tid; i < group.square_blocks[item]; i += 64) sum += s.squares[i];
        sum = wave_total(sum);
        if (tid == 0) factor = static_cast<double>(SCALE) / (sqrt(sum) + static_cast<double>(group.eps));
    }
    __syncthreads();
    const int block = blockIdx.x - group.first_block[item], across = s.padded_cols / 64;
    const int row0 = block / across * 64, col0 = block % across * 64;
    const T* in = static_cast<const T*>(s.in);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int row = k * 4 + tid / 64, col = tid & 63;
        const bool there = row0 + row < s.rows && col0 + col < s.cols;
        tile[row][col] = there ? static_cast<float>(static_cast<float>(in[(row0 + row) * s.stride + col0 + col]) * factor) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int row = (k * THREADS + tid) / 8, part = (k * THREADS + tid) % 8;
        half8 hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v[2] = {tile[row][part * 8 + e], tile[part * 8 + e][row]};
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                hi[o][e] = static_cast<_Float16>(v[o]);
                lo[o][e] = static_cast<_Float16>(v[o] - static_cast<float>(hi[o][e]));
            }
        }
        const int at = part * 8 / K_STEP * ROW_STEP + part * 8 % K_STEP;
        _Float16* same = s.same + static_cast<std::int64_t>(row0 + row) * s.padded_cols * 2 + col0 * 2 + at;
        _Float16* other = s.across + static_cast<std::int64_t>(col0 + row) * s.padded_rows * 2 + row0 * 2 + at;
        *reinterpret_cast<half8*>(same) = hi[0];
        *reinterpret_cast<half8*>(same + K_STEP) = lo[0];
        *reinterpret_cast<half8*>(other) = hi[1];
        *reinterpret_cast<half8*>(other + K_STEP) = lo[1];
    }
}

// ---- matrices of one tile's width -------------------------------------------------------------
// With at most 64 rows, G is one tile. A workgroup takes some of X's columns through a whole step: it forms its new
// columns from B, writes them, and adds their part of the next G; the workgroup that comes last joins the parts and forms
// the next B. One launch a step instead of three: for such matrices the launches are what takes the time (64 x 576
// float32 in five steps: a call takes 68 us, 100 with the products above).
struct Narrow {
    const _Float16* x;  // rows of X, for the first G; then null
    _Float16* x_t;      // X^T, rows of 64
    _Float16* b;
    float* parts;
    unsigned* arrived;
    void* final;
    std::int64_t final_stride;
    int rows, cols, x_pitch, tiles, each, splits;  // tiles of 64 columns, those of a workgroup, workgroups
    bool tall;
};

struct NarrowGroup {
    Narrow m[GROUP];
    int first_block[GROUP + 1];
    float a, b, c;
};
static_assert(sizeof(NarrowGroup) <= 4096, "descriptors must fit the kernel arguments");

constexpr int NARROW_STEP = SMALL * ROW_STEP;  // halves of 64 rows in one step; a tile has two steps

// The tile's two steps from memory to LDS.
__device__ __forceinline__ void stage_tile(const _Float16* rows, std::int64_t pitch, _Float16* lds) {
    StagedRows<SMALL> staged[2];
    const _Float16* lane_rows = StagedRows<SMALL>::lane_rows(rows, pitch);
#pragma unroll
    for (int step = 0; step < 2; ++step) staged[step].load(lane_rows, pitch, step);
#pragma unroll
    for (int step = 0; step < 2; ++step) staged[step].store(lds + step * NARROW_STEP);
}

// This wave's 32 x 32 piece of x y^T, over the 64 values of the rows of both, added to sum + cross.
__device__ __forceinline__ void multiply_tile(const _Float16* x, const _Float16* y, int wave_i, int wave_j, float16v& sum,
                                              float16v& cross) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        half8 a[2], b[2];
#pragma unroll
        for (int low = 0; low < 2; ++low) {
            a[low] = operand(x + k / 2 * NARROW_STEP, wave_i + (lane & 31), low * 4 + k % 2 * 2 + lane / 32);
            b[low] = operand(y + k / 2 * NARROW_STEP, wave_j + (lane & 31), low * 4 + k % 2 * 2 + lane / 32);
        }
#pragma unroll
        for (int term = 0; term < 4; ++term) add_term(term, a, b, sum, cross);
    }
}

__device__ __forceinline__ void split_piece(const float (&v)[16], half4 (&hi)[4], half4 (&lo)[4]) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        hi[e / 4][e % 4] = static_cast<_Float16>(v[e]);
        lo[e / 4][e % 4] = static_cast<_Float16>(v[e] - static_cast<float>(hi[e / 4][e % 4]));
    }
}

// The lane's column of a piece, as 16 of the 32 values of row `row`, at 32 rows of a step in LDS.
__device__ __forceinline__ void write_quads(_Float16* step, int row, const half4 (&hi)[4], const half4 (&lo)[4]) {
    const int high = (threadIdx.x & 63) / 32;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        *reinterpret_cast<half4*>(scratch_at(step, row, 8 * q + 4 * high, 0)) = hi[q];
        *reinterpret_cast<half4*>(scratch_at(step, row, 8 * q + 4 * high, 1)) = lo[q];
    }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void narrow_kernel(NarrowGroup group) {
    __shared__ __align__(1024) _Float16 columns[2 * NARROW_STEP], factor[2 * NARROW_STEP], rows[2 * NARROW_STEP];
    __shared__ __align__(16) _Float16 scratches[THREADS / 64 * SCRATCH];
    const int item = item_of(group, blockIdx.x), part = blockIdx.x - group.first_block[item];
    const Narrow& m = group.m[item];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wave_i = wave / 2 * 32, wave_j = wave % 2 * 32, column = lane & 31, high = lane / 32;
    _Float16* scratch = scratches + wave * SCRATCH;
    constexpr std::int64_t PITCH = 2 * SMALL;
    float16v gram = {}, gram_cross = {};
    half4 hi[4], lo[4];
    float v[16];
    if (!m.x) stage_tile(m.b, PITCH, factor);
    for (int tile = part * m.each; tile < min((part + 1) * m.each, m.tiles); ++tile) {
        if (m.x) {
            stage_tile(m.x + tile * PITCH, m.x_pitch, rows);
        } else {
            stage_tile(m.x_t + tile * SMALL * PITCH, PITCH, columns);
            __syncthreads();
            float16v sum = {}, cross = {};
            multiply_tile(factor, columns, wave_i, wave_j, sum, cross);
            sum += cross;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const _Float16* step = columns + wave_i / 32 * NARROW_STEP;
                const half4 old_hi = *reinterpret_cast<const half4*>(scratch_at(const_cast<_Float16*>(step), wave_j + column, 8 * q + 4 * high, 0));
                const half4 old_lo = *reinterpret_cast<const half4*>(scratch_at(const_cast<_Float16*>(step), wave_j + column, 8 * q + 4 * high, 1));
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    v[4 * q + k] = sum[4 * q + k] * UNSCALE + group.a * (static_cast<float>(old_hi[k]) + static_cast<float>(old_lo[k]));
            }
            if (m.final) {
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] *= UNSCALE;
                write_final<T>(m, v, wave_i, tile * SMALL + wave_j, scratch);
                __syncthreads();
                continue;
            }
            split_piece(v, hi, lo);
            write_quads(scratch, column, hi, lo);
            write_scratch(scratch, m.x_t, tile * SMALL + wave_j, wave_i, PITCH);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = wave_i + e / 4 * 8 + 4 * high + e % 4;
                *scratch_at(rows + wave_j / 32 * NARROW_STEP, row, column, 0) = hi[e / 4][e % 4];
                *scratch_at(rows + wave_j / 32 * NARROW_STEP, row, column, 1) = lo[e / 4][e % 4];
            }
        }
        __syncthreads();
        multiply_tile(rows, rows, wave_i, wave_j, gram, gram_cross);
        __syncthreads();
    }
    if (m.final) return;
    float flat[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) flat[e] = gram[e] + gram_cross[e];
    if (m.splits > 1 && !join_parts(m, 0, part, flat)) return;
    // G, symmetric, and the next B.
#pragma unroll
    for (int e = 0; e < 16; ++e) flat[e] *= UNSCALE;
    split_piece(flat, hi, lo);
    // B is formed from one G, as it is held: near G = 1 the errors of b G and c G G cancel but for a fiftieth.
#pragma unroll
    for (int e = 0; e < 16; ++e) flat[e] = static_cast<float>(hi[e / 4][e % 4]) + static_cast<float>(lo[e / 4][e % 4]);
    write_quads(rows + wave_i / 32 * NARROW_STEP, wave_j + column, hi, lo);
    __syncthreads();
    float16v square = {}, square_cross = {};
    multiply_tile(rows, rows, wave_i, wave_j, square, square_cross);
    square += square_cross;
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = group.c * square[e] * UNSCALE + group.b * flat[e];
    split_piece(v, hi, lo);
    write_quads(scratch, column, hi, lo);
    write_scratch(scratch, m.b, wave_j, wave_i, PITCH);
}

// ---- matrices of a few rows -------------------------------------------------------------------
// A step takes X to M X and G to M G M with M = a + b G + c G G, so that the result is T X of a T that follows from the
// first G alone. With at most 8 rows these small matrices cost nothing in 64 bits, the result is rounded once, and two launches
// serve for all steps: the first adds up G (its trace is the norm's square), the second forms T, once a workgroup, and T X. In split
// float16 the few errors of such a matrix do not average out: 512 x 2 was off by 8.5e-7 of it, twice the float32 steps'
// 4.2e-7. Taken for more rows it would need sums beyond the registers.
constexpr int THIN = 8;
constexpr int THIN_SUMS = THIN * (THIN + 1) / 2;  // of G, on and below the diagonal
constexpr int THIN_SPLITS = 64;                   // workgroups that share a matrix's sums
constexpr int THIN_COLUMNS = 4 * THREADS;         // columns of T X of a workgroup, and the fewest of the sums

struct Thin {
    const void* in;
    void* out;
    std::int64_t in_row, in_col, out_row, out_col;  // steps along the longer side's columns and the shorter one's rows
    float* x;      // the values, rows of `cols`: out may lie across the matrix
    double* sums;  // THIN_SUMS a workgroup of the first launch
    int rows, cols, splits, each;
};

struct ThinGroup {
    Thin m[GROUP];
    int first_block[GROUP + 1];
    int steps;
    float a, b, c, eps;
};
static_assert(sizeof(ThinGroup) <= 4096, "descriptors must fit the kernel arguments");

template <typename T>
__global__ __launch_bounds__(THREADS) void thin_sums_kernel(ThinGroup group) {
    __shared__ double parts[THREADS / 64][THIN_SUMS];
    const int item = item_of(group, blockIdx.x), part = blockIdx.x - group.first_block[item];
    const Thin& m = group.m[item];
    const T* in = static_cast<const T*>(m.in);
    double sums[THIN_SUMS] = {};
    const int end = min((part + 1) * m.each, m.cols);
    for (int column = part * m.each + threadIdx.x; column < end; column += THREADS) {
        float v[THIN];
#pragma unroll
        for (int i = 0; i < THIN; ++i) v[i] = i < m.rows ? static_cast<float>(in[i * m.in_row + column * m.in_col]) : 0.0f;
#pragma unroll
        for (int i = 0; i < THIN; ++i) {
            if (i >= m.rows) break;
            m.x[static_cast<std::int64_t>(i) * m.cols + column] = v[i];
#pragma unroll
            for (int k = 0; k <= i; ++k) sums[i * (i + 1) / 2 + k] += static_cast<double>(v[i]) * static_cast<double>(v[k]);
        }
    }
#pragma unroll
    for (int i = 0; i < THIN_SUMS; ++i) {
        if (i >= m.rows * (m.rows + 1) / 2) break;
        const double total = wave_total(sums[i]);
        if ((threadIdx.x & 63) == 0) parts[threadIdx.x / 64][i] = total;
    }
    __syncthreads();
    if (threadIdx.x < m.rows * (m.rows + 1) / 2)
        m.sums[part * THIN_SUMS + threadIdx.x] =
            (parts[0][threadIdx.x] + parts[1][threadIdx.x]) + (parts[2][threadIdx.x] + parts[3][threadIdx.x]);
}

using ThinMatrix = double[THIN][THIN];

// The lane's element of a product; lane 8 i + j has element (i, j).
__device__ __forceinline__ double thin_product(const ThinMatrix& a, const ThinMatrix& b) {
    const int i = (threadIdx.x & 63) / THIN, j = threadIdx.x % THIN;
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < THIN; ++k) sum += a[i][k] * b[k][j];
    return sum;
}
__device__ __forceinline__ void set_thin(ThinMatrix& to, double v) {
    wave_order();
    to[(threadIdx.x & 63) / THIN][threadIdx.x % THIN] = v;
    wave_order();
}

template <typename T>
__global__ __launch_bounds__(THREADS) void thin_apply_kernel(ThinGroup group) {
    static_assert(THIN * THIN == 64, "a wave has a small matrix");
    __shared__ ThinMatrix gram, factor, applied, held;
    const int item = item_of(group, blockIdx.x), part = blockIdx.x - group.first_block[item];
    const Thin& m = group.m[item];
    if (threadIdx.x < 64) {
        const int i = threadIdx.x / THIN, j = threadIdx.x % THIN, high = max(i, j), at = high * (high + 1) / 2 + min(i, j);
        const bool there = high < m.rows;
        double g = 0.0;
        if (there)
            for (int split = 0; split < m.splits; ++split) g += m.sums[split * THIN_SUMS + at];
        const double squares = wave_total(i == j ? g : 0.0);
        const double scale = 1.0 / (sqrt(squares) + static_cast<double>(group.eps));
        const double unit = there && i == j ? 1.0 : 0.0;
        set_thin(gram, there ? g * scale * scale : 0.0);
        set_thin(applied, unit);
        for (int step = 0; step < group.steps; ++step) {
            const double own = gram[i][j];
            set_thin(factor, group.a * unit + group.b * own + group.c * thin_product(gram, gram));
            const double next = thin_product(factor, applied);
            set_thin(held, thin_product(factor, gram));
            set_thin(applied, next);
            set_thin(gram, thin_product(held, factor));
        }
        set_thin(applied, applied[i][j] * scale);
    }
    __syncthreads();
    T* out = static_cast<T*>(m.out);
    const int end = min((part + 1) * THIN_COLUMNS, m.cols);
    for (int column = part * THIN_COLUMNS + threadIdx.x; column < end; column += THREADS) {
        double v[THIN];
#pragma unroll
        for (int k = 0; k < THIN; ++k) v[k] = k < m.rows ? m.x[static_cast<std::int64_t>(k) * m.cols + column] : 0.0f;
        for (int i = 0; i < m.rows; ++i) {
            double sum = 0.0;
#pragma unroll
            for (int k = 0; k < THIN; ++k)
                if (k < m.rows) sum += applied[i][k] * v[k];
            out[i * m.out_row + column * m.out_col] = static_cast<T>(static_cast<float>(sum));
        }
    }
}

bool is_thin(const OrthogonalMatrix& m) { return std::min(m.rows, m.cols) <= THIN; }

std::int64_t aligned(std::int64_t bytes) { return (bytes + 255) / 256 * 256; }

std::int64_t thin_bytes(const OrthogonalMatrix& m) {
    return aligned(static_cast<std::int64_t>(m.rows) * m.cols * 4) + aligned(THIN_SPLITS * THIN_SUMS * 8);
}

template <typename T>
int run_thin(const OrthogonalMatrix* matrices, int count, const OrthogonalSteps& o, char* workspace, hipStream_t stream) {
    ThinGroup group{};
    group.steps = o.steps, group.a = o.a, group.b = o.b, group.c = o.c, group.eps = o.eps;
    for (int i = 0; i < count; ++i) {
        const OrthogonalMatrix& from = matrices[i];
        const bool tall = from.rows > from.cols;
        Thin& m = group.m[i];
        m.in = from.in, m.out = from.out;
        m.in_row = tall ? 1 : from.in_stride, m.in_col = tall ? from.in_stride : 1;
        m.out_row = tall ? 1 : from.out_stride, m.out_col = tall ? from.out_stride : 1;
        m.rows = std::min(from.rows, from.cols), m.cols = std::max(from.rows, from.cols);
        m.x = reinterpret_cast<float*>(workspace);
        m.sums = reinterpret_cast<double*>(workspace + aligned(static_cast<std::int64_t>(m.rows) * m.cols * 4));
        workspace += thin_bytes(from);
        m.each = std::max((m.cols + THIN_SPLITS - 1) / THIN_SPLITS, THIN_COLUMNS);
        m.splits = (m.cols + m.each - 1) / m.each;
        group.first_block[i + 1] = group.first_block[i] + m.splits;
    }
    launch(thin_sums_kernel<T>, dim3(group.first_block[count]), dim3(THREADS), 0, stream, group);
    MFH_TRY(MFH_CHECK_LAUNCH("orthogonal thin sums", stream));
    for (int i = 0; i < count; ++i)
        group.first_block[i + 1] = group.first_block[i] + (group.m[i].cols + THIN_COLUMNS - 1) / THIN_COLUMNS;
    launch(thin_apply_kernel<T>, dim3(group.first_block[count]), dim3(THREADS), 0, stream, group);
    return MFH_CHECK_LAUNCH("orthogonal thin result", stream);
}

// ---- the plan of one matrix -------------------------------------------------------------------
// The padding allows large tiles from here on.
int padding_of(int shorter) { return shorter >= 256 ? LARGE : SMALL; }

int tiles_of(int shorter, int longer, bool symmetric, int side) {
    const int m = (shorter + side - 1) / side;
    return symmetric ? m * (m + 1) / 2 : m * ((longer + side - 1) / side);
}

struct Plan {
    int s, l;                    // sides as they lie in memory
    int shorter, longer;         // and as they are
    std::int64_t x, square;      // bytes of X and of a square matrix
    int square_blocks;
    explicit Plan(const OrthogonalMatrix& m) : shorter(std::min(m.rows, m.cols)), longer(std::max(m.rows, m.cols)) {
        const int padding = padding_of(shorter);
        s = (shorter + padding - 1) / padding * padding, l = (longer + padding - 1) / padding * padding;
        x = static_cast<std::int64_t>(s) * l * 4, square = static_cast<std::int64_t>(s) * s * 4;
        const std::int64_t blocks = (static_cast<std::int64_t>(m.rows) * m.cols + SQUARES_EACH - 1) / SQUARES_EACH;
        square_blocks = static_cast<int>(std::min<std::int64_t>(blocks, SQUARES_BLOCKS));
    }
    std::int64_t bytes() const { return 3 * x + 2 * square + SQUARES_BLOCKS * 8; }
};

struct Buffers {
    _Float16 *x, *x_t[2], *g, *p;
    double* squares;
    Buffers(const Plan& plan, char* at) {
        const auto take = [&](std::int64_t bytes) {
            char* here = at;
            at += bytes;
            return reinterpret_cast<_Float16*>(here);
        };
        x = take(plan.x), x_t[0] = take(plan.x), x_t[1] = take(plan.x), g = take(plan.square), p = take(plan.square);
        squares = reinterpret_cast<double*>(at);
    }
};

constexpr int NARROW_SPLITS = 16;  // workgroups of a narrow matrix: the last one reads all their parts
constexpr std::int64_t NARROW_PARTS_BYTES = NARROW_SPLITS * SMALL * SMALL * 4;

bool is_narrow(const Plan& plan) { return plan.shorter <= SMALL; }

template <typename T>
int run_narrow(const OrthogonalMatrix* matrices, int count, const OrthogonalSteps& o, const std::vector<Plan>& plans,
               const std::vector<Buffers>& buffers, char* parts, hipStream_t stream) {
    static_assert(GROUP <= LOGIT_COUNTERS, "a counter a matrix");
    for (int step = 0; step <= o.steps; ++step) {  // the first G and B, then the steps
        NarrowGroup group{};
        group.a = o.a, group.b = o.b, group.c = o.c;
        for (int i = 0; i < count; ++i) {
            Narrow& m = group.m[i];
            const Plan& plan = plans[i];
            m.x = step == 0 ? buffers[i].x : nullptr, m.x_t = buffers[i].x_t[0], m.b = buffers[i].p, m.x_pitch = plan.l * 2;
            m.parts = reinterpret_cast<float*>(parts + static_cast<std::int64_t>(i) * NARROW_PARTS_BYTES);
            m.arrived = o.counters + i;
            if (step == o.steps) m.final = matrices[i].out, m.final_stride = matrices[i].out_stride;
            m.rows = plan.shorter, m.cols = plan.longer, m.tall = matrices[i].rows > matrices[i].cols;
            m.tiles = (plan.longer + SMALL - 1) / SMALL;
            m.each = (m.tiles + NARROW_SPLITS - 1) / NARROW_SPLITS, m.splits = (m.tiles + m.each - 1) / m.each;
            group.first_block[i + 1] = group.first_block[i] + m.splits;
        }
        launch(narrow_kernel<T>, dim3(group.first_block[count]), dim3(THREADS), 0, stream, group);
        MFH_TRY(MFH_CHECK_LAUNCH("orthogonal narrow step", stream));
    }
    return OK;
}

template <typename T>
int run_group(const OrthogonalMatrix* matrices, int count, const OrthogonalSteps& o, char* workspace, hipStream_t stream) {
    std::vector<Plan> plans;
    std::vector<Buffers> buffers;
    for (int i = 0; i < count; ++i) {
        plans.emplace_back(matrices[i]);
        buffers.emplace_back(plans[i], workspace);
        workspace += plans[i].bytes();
    }
    char* const parts = workspace;
    SourceGroup sources{};
    sources.eps = o.eps;
    for (int i = 0; i < count; ++i) {
        const OrthogonalMatrix& m = matrices[i];
        const bool tall = m.rows > m.cols;
        Source& s = sources.s[i];
        s.in = m.in, s.stride = m.in_stride, s.rows = m.rows, s.cols = m.cols, s.columns = FastDiv(m.cols);
        s.same = tall ? buffers[i].x_t[0] : buffers[i].x, s.across = tall ? buffers[i].x : buffers[i].x_t[0];
        s.padded_rows = tall ? plans[i].l : plans[i].s, s.padded_cols = tall ? plans[i].s : plans[i].l;
        s.squares = buffers[i].squares;
        sources.square_blocks[i] = plans[i].square_blocks;
        sources.first_block[i + 1] = sources.first_block[i] + plans[i].square_blocks;
    }
    launch(squares_kernel<T>, dim3(sources.first_block[count]), dim3(THREADS), 0, stream, sources);
    MFH_TRY(MFH_CHECK_LAUNCH("orthogonal squares", stream));
    for (int i = 0; i < count; ++i)
        sources.first_block[i + 1] = sources.first_block[i] + sources.s[i].padded_rows / 64 * (sources.s[i].padded_cols / 64);
    launch(split_kernel<T>, dim3(sources.first_block[count]), dim3(THREADS), 0, stream, sources);
    MFH_TRY(MFH_CHECK_LAUNCH("orthogonal split", stream));
    if (std::all_of(plans.begin(), plans.end(), is_narrow))
        return run_narrow<T>(matrices, count, o, plans, buffers, parts, stream);
    const int cus = device_cu_count();
    const auto products = [&](auto&& describe) {
        ProductGroup group{};
        // Large tiles need half the loads of small ones a product, where there are enough of them.
        int large_tiles = 0, tiles[GROUP], units[GROUP];
        for (int i = 0; i < count; ++i) {
            Product& p = group.p[i];
            const OrthogonalMatrix& m = matrices[i];
            p.alpha = 1.0f, p.tall = m.rows > m.cols;
            p.rows = std::min(m.rows, m.cols), p.cols = std::max(m.rows, m.cols);
            describe(i, p);
            if (padding_of(plans[i].shorter) == LARGE) large_tiles += tiles_of(plans[i].shorter, plans[i].longer, p.symmetric, LARGE);
        }
        // Whole calls with large and with small ones, us, by their number on 256 CUs. Symmetric products: 66 of 1408 x 1408
        // 472 and 420, 80 of eight 512 x 2048 555 and 467, 100 of ten 692 and 600, 108 of three 1000 x 3000 851 and 848,
        // 136 of 2048 x 2048 856 and 891, 210 of 2560 x 2560 1463 and 1673. Others: 196 of 896 x 3584 425 and 408, 256 of 1024 x 4096
        // 503 and 477, 256 of 2048 x 2048 833 and 856, 320 of five 512 x 2048 381 and 384, 324 of 1152 x 4608 611 and 666,
        // 448 of seven 512 x 2048 524 and 569, 484 of 1408 x 5632 857 and 999, 576 of 3000 x 3000 2064 and 2244.
        const bool use_large = large_tiles >= (group.p[0].symmetric ? cus / 2 : cus + cus / 4);
        bool all_small = true;
        std::int64_t steps = 0;
        for (int i = 0; i < count; ++i) {
            Product& p = group.p[i];
            const Plan& plan = plans[i];
            p.small = !use_large || padding_of(plan.shorter) == SMALL, all_small = all_small && p.small;
            const int side = p.small ? SMALL : LARGE;
            p.k_padded = p.over_longer ? plan.l : plan.s;
            p.ksteps = ((p.over_longer ? plan.longer : plan.shorter) + K_STEP - 1) / K_STEP;
            p.m_padded = plan.s, p.n_padded = p.symmetric ? plan.s : plan.l;
            p.m_tiles = (plan.shorter + side - 1) / side;
            p.n_tiles = p.symmetric ? p.m_tiles : (plan.longer + side - 1) / side;
            tiles[i] = tiles_of(plan.shorter, plan.longer, p.symmetric, side);
            steps += static_cast<std::int64_t>(tiles[i]) * p.ksteps;
        }
        const int slots = cus * (all_small ? 4 : 2);
        // Tiles whose steps are shared by several workgroups: all of them where they would leave CUs idle, as many parts as
        // fill the GPU but no more than half the root of the steps, since the last workgroup reads all parts' sums (1999 x 517
        // and 771 x 1003 float16, G: 18 us, 24 with up to 1.2 times the root); else those that a last, short round would
        // hold (4096 x 4096, 528 tiles for 512 places: 222 us, 292 with whole tiles).
        const int all = std::accumulate(tiles, tiles + count, 0);
        int rest = all >= slots ? all % slots : all;
        const std::int64_t share = all >= slots ? 1 : std::max<std::int64_t>(steps / slots, 4);
        if (all >= slots && 2 * rest > slots) rest = 0;
        char* part = parts;
        int split_tiles = 0;
        for (int i = count - 1; i >= 0; --i) {
            Product& p = group.p[i];
            const std::int64_t bytes = p.small ? SMALL * SMALL * 4 : LARGE * LARGE * 4;
            const int here = std::min(rest, tiles[i]), most = static_cast<int>(std::sqrt(p.ksteps * 0.25));
            rest -= here;
            std::int64_t splits = std::min<std::int64_t>(all >= slots ? p.ksteps / 4 : p.ksteps / share, most);
            if (all >= slots) splits = std::min<std::int64_t>(splits, slots / std::max(1, all % slots));
            if (split_tiles + here > LOGIT_COUNTERS || part + bytes * splits * here > parts + PARTS_BYTES) splits = 1;
            p.splits = static_cast<int>(std::max<std::int64_t>(splits, 1));
            p.whole = p.splits > 1 ? tiles[i] - here : tiles[i];
            if (p.splits > 1) {
                p.parts = reinterpret_cast<float*>(part), p.arrived = o.counters + split_tiles;
                part += bytes * p.splits * here, split_tiles += here;
            }
            units[i] = p.whole + (tiles[i] - p.whole) * p.splits;
        }
        for (int i = 0; i < count; ++i) group.first_unit[i + 1] = group.first_unit[i] + units[i];
        group.round = all >= slots ? all / slots * slots : group.first_unit[count];
        launch(all_small ? product_kernel<SMALL, T> : product_kernel<LARGE, T>, dim3(group.first_unit[count]), dim3(THREADS), 0,
               stream, group);
        return MFH_CHECK_LAUNCH("orthogonal product", stream);
    };
    for (int step = 0; step < o.steps; ++step) {
        const int from = step & 1;
        MFH_TRY(products([&](int i, Product& p) {
            const Buffers& at = buffers[i];
            p.symmetric = true, p.a = p.b = at.x, p.out = p.out_t = at.g, p.over_longer = true;
        }));
        MFH_TRY(products([&](int i, Product& p) {
            const Buffers& at = buffers[i];
            p.symmetric = true, p.a = p.b = p.add_t = at.g, p.out = p.out_t = at.p;
            p.alpha = o.c, p.beta = o.b;
        }));
        MFH_TRY(products([&](int i, Product& p) {
            const Buffers& at = buffers[i];
            p.a = at.p, p.b = p.add_t = at.x_t[from], p.beta = o.a;
            if (step + 1 == o.steps) p.final = matrices[i].out, p.final_stride = matrices[i].out_stride;
            else p.out = at.x, p.out_t = at.x_t[from ^ 1];
        }));
    }
    return OK;
}

std::int64_t group_bytes(const OrthogonalMatrix* matrices, int count) {
    std::int64_t bytes = 0;
    bool narrow = true;
    for (int i = 0; i < count; ++i) {
        const Plan plan(matrices[i]);
        bytes += plan.bytes(), narrow = narrow && is_narrow(plan);
    }
    return bytes + (narrow ? count * NARROW_PARTS_BYTES : PARTS_BYTES);
}

// Groups of a list, the thin matrices apart: thin(first, count) and others(first, count) until one fails.
template <typename Few, typename Others>
int each_group(const OrthogonalMatrix* matrices, int count, Few&& thin, Others&& others) {
    std::vector<OrthogonalMatrix> held(matrices, matrices + count);
    const int first = static_cast<int>(std::stable_partition(held.begin(), held.end(), is_thin) - held.begin());
    for (int i = 0; i < first; i += GROUP) MFH_TRY(thin(held.data() + i, std::min(GROUP, first - i)));
    for (int i = first; i < count; i += GROUP) MFH_TRY(others(held.data() + i, std::min(GROUP, count - i)));
    return OK;
}

std::int64_t list_bytes(const OrthogonalMatrix* matrices, int count) {
    std::int64_t most = 0;
    const auto thin = [&](const OrthogonalMatrix* group, int here) {
        std::int64_t bytes = 0;
        for (int i = 0; i < here; ++i) bytes += thin_bytes(group[i]);
        most = std::max(most, bytes);
        return static_cast<int>(OK);
    };
    each_group(matrices, count, thin, [&](const OrthogonalMatrix* group, int here) {
        most = std::max(most, group_bytes(group, here));
        return static_cast<int>(OK);
    });
    return most;
}

template <typename T>
int run_list(const OrthogonalMatrix* matrices, int count, const OrthogonalSteps& o, char* workspace, hipStream_t stream) {
    return each_group(
        matrices, count, [&](const OrthogonalMatrix* group, int here) { return run_thin<T>(group, here, o, workspace, stream); },
        [&](const OrthogonalMatrix* group, int here) { return run_group<T>(group, here, o, workspace, stream); });
}

// ---- the optimiser's step around it -----------------------------------------------------------
struct MomentumGroup {
    MuonTensor t[GROUP];
    float* direction[GROUP];
    unsigned first_block[GROUP + 1];
    float momentum, grad_scale;
    int nesterov;
};
static_assert(sizeof(MomentumGroup) <= 4096, "descriptors must fit the kernel arguments");

constexpr int ELEMENTWISE = 4;  // elements of a thread

template <typename F>
__device__ __forceinline__ void each_element(const MomentumGroup& group, F&& f) {
    const int item = item_of(group, blockIdx.x);
    const MuonTensor& t = group.t[item];
    const std::int64_t size = static_cast<std::int64_t>(t.rows) * t.cols;
    const std::int64_t first = static_cast<std::int64_t>(blockIdx.x - group.first_block[item]) * THREADS * ELEMENTWISE + threadIdx.x;
#pragma unroll
    for (int k = 0; k < ELEMENTWISE; ++k)
        if (first + k * THREADS < size) f(t, group.direction[item], first + k * THREADS);
}

// m = momentum m + g; the direction is g + momentum m (Nesterov's), or m.
__global__ __launch_bounds__(THREADS) void momentum_kernel(MomentumGroup group) {
    each_element(group, [&](const MuonTensor& t, float* direction, std::int64_t at) {
        const float g = t.grad[at] * group.grad_scale, m = group.momentum * t.momentum[at] + g;
        t.momentum[at] = m;
        direction[at] = group.nesterov ? g + group.momentum * m : m;
    });
}

// p = keep p - rate direction, of the direction made orthogonal.
__global__ __launch_bounds__(THREADS) void descend_kernel(MomentumGroup group) {
    each_element(group, [&](const MuonTensor& t, const float* direction, std::int64_t at) {
        t.param[at] = t.keep * t.param[at] - t.rate * direction[at];
    });
}

OrthogonalMatrix direction_of(const MuonTensor& t, float* direction) {
    return {direction, direction, t.cols, t.cols, t.rows, t.cols};
}

std::int64_t direction_bytes(const MuonTensor& t) { return aligned(static_cast<std::int64_t>(t.rows) * t.cols * 4); }

int run_muon_group(const MuonTensor* tensors, int count, const MuonSteps& o, char* workspace, hipStream_t stream) {
    MomentumGroup group{};
    group.momentum = o.momentum, group.grad_scale = o.grad_scale, group.nesterov = o.nesterov;
    std::vector<OrthogonalMatrix> directions;
    for (int i = 0; i < count; ++i) {
        group.t[i] = tensors[i];
        group.direction[i] = reinterpret_cast<float*>(workspace);
        workspace += direction_bytes(tensors[i]);
        directions.push_back(direction_of(tensors[i], group.direction[i]));
        group.first_block[i + 1] =
            group.first_block[i] + blocks_for(static_cast<std::int64_t>(tensors[i].rows) * tensors[i].cols, THREADS * ELEMENTWISE);
    }
    launch(momentum_kernel, dim3(group.first_block[count]), dim3(THREADS), 0, stream, group);
    MFH_TRY(MFH_CHECK_LAUNCH("muon momentum", stream));
    MFH_TRY(run_list<float>(directions.data(), count, o.orthogonal, workspace, stream));
    launch(descend_kernel, dim3(group.first_block[count]), dim3(THREADS), 0, stream, group);
    return MFH_CHECK_LAUNCH("muon step", stream);
}

}  // namespace

std::int64_t muon_workspace(const MuonTensor* tensors, int count) {
    std::int64_t most = 0;
    for (int i = 0; i < count; i += GROUP) {
        const int here = std::min(count - i, GROUP);
        std::vector<OrthogonalMatrix> directions;
        std::int64_t bytes = 0;
        for (int k = 0; k < here; ++k) {
            directions.push_back(direction_of(tensors[i + k], nullptr));
            bytes += direction_bytes(tensors[i + k]);
        }
        most = std::max(most, bytes + list_bytes(directions.data(), here));
    }
    return most;
}

int launch_muon(const MuonTensor* tensors, int count, const MuonSteps& o, void* workspace, hipStream_t stream) {
    for (int i = 0; i < count; i += GROUP)
        MFH_TRY(run_muon_group(tensors + i, std::min(GROUP, count - i), o, static_cast<char*>(workspace), stream));
    return OK;
}

std::int64_t orthogonal_workspace(const OrthogonalMatrix* matrices, int count) { return list_bytes(matrices, count); }

int launch_orthogonal(const OrthogonalMatrix* matrices, int count, int type, const OrthogonalSteps& o, void* workspace,
                      hipStream_t stream) {
    return with_type(type, [&](auto element) { return run_list<decltype(element)>(matrices, count, o, static_cast<char*>(workspace), stream); });
}

}  // namespace mfh
