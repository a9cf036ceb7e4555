// Rows of bfloat16 times a matrix kept in 4 bits, with a scale and a zero point per group of its columns:
//
//     out[m, n] = sum over groups g of  s[n, g] ( sum_{k in g} x[m, k] c[n, k]  -  z[n, g] sum_{k in g} x[m, k] )
//
// The matrix is read as it is stored, a row after the other, two codes a byte.  A wavefront takes NT tiles of 16 matrix rows
// and walks K in pieces of 128: a lane loads 16 bytes, 32 codes of one row, and four lane swaps turn the 4 x 4 words that
// the four lanes of a row hold, so that step s of the piece has columns 32 s + 8 j .. +7 in lane group j: the operand order of
// the matrix cores' 16 x 16 x 32 product, with x loaded in the same order.
//
// A code c becomes a bfloat16 by three bits of arithmetic: a number from 2^-8 on has a step of 2^-15 in its last place, so 0x3B80 | c << 3
// is (16 + c) / 4096, exactly, and two codes that lie 16 bits apart in a word turn in one instruction pair (mask and or after a shift).
// What that adds, s (16 + z) / 4096 sum x, goes out again: the sums of x are made of the same operands against numbers of 1/128, and their
// products with s (16 + z) / 32 are a product in float32 over the groups, four of them in an instruction of the matrix cores, whose operand
// order is the order in which the lanes hold what they have loaded of s and z.  All sums are float32; taking off what was added
// costs the result some three of its 24 bits.  A result is multiplied by 4096 when it is stored: so much smaller no sum over 128 columns
// leaves float32's range, however large x is (with 16 + c itself x of 3e35 did), and results from 2^-114 on keep all their bits.  Two codes
// that neighbour in a word are four columns apart, so x's words are permuted alike.
//
// The wavefronts of a workgroup share the K pieces in turn and meet in LDS, in order.  A piece's codes (and x, where the
// registers hold it twice) are asked for while the piece before is worked on; a lane group of four loads the scales and zero points
// of the next four groups it meets, a group each, and three lane swaps hand all four to everybody.  Rows of x beyond M
// repeat the last one (a row of the product depends on its own row of x alone) and are not stored; columns beyond K are zeros
// of x.
#include "api.h"
#include "common.h"
#include "matrix_async.h"

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 i4_bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float i4_floatx4;

union I4Frag {
    i4_bf16x8 v;
    uint4 u;
    uint32_t w[4];
};

#define I4_PIECE 128             // columns a wavefront takes at a time: 16 bytes of codes a lane

struct I4Args {
    void* out;
    const bf16_t* x;
    const uint8_t* codes;
    const void* scales;
    const uint8_t* zeros;        // NULL: every zero point is 8
    int rows, n, k, groups, per; // per: pieces of 128 columns that share a group (groups of 128 and more)
    int out_f32;
};

// What a matrix without zero points reads in their place.
static __device__ uint8_t i4_zero_point[4] = {8, 8, 8, 8};

// Sixteen bytes from an address that is a multiple of four.  ONCE: marked as read once, for loads that take whole lines (a half line
// marked so is fetched again for the other half).
template <bool ONCE>
__device__ __forceinline__ uint4 load16_by4(const uint8_t* p) {
    typedef unsigned int u32x4_t __attribute__((ext_vector_type(4), aligned(4)));
    const u32x4_t* at = reinterpret_cast<const u32x4_t*>(p);
    const u32x4_t v = ONCE ? __builtin_nontemporal_load(at) : *at;
    return make_uint4(v.x, v.y, v.z, v.w);
}

// The words that the four lanes of a row hold, 8 columns each, brought to where a step's 32 columns are those of few groups.
// STEPS 1: word s of lane group j has columns 32 s + 8 j .. +7; 2: those of 64 (s / 2) ..+63 in steps 2 (s / 2) and + 1; 4: as loaded.
// column_of: the first of the eight.
template <int STEPS>
__device__ __forceinline__ int column_of(int s, int j) {
    return STEPS == 1 ? 32 * s + 8 * j : STEPS == 2 ? 64 * (s >> 1) + 32 * (j & 1) + 16 * (j >> 1) + 8 * (s & 1) : 32 * j + 8 * s;
}
template <int STEPS>
__device__ __forceinline__ void turn_words(uint32_t (&w)[4]) {
    typedef unsigned __attribute__((ext_vector_type(2))) pair_t;
    if (STEPS == 4) return;
    const pair_t a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const pair_t b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    if (STEPS == 2) {
        w[0] = a.x;
        w[1] = b.x;
        w[2] = a.y;
        w[3] = b.y;
        return;
    }
    const pair_t c = __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false);
    const pair_t d = __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false);
    w[0] = c.x;
    w[1] = c.y;
    w[2] = d.x;
    w[3] = d.y;
}

// What a code is smaller by, and its parts: the sums' of x and the zero points'.
#define I4_BACK 4096.f
#define I4_SIXTEEN 0x3B803B80u   // two times 16 / 4096
#define I4_ONES 0x3C003C00u      // two times 1 / 128
__device__ __forceinline__ float taken_off(float scale, uint8_t zero) { return -scale * fmaf((float)zero, 1.f / 32.f, 16.f / 32.f); }

// Eight codes as (16 + c) / 4096, in the order 0 4 1 5 2 6 3 7 of the word's nibbles.  mask is 0x00780078 and sixteen I4_SIXTEEN, held in
// registers that the compiler does not see through: an instruction takes one literal, and with two the and and the or would be
// one each.
__device__ __forceinline__ void widen(I4Frag& f, uint32_t w, uint32_t mask, uint32_t sixteen) {
    f.w[0] = ((w << 3) & mask) | sixteen;
    f.w[1] = ((w >> 1) & mask) | sixteen;
    f.w[2] = ((w >> 5) & mask) | sixteen;
    f.w[3] = ((w >> 9) & mask) | sixteen;
}
// Eight neighbouring numbers in the same order.
__device__ __forceinline__ void reorder(I4Frag& f, const uint4 u) {
    f.w[0] = __builtin_amdgcn_perm(u.z, u.x, 0x05040100u);
    f.w[1] = __builtin_amdgcn_perm(u.z, u.x, 0x07060302u);
    f.w[2] = __builtin_amdgcn_perm(u.w, u.y, 0x05040100u);
    f.w[3] = __builtin_amdgcn_perm(u.w, u.y, 0x07060302u);
}

// acc += a . b of the matrix cores' 16 x 16 x 4 product in float32: lane l holds a[l % 16][l / 16] and b[l / 16][l % 16].
__device__ __forceinline__ void add_product4(i4_floatx4& acc, float a, float b) { acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, acc, 0, 0, 0); }

// 1 / 128 of the sum over the 32 STEPS columns of x's fragments from xf on, of row l % 16 in lane l.
template <int STEPS>
__device__ __forceinline__ float sum_of(const I4Frag* xf, const I4Frag& ones) {
    i4_floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones.v, xf[i].v, s, 0, 0, 0);
    return s[0];
}

// A lane group's value in every one of the four.
__device__ __forceinline__ void to_all(float (&all)[4], float v) {
    typedef unsigned __attribute__((ext_vector_type(2))) pair_t;
    const unsigned u = __float_as_uint(v);
    const pair_t a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const pair_t low = __builtin_amdgcn_permlane16_swap(a.x, a.x, false, false), high = __builtin_amdgcn_permlane16_swap(a.y, a.y, false, false);
    const unsigned r0 = low.x, r1 = low.y, r2 = high.x, r3 = high.y;
    all[0] = __uint_as_float(r0);
    all[1] = __uint_as_float(r1);
    all[2] = __uint_as_float(r2);
    all[3] = __uint_as_float(r3);
}

// MT tiles of 16 rows of x, NT tiles of 16 rows of the matrix, W wavefronts.  STEPS: steps of 32 columns that share a group
// (4: groups are multiples of 128).
template <int MT, int NT, int W, int STEPS, typename S>
__global__ __launch_bounds__(W * RI_WAVE) void gemm_int4_kernel(const I4Args a) {
    constexpr int USES = 4 / STEPS, ROUND = STEPS;            // groups that a piece meets; pieces that meet four groups
    constexpr int TURN = ROUND < 2 ? 2 : ROUND;               // pieces a turn of the loop: an even number, two buffers
    constexpr bool X_TWICE = MT == 1;
    const int lane = threadIdx.x & (RI_WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / RI_WAVE), i = lane & 15, j = lane >> 4;
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
    const int full = a.k / I4_PIECE, pieces = (a.k + I4_PIECE - 1) / I4_PIECE;
    const size_t row_bytes = (size_t)a.k / 2;
    const S* scales = (const S*)a.scales;
    const uint8_t* zeros = a.zeros ? a.zeros : i4_zero_point;
    const int zero_step = a.zeros ? 1 : 0;
    const uint8_t* code_row[NT];
    size_t group_row[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const size_t col = min(n0 + 16 * t + i, a.n - 1);
        code_row[t] = a.codes + col * row_bytes + 16 * j;
        group_row[t] = col * a.groups;
    }
    const bf16_t* x_row[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x_row[t] = a.x + (size_t)min(m0 + 16 * t + i, a.rows - 1) * a.k + 8 * j;

    i4_floatx4 total[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int t = 0; t < NT; ++t) total[mt][t] = i4_floatx4{0.f, 0.f, 0.f, 0.f};
    uint32_t mask = 0x00780078u, sixteen = I4_SIXTEEN;
    ma_opaque(mask);
    ma_here(sixteen);
    I4Frag ones;
    ones.w[0] = ones.w[1] = ones.w[2] = ones.w[3] = I4_ONES;

    struct Groups { S scale[NT]; uint8_t zero[NT]; };        // as loaded: a conversion would wait for the load
    // Loads stay out of branches, so that the compiler counts them in flight: one that nobody wants reads what every lane reads.
    auto load_codes = [&](uint4 (&c)[NT], int p, bool wanted) {
#pragma unroll
        for (int t = 0; t < NT; ++t) c[t] = load16_by4<false>(wanted ? code_row[t] + p * (I4_PIECE / 2) : a.codes);
    };
    auto load_x = [&](uint4 (&x)[MT][4], int p, bool wanted) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int s = 0; s < 4; ++s) x[mt][s] = *reinterpret_cast<const uint4*>(wanted ? x_row[mt] + p * I4_PIECE + 32 * s : a.x);
    };
    // The four groups that the wavefront meets from piece p on, group e of them by lane group e.
    auto load_groups = [&](Groups& g, int p) {
        const int piece = min(p + (j / USES) * W, pieces - 1);
        const int group = STEPS == 4 ? (a.per == 1 ? piece : piece / a.per) : min(piece * USES + j % USES, a.groups - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            g.scale[t] = scales[group_row[t] + group];
            g.zero[t] = zeros[(group_row[t] + group) * zero_step];
        }
    };
    float scale[NT][4], less[NT];                            // of four groups: every lane all of them; lane group e of the e-th
    auto spread = [&](const Groups& g) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float own = to_f32(g.scale[t]);
            to_all(scale[t], own);
            less[t] = taken_off(own, g.zero[t]);
        }
    };
    // first: which of the four groups the piece meets first
    auto work = [&](const uint4 (&codes)[NT], const uint4 (&x)[MT][4], int first) {
        I4Frag xf[MT][4];
        float sum[MT];                                        // of the group that lane group j holds, 0 where the piece has none such
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int s = 0; s < 4; ++s) reorder(xf[mt][s], x[mt][s]);
            sum[mt] = 0.f;
#pragma unroll
            for (int e = 0; e < USES; ++e) {
                const float one = sum_of<STEPS>(xf[mt] + e * STEPS, ones);
                sum[mt] = j == first + e ? one : sum[mt];
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            uint32_t w[4] = {codes[t].x, codes[t].y, codes[t].z, codes[t].w};
            turn_words<1>(w);
#pragma unroll
            for (int e = 0; e < USES; ++e) {
                I4Frag wf[STEPS];
#pragma unroll
                for (int s = 0; s < STEPS; ++s) widen(wf[s], w[e * STEPS + s], mask, sixteen);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    i4_floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < STEPS; ++s)
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[mt][e * STEPS + s].v, wf[s].v, acc, 0, 0, 0);
#pragma unroll
                    for (int q = 0; q < 4; ++q) total[mt][t][q] = fmaf(scale[t][first + e], acc[q], total[mt][t][q]);
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) add_product4(total[mt][t], sum[mt], less[t]);
        }
    };

    if (wave < full) {
        uint4 codes[2][NT], x[X_TWICE ? 2 : 1][MT][4];
        Groups g;
        load_groups(g, wave);
        if (X_TWICE) load_x(x[0], wave, true);
        load_codes(codes[0], wave, true);
        for (int p = wave;; p += TURN * W) {
#pragma unroll
            for (int q = 0; q < TURN; ++q) {
                const int at = p + q * W;
                const bool more = at + W < full;
                if (q > 0 && at >= full) break;
                if (q % ROUND == 0) {
                    spread(g);
                    load_groups(g, at + ROUND * W);
                }
                if (X_TWICE) load_x(x[X_TWICE ? (q + 1) % 2 : 0], at + W, more);
                else load_x(x[0], at, true);
                load_codes(codes[(q + 1) % 2], at + W, more);
                work(codes[q % 2], x[X_TWICE ? q % 2 : 0], q % ROUND * USES);
            }
            if (p + TURN * W >= full) break;
        }
    }
    if (pieces > full && full % W == wave) {                  // the row ends within the last piece
        const int k0 = full * I4_PIECE;
        uint4 codes[NT], x[MT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)                       // (a word of eight codes is there whole or not at all)
                w[q] = *reinterpret_cast<const uint32_t*>(code_row[t] - 16 * j + min((size_t)(k0 / 2 + 16 * j + 4 * q), row_bytes - 4));
            codes[t] = make_uint4(w[0], w[1], w[2], w[3]);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int s = 0; s < 4; ++s)
                x[mt][s] = *reinterpret_cast<const uint4*>(k0 + 32 * s + 8 * j < a.k ? x_row[mt] + k0 + 32 * s : ri_zero_fragment + 8 * lane);
        Groups g;
        load_groups(g, full);
        spread(g);
        work(codes, x, 0);
    }

    // the wavefronts' sums, added in their order: lane l holds rows 4 j .. +3 of column i of every tile
    __shared__ float meet[W > 1 ? (W - 1) * MT * NT * 4 * RI_WAVE : 1];
    if (W > 1) {
        if (wave > 0) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        meet[((((wave - 1) * MT + mt) * NT + t) * 4 + e) * RI_WAVE + lane] = total[mt][t][e];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int v = 0; v < W - 1; ++v)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) total[mt][t][e] += meet[(((v * MT + mt) * NT + t) * 4 + e) * RI_WAVE + lane];
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int c = n0 + 16 * t + i;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int m = m0 + 16 * mt + 4 * j + e;
                if (m < a.rows && c < a.n) {
                    const float value = total[mt][t][e] * I4_BACK;
                    if (a.out_f32) ((float*)a.out)[(size_t)m * a.n + c] = value;
                    else ((bf16_t*)a.out)[(size_t)m * a.n + c] = f32_to_bf16(value);
                }
            }
        }
}

// Of two neighbouring lanes: the even one's low in itself and its high in the odd one; the odd one's low in the even one and its high.
__device__ __forceinline__ uint32_t neighbour(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false); }
__device__ __forceinline__ uint32_t from_even(bool odd, uint32_t low, uint32_t high) {
    const uint32_t other = neighbour(high);                   // (all lanes take part)
    return odd ? other : low;
}
__device__ __forceinline__ uint32_t from_odd(bool odd, uint32_t low, uint32_t high) {
    const uint32_t other = neighbour(low);
    return odd ? high : other;
}

// Many matrix rows, up to 16 rows of x: a workgroup's eight wavefronts hold x for the whole of K, PP pieces each in the order of the
// product and summed per group, and go from one tile of 16 matrix rows to the next; of a tile a wavefront reads its PP pieces, so
// that the workgroup reads 16 whole rows, neighbours in memory.  AHEAD tiles' codes are on their way while one is worked on.  The
// wavefronts' sums of eight tiles wait in LDS; then they meet, and each adds up and stores one tile (16 rows x 151,936 x 4,096, groups of
// 64: 74 to 78 us, 5 TB/s, bound by the instructions issued, the gathers of scales among them; a place to meet for every
// tile, and one wavefront there adding while the others wait at the next, took 88 us).
template <int PP, int AHEAD, int STEPS, typename S>
__global__ __launch_bounds__(8 * RI_WAVE, 2) void gemm_int4_rows_kernel(const I4Args a) {
    constexpr int W = 8, USES = 4 / STEPS, BLOCKS = (PP * USES + 3) / 4;       // groups that a piece meets; loads of four groups for the pieces
    __shared__ __attribute__((aligned(16))) float4 meet[2][W][W][RI_WAVE];
    const int lane = threadIdx.x & (RI_WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / RI_WAVE), i = lane & 15, j = lane >> 4;
    const int tiles = (a.n + 15) / 16, pieces = (a.k + I4_PIECE - 1) / I4_PIECE, first = wave * PP;
    const size_t row_bytes = (size_t)a.k / 2;
    const S* scales = (const S*)a.scales;
    const uint8_t* zeros = a.zeros ? a.zeros : i4_zero_point;
    const uint32_t zero_mask = a.zeros ? ~0u : 0u;

    uint32_t mask = 0x00780078u, sixteen = I4_SIXTEEN;
    ma_opaque(mask);
    ma_here(sixteen);
    I4Frag ones, xf[PP][4];
    float sum[BLOCKS];                                        // of the groups that lane group j holds
    ones.w[0] = ones.w[1] = ones.w[2] = ones.w[3] = I4_ONES;
    const bf16_t* x_row = a.x + (size_t)min(i, a.rows - 1) * a.k;
#pragma unroll
    for (int p = 0; p < PP; ++p)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k = (first + p) * I4_PIECE + column_of<STEPS>(s, j);
            xf[p][s].u = *reinterpret_cast<const uint4*>(k < a.k ? x_row + k : ri_zero_fragment + 8 * lane);
        }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) sum[b] = 0.f;
#pragma unroll
    for (int p = 0; p < PP; ++p) {
#pragma unroll
        for (int s = 0; s < 4; ++s) reorder(xf[p][s], xf[p][s].u);
#pragma unroll
        for (int e = 0; e < USES; ++e) {
            const float one = sum_of<STEPS>(xf[p] + e * STEPS, ones);
            const int use = p * USES + e;
            sum[use / 4] = j == use % 4 ? one : sum[use / 4];
        }
    }
    // A load takes whole 128-byte lines of eight rows: of a pair of pieces lanes 2 r and 2 r + 1 of every sixteen ask for row r's 256 columns
    // in one and for row 8 + r's in the other; then neighbours exchange, so that an even lane holds row r and an odd one row
    // 8 + r, of the first piece and of the second.  (151,936 x 4,096: 79 us; with loads of half a line of sixteen rows, fewer
    // instructions, 87.)  A lane's 32 columns are there whole or not at all: then the row's first, against zeros of x.
    const bool odd = i & 1;
    const int row_of = (i >> 1) + 8 * (i & 1);               // the row of a tile that a lane's column of the product is
    uint32_t at[PP / 2], group[BLOCKS];
#pragma unroll
    for (int p = 0; p < PP / 2; ++p) {
        const int k = (first + 2 * p) * I4_PIECE + 128 * (i & 1) + 32 * j;
        at[p] = k < a.k ? k / 2 : 0;
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        const int use = 4 * b + j, piece = min(first + min(use / USES, PP - 1), pieces - 1);
        group[b] = STEPS == 4 ? (a.per == 1 ? piece : piece / a.per) : min(piece * USES + use % USES, a.groups - 1);
    }
    struct Tile { uint4 codes[PP]; S scale[BLOCKS]; uint8_t zero[BLOCKS]; };      // as loaded: a conversion would wait for the load
    // The tiles follow one another at a fixed distance; rows behind the last are the last.  (Offsets of 32 bits, moved on, not made anew:
    // what this loop does is bound by the instructions that it issues.)
    const uint32_t last_row = (uint32_t)(a.n - 1) * (uint32_t)row_bytes, last_groups = (uint32_t)(a.n - 1) * (uint32_t)a.groups;
    const uint32_t row_step = 16u * gridDim.x * (uint32_t)row_bytes, groups_step = 16u * gridDim.x * (uint32_t)a.groups;
    auto row_at = [&](int r) { return (uint32_t)min(16 * (int)blockIdx.x + r, a.n - 1); };
    uint32_t low = row_at(i >> 1) * (uint32_t)row_bytes, high = row_at(8 + (i >> 1)) * (uint32_t)row_bytes, groups = row_at(row_of) * (uint32_t)a.groups;
    auto load = [&](Tile& t) {                                // the next tile's
#pragma unroll
        for (int p = 0; p < PP / 2; ++p) {
            t.codes[2 * p] = load16_by4<true>(a.codes + (low + at[p]));
            t.codes[2 * p + 1] = load16_by4<true>(a.codes + (high + at[p]));
        }
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const uint32_t g = groups + group[b];
            t.scale[b] = *reinterpret_cast<const S*>(reinterpret_cast<const char*>(scales) + (uint32_t)(g * sizeof(S)));
            t.zero[b] = zeros[g & zero_mask];
        }
        low = last_row - low < row_step ? last_row : low + row_step;
        high = last_row - high < row_step ? last_row : high + row_step;
        groups = last_groups - groups < groups_step ? last_groups : groups + groups_step;
    };
    auto work = [&](const Tile& t, int turn) {
        i4_floatx4 total = {0.f, 0.f, 0.f, 0.f};
        float scale[BLOCKS][4];
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const float own = to_f32(t.scale[b]);
            to_all(scale[b], own);
            add_product4(total, sum[b], taken_off(own, t.zero[b]));
        }
        I4Frag wf[2][4];
#pragma unroll
        for (int p = 0; p < PP; ++p) {
            const uint4 lo = t.codes[p & ~1], hi = t.codes[p | 1];
            uint32_t w[4];
            if (p % 2 == 0) {
                w[0] = from_even(odd, lo.x, hi.x), w[1] = from_even(odd, lo.y, hi.y);
                w[2] = from_even(odd, lo.z, hi.z), w[3] = from_even(odd, lo.w, hi.w);
            } else {
                w[0] = from_odd(odd, lo.x, hi.x), w[1] = from_odd(odd, lo.y, hi.y);
                w[2] = from_odd(odd, lo.z, hi.z), w[3] = from_odd(odd, lo.w, hi.w);
            }
            turn_words<STEPS>(w);
#pragma unroll
            for (int s = 0; s < 4; ++s) widen(wf[p % 2][s], w[s], mask, sixteen);
            if (p % 2 == 0) continue;
            // two pieces' products, none of which waits for another one's sum, then what they weigh
            i4_floatx4 acc[2][USES];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < USES; ++e) acc[h][e] = i4_floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < USES; ++e)
                        acc[h][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[p - 1 + h][e * STEPS + s].v, wf[h][e * STEPS + s].v, acc[h][e], 0, 0, 0);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < USES; ++e) {
                    const int use = (p - 1 + h) * USES + e;
#pragma unroll
                    for (int q = 0; q < 4; ++q) total[q] = fmaf(scale[use / 4][use % 4], acc[h][e][q], total[q]);
                }
        }
        meet[turn / W & 1][turn % W][wave][lane] = make_float4(total[0], total[1], total[2], total[3]);
    };
    auto store = [&](int tile, int turn) {                    // the tile of that turn, added up
        const auto& from = meet[turn / W & 1][turn % W];
        float4 o = from[0][lane];
#pragma unroll
        for (int v = 1; v < W; ++v) {
            const float4 more = from[v][lane];
            o = make_float4(o.x + more.x, o.y + more.y, o.z + more.z, o.w + more.w);
        }
        const int col = 16 * tile + row_of;
        const float value[4] = {o.x * I4_BACK, o.y * I4_BACK, o.z * I4_BACK, o.w * I4_BACK};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int m = 4 * j + e;
            if (m < a.rows && col < a.n) {
                if (a.out_f32) ((float*)a.out)[(size_t)m * a.n + col] = value[e];
                else ((bf16_t*)a.out)[(size_t)m * a.n + col] = f32_to_bf16(value[e]);
            }
        }
    };
    const int step = gridDim.x;
    Tile ring[AHEAD + 1];
    int tile = blockIdx.x, turn = 0;
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
        load(ring[d]);
        __builtin_amdgcn_sched_barrier(0);                    // (in this order: the loop's waits count by the order of entry too)
    }
    do {                                                      // (one way out: with one a tile the compiler waits for every load at the top)
#pragma unroll
        for (int d = 0; d <= AHEAD; ++d) {
            load(ring[(d + AHEAD) % (AHEAD + 1)]);
            __builtin_amdgcn_sched_barrier(0);
            if (tile < tiles) {
                work(ring[d], turn);
                if (turn % W == W - 1 || tile + step >= tiles) {
                    __syncthreads();                          // (a buffer is written again behind the next such place)
                    const int mine = turn / W * W + wave;
                    if (mine <= turn) store(blockIdx.x + mine * step, mine);
                }
                ++turn;
            }
            tile += step;
        }
    } while (tile < tiles);
}

template <int PP, int AHEAD>
static void int4_rows(const I4Args& a, int group, bool scale_f32, hipStream_t s) {
    const int tiles = (a.n + 15) / 16, rounds = (tiles + ri_compute_units() - 1) / ri_compute_units();
    const unsigned grid = (tiles + rounds - 1) / rounds;      // (as many tiles a workgroup)
#define I4_ROWS_LAUNCH(STEPS)                                                                                    \
    do {                                                                                                         \
        if (scale_f32) gemm_int4_rows_kernel<PP, AHEAD, STEPS, float><<<grid, 8 * RI_WAVE, 0, s>>>(a);           \
        else gemm_int4_rows_kernel<PP, AHEAD, STEPS, bf16_t><<<grid, 8 * RI_WAVE, 0, s>>>(a);                    \
    } while (0)
    if (group == 32) I4_ROWS_LAUNCH(1);
    else if (group == 64) I4_ROWS_LAUNCH(2);
    else I4_ROWS_LAUNCH(4);
#undef I4_ROWS_LAUNCH
}

template <int MT, int NT, int W>
static void int4_tiles(const I4Args& a, int group, bool scale_f32, hipStream_t s) {
    const dim3 grid((a.n + 16 * NT - 1) / (16 * NT), (a.rows + 16 * MT - 1) / (16 * MT));
#define I4_LAUNCH(STEPS)                                                                                         \
    do {                                                                                                         \
        if (scale_f32) gemm_int4_kernel<MT, NT, W, STEPS, float><<<grid, W * RI_WAVE, 0, s>>>(a);                \
        else gemm_int4_kernel<MT, NT, W, STEPS, bf16_t><<<grid, W * RI_WAVE, 0, s>>>(a);                         \
    } while (0)
    if (group == 32) I4_LAUNCH(1);
    else if (group == 64) I4_LAUNCH(2);
    else I4_LAUNCH(4);
#undef I4_LAUNCH
}

// What a compute unit does: the rounds in which the workgroups of `tall` x `wide` tiles go, times their tiles.
static long int4_rounds(const I4Args& a, int tall, int wide) {
    const long rows = (a.rows + 16 * tall - 1) / (16 * tall), cols = (a.n + 16 * wide - 1) / (16 * wide), units = ri_compute_units();
    return (rows * cols + units - 1) / units * tall * wide;
}

extern "C" int ri_gemm_int4_bf16(void* out, int out_dtype, const void* x, const void* codes, const void* scales, int scale_dtype,
                                 const void* zeros, int rows, int n, int k, int group, void* stream) {
    RI_REQUIRE(rows >= 1 && n >= 1 && k >= 8, "gemm_int4: %d rows, n %d, k %d", rows, n, k);
    RI_REQUIRE(k % 8 == 0, "gemm_int4: k %d is no multiple of 8", k);
    RI_REQUIRE(group == 32 || group == 64 || (group > 0 && group % 128 == 0),
               "gemm_int4: groups of %d columns, 32, 64 and multiples of 128 are taken", group);
    RI_REQUIRE(rows <= 65535 * 16 && n <= 0x7fffffff - 64, "gemm_int4: %d rows, n %d are too many", rows, n);
    RI_REQUIRE((out_dtype == RI_F32 || out_dtype == RI_BF16) && (scale_dtype == RI_F32 || scale_dtype == RI_BF16), "gemm_int4: unknown dtype");
    RI_REQUIRE(out && x && codes && scales, "gemm_int4: an operand is missing");
    RI_REQUIRE((uintptr_t)x % 16 == 0, "gemm_int4: x must start on a 16-byte boundary");
    RI_REQUIRE((uintptr_t)codes % 4 == 0, "gemm_int4: the codes must start on a 4-byte boundary");
    const int groups = (k - 1) / group + 1;                   // (k + group may pass 32 bits)
    const I4Args a = {out, (const bf16_t*)x, (const uint8_t*)codes, scales, (const uint8_t*)zeros, rows, n, k, groups,
                      group >= 128 ? group / 128 : 1, out_dtype == RI_F32};
    const bool f = scale_dtype == RI_F32;
    const hipStream_t s = (hipStream_t)stream;
    const int pieces = (k + I4_PIECE - 1) / I4_PIECE, tiles = (n + 15) / 16, units = ri_compute_units();
    // More tiles of matrix rows than compute units: x is held and the matrix walked.  In us, so and by tiles: 1 x 8192 x 4096 7.1 and 8.5,
    // 4 x 12288 x 4096 8.8 and 13.4, 16 x 24576 x 4096 15.5 and 25, 16 x 151936 x 4096 77 and 135; 4 x 5120 x 2560 level.  The registers of
    // eight wavefronts hold 32 pieces of 16 rows; beyond K = 4096 all products go by tiles (1 and 16 rows, of the time that the bytes take:
    // 55296 x 5120 1.5 and 2.1 times, 57344 x 8192 1.5 and 2.0, where 24576 x 4096 takes 1.2 and 1.4).
    if (rows <= 16 && k % 32 == 0 && pieces <= 32 && (long)n * (k / 2) <= 0xffffffffL && tiles > units) {
        if (pieces <= 16) int4_rows<2, 2>(a, group, f, s);
        else int4_rows<4, 1>(a, group, f, s);
    } else if ((long)tiles * ((rows + 15) / 16) <= units) {
        // A tile a workgroup, and eight wavefronts on the length of K, where every one has a compute unit to itself: 4096 x 4096 takes
        // 5.6 us with one row and 8.5 with 16 (two tiles by four wavefronts: 8.2 and 9.8; four tiles: 11.7 and 13.3).
        int4_tiles<1, 1, 8>(a, group, f, s);
    } else {
        // Else the tiles that leave the compute units the least to do, and up to an eighth more of it where they are larger: x, or the
        // codes, are then read less often.  In us, 1 x 2, 1 x 4 and 4 x 2 tiles: 45 x 2560 x 9728 17.7, 24.4, 36.8; 48 x 19456 x 2560
        // 33.0, 27.8, 33.4; 64 x 151936 x 2560 284, 225, 214; 256 x 4096 x 4096 57, 45, 40.  (Eight wavefronts: up to 8% more.)
        const long two = int4_rounds(a, 1, 2), four = int4_rounds(a, 1, 4), eight = int4_rounds(a, 4, 2);
        if (8 * eight <= 9 * min(two, four)) int4_tiles<4, 2, 4>(a, group, f, s);
        else if (8 * four <= 9 * two) int4_tiles<1, 4, 4>(a, group, f, s);
        else int4_tiles<1, 2, 4>(a, group, f, s);
    }
    RI_LAUNCH_CHECK("gemm_int4");
    return 0;
}
