// Rows of bfloat16 times a matrix kept in 4 bits, with a scale and a zero point per group of its columns:
//
//     out[m, n] = sum over groups g of  s[n, g] ( sum_{k in g} x[m, k] c[n, k]  -  z[n, g] sum_{k in g} x[m, k] )
//
// The matrix is read as it is stored, a row after the other, two codes a byte.  A wavefront takes NT tiles of 16 matrix rows
// and walks K in pieces of 128: a lane loads 16 bytes, 32 codes of one row, and four lane swaps turn the 4 x 4 words that
// the four lanes of a row hold, so that step s of the piece has columns 32 s + 8 j .. +7 in lane group j: the operand order of
// the matrix cores' 16 x 16 x 32 product, with x loaded in the same order.
//
// A code c becomes a bfloat16 by three bits of arithmetic: 16.0 has a step of 1/8 in its last place, so 0x4180 | c << 3 is
// 16 + c, exactly, and two codes that lie 16 bits apart in a word turn in one instruction pair (mask and or after a shift).
// What that adds, (16 + z) sum x, goes out again with sums of x that the matrix cores make of the same operands against
// ones; both sums are float32 and the groups are short, so a sum of 128 numbers of 16 to 31 costs the result some three bits
// of float32's 24.  Two codes that neighbour in a word are four columns apart, so x's words are permuted alike.
//
// The wavefronts of a workgroup share the K pieces in turn and meet in LDS, in order.  Rows of x beyond M repeat the last
// one (a row of the product depends on its own row of x alone) and are not stored; columns beyond K are zeros of x.
#include "api.h"
#include "common.h"

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 i4_bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float i4_floatx4;

union I4Frag {
    i4_bf16x8 v;
    uint4 u;
    uint32_t w[4];
};

#define I4_PIECE 128             // columns a wavefront takes at a time: 16 bytes of codes a lane
#define I4_ROWS 64               // rows of x a workgroup takes at most

struct I4Args {
    void* out;
    const bf16_t* x;
    const uint8_t* codes;
    const void* scales;
    const uint8_t* zeros;        // NULL: every zero point is 8
    int rows, n, k, groups, per; // per: pieces of 128 columns that share a group (groups of 128 and more)
    int out_f32;
};

// Sixteen bytes from an address that is a multiple of four.
__device__ __forceinline__ uint4 load16_by4(const uint8_t* p) {
    typedef unsigned int u32x4_t __attribute__((ext_vector_type(4), aligned(4)));
    const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
    return make_uint4(v.x, v.y, v.z, v.w);
}

// Word w of lane group s and word s of lane group w change places.
__device__ __forceinline__ void turn_words(uint32_t (&w)[4]) {
    typedef unsigned __attribute__((ext_vector_type(2))) pair_t;
    const pair_t a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const pair_t b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const pair_t c = __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false);
    const pair_t d = __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false);
    w[0] = c.x;
    w[1] = c.y;
    w[2] = d.x;
    w[3] = d.y;
}

// Eight codes as 16 + c, in the order 0 4 1 5 2 6 3 7 of the word's nibbles.
__device__ __forceinline__ void widen(I4Frag& f, uint32_t w) {
    f.w[0] = ((w << 3) & 0x00780078u) | 0x41804180u;
    f.w[1] = ((w >> 1) & 0x00780078u) | 0x41804180u;
    f.w[2] = ((w >> 5) & 0x00780078u) | 0x41804180u;
    f.w[3] = ((w >> 9) & 0x00780078u) | 0x41804180u;
}
// Eight neighbouring numbers in the same order.
__device__ __forceinline__ void reorder(I4Frag& f, const uint4 u) {
    f.w[0] = __builtin_amdgcn_perm(u.z, u.x, 0x05040100u);
    f.w[1] = __builtin_amdgcn_perm(u.z, u.x, 0x07060302u);
    f.w[2] = __builtin_amdgcn_perm(u.w, u.y, 0x05040100u);
    f.w[3] = __builtin_amdgcn_perm(u.w, u.y, 0x07060302u);
}

__device__ __forceinline__ float scale_at(const float* s, size_t i) { return s[i]; }
__device__ __forceinline__ float scale_at(const bf16_t* s, size_t i) { return bf16_to_f32(s[i]); }

// MT tiles of 16 rows of x, NT tiles of 16 rows of the matrix, W wavefronts.  STEPS: steps of 32 columns that share a group
// (4: groups are multiples of 128).
template <int MT, int NT, int W, int STEPS, typename S>
__global__ __launch_bounds__(W * RI_WAVE) void gemm_int4_kernel(const I4Args a) {
    const int lane = threadIdx.x & (RI_WAVE - 1), wave = threadIdx.x / RI_WAVE, i = lane & 15, j = lane >> 4;
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * I4_ROWS;
    const int pieces = (a.k + I4_PIECE - 1) / I4_PIECE;
    const size_t row_bytes = (size_t)a.k / 2;
    const S* scales = (const S*)a.scales;
    int col[NT];
    const uint8_t* code_row[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        col[t] = min(n0 + 16 * t + i, a.n - 1);
        code_row[t] = a.codes + col[t] * row_bytes;
    }
    const bf16_t* x_row[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x_row[t] = a.x + (size_t)min(m0 + 16 * t + i, a.rows - 1) * a.k;

    i4_floatx4 total[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int t = 0; t < NT; ++t) total[mt][t] = i4_floatx4{0.f, 0.f, 0.f, 0.f};
    I4Frag ones;
    ones.w[0] = ones.w[1] = ones.w[2] = ones.w[3] = 0x3F803F80u;

    for (int p = wave; p < pieces; p += W) {
        const int k0 = p * I4_PIECE;
        uint32_t w[NT][4];
        if (k0 + I4_PIECE <= a.k) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint4 u = load16_by4(code_row[t] + k0 / 2 + 16 * j);
                w[t][0] = u.x, w[t][1] = u.y, w[t][2] = u.z, w[t][3] = u.w;
            }
        } else {                                              // the row ends within the piece
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    w[t][q] = *reinterpret_cast<const uint32_t*>(code_row[t] + min((size_t)(k0 / 2 + 16 * j + 4 * q), row_bytes - 4));
        }
        I4Frag xf[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k = k0 + 32 * s + 8 * j;
                const uint4 u = *reinterpret_cast<const uint4*>(k < a.k ? x_row[mt] + k : ri_zero_fragment + 8 * lane);
                reorder(xf[mt][s], u);
            }
#pragma unroll
        for (int t = 0; t < NT; ++t) turn_words(w[t]);
#pragma unroll
        for (int s0 = 0; s0 < 4; s0 += STEPS) {
            const int group = STEPS == 4 ? (a.per == 1 ? p : p / a.per) : min((4 * p + s0) / STEPS, a.groups - 1);
            i4_floatx4 sum[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                sum[mt] = i4_floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = s0; s < s0 + STEPS; ++s)
                    sum[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[mt][s].v, ones.v, sum[mt], 0, 0, 0);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const size_t at = (size_t)col[t] * a.groups + group;
                const float scale = scale_at(scales, at), off = 16.f + (a.zeros ? (float)a.zeros[at] : 8.f);
                I4Frag wf[STEPS];
#pragma unroll
                for (int s = 0; s < STEPS; ++s) widen(wf[s], w[t][s0 + s]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    i4_floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < STEPS; ++s)
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[mt][s0 + s].v, wf[s].v, acc, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) total[mt][t][e] = fmaf(scale, fmaf(-off, sum[mt][e], acc[e]), total[mt][t][e]);
                }
            }
        }
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
                    if (a.out_f32) ((float*)a.out)[(size_t)m * a.n + c] = total[mt][t][e];
                    else ((bf16_t*)a.out)[(size_t)m * a.n + c] = f32_to_bf16(total[mt][t][e]);
                }
            }
        }
}

template <int MT, int NT, int W, int STEPS>
static void int4_launch(const I4Args& a, bool scale_f32, hipStream_t s) {
    const dim3 grid((a.n + 16 * NT - 1) / (16 * NT), (a.rows + I4_ROWS - 1) / I4_ROWS);
    if (scale_f32) gemm_int4_kernel<MT, NT, W, STEPS, float><<<grid, W * RI_WAVE, 0, s>>>(a);
    else gemm_int4_kernel<MT, NT, W, STEPS, bf16_t><<<grid, W * RI_WAVE, 0, s>>>(a);
}

template <int MT>
static void int4_by_group(const I4Args& a, int group, bool scale_f32, hipStream_t s) {
    if (group == 32) int4_launch<MT, 1, 8, 1>(a, scale_f32, s);
    else if (group == 64) int4_launch<MT, 1, 8, 2>(a, scale_f32, s);
    else int4_launch<MT, 1, 8, 4>(a, scale_f32, s);
}

extern "C" int ri_gemm_int4_bf16(void* out, int out_dtype, const void* x, const void* codes, const void* scales, int scale_dtype,
                                 const void* zeros, int rows, int n, int k, int group, void* stream) {
    RI_REQUIRE(rows >= 1 && n >= 1 && k >= 8, "gemm_int4: %d rows, n %d, k %d", rows, n, k);
    RI_REQUIRE(k % 8 == 0, "gemm_int4: k %d is no multiple of 8", k);
    RI_REQUIRE(group == 32 || group == 64 || (group > 0 && group % 128 == 0),
               "gemm_int4: groups of %d columns, 32, 64 and multiples of 128 are taken", group);
    RI_REQUIRE(rows <= 65535 * I4_ROWS && n <= 0x7fffffff - 64, "gemm_int4: %d rows, n %d are too many", rows, n);
    RI_REQUIRE((out_dtype == RI_F32 || out_dtype == RI_BF16) && (scale_dtype == RI_F32 || scale_dtype == RI_BF16), "gemm_int4: unknown dtype");
    RI_REQUIRE(out && x && codes && scales, "gemm_int4: an operand is missing");
    RI_REQUIRE((uintptr_t)x % 16 == 0, "gemm_int4: x must start on a 16-byte boundary");
    RI_REQUIRE((uintptr_t)codes % 4 == 0, "gemm_int4: the codes must start on a 4-byte boundary");
    const int groups = (k + group - 1) / group;
    const I4Args a = {out, (const bf16_t*)x, (const uint8_t*)codes, scales, (const uint8_t*)zeros, rows, n, k, groups,
                      group >= 128 ? group / 128 : 1, out_dtype == RI_F32};
    const bool f = scale_dtype == RI_F32;
    const hipStream_t s = (hipStream_t)stream;
    const int mt = rows >= I4_ROWS ? 4 : (rows + 15) / 16;
    if (mt == 1) int4_by_group<1>(a, group, f, s);
    else if (mt == 2) int4_by_group<2>(a, group, f, s);
    else if (mt == 3) int4_by_group<3>(a, group, f, s);
    else int4_by_group<4>(a, group, f, s);
    RI_LAUNCH_CHECK("gemm_int4");
    return 0;
}
