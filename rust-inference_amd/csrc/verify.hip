// Drafted tokens held to the target's distribution.  A sequence brings n rows of logits: its last known token's and
// those of the n - 1 tokens drafted behind it (tokens[r0 + 1 ..]).  With p_r = softmax(logits_r / T), q_j the
// distribution that token j was drafted from and u the given random numbers, the draft at row r + 1 stands if
//
//     u_r q_{r+1}(d) < p_r(d),  d = tokens[r + 1]
//
// and every draft before it stands.  At the first row r that has no draft left or whose draft falls, one more token is
// drawn with the sequence's last number u_last: from p_r where no draft is left, else from max(p_r - q_{r+1}, 0) made a
// distribution again.  Then the token put out at every place is distributed as p.  Without draft logits the drafts are
// given (looked up, not drawn): q is 1 at the draft and 0 elsewhere.  The draw takes the first token whose running
// weight, by rising id, passes u_last times the weight of all.
//
// Everything that is compared is a float64: a token is the answer to "on which side of a border does u lie", a
// vocabulary has 10^5 borders, and float32 weights put one draw in 10^3 to 10^5 on the wrong side.  The exponential keeps 40 of the 53
// bits (relative error 1.1e-12, which puts less than one draw in 10^6 on the other side): the vector unit takes
// float64 well, so that its fourteen instructions (Exps, below) stand beside an entry's 4 bytes; each bit more would cost time in a pass
// that it bounds already.
//
// Four launches.  `stats` cuts every row that is asked about into chunks of 4,096 entries, a wavefront each, and leaves a
// chunk's largest logit and its sum of exponentials: the one pass over the logits.  `end` (a workgroup a sequence) joins the
// rows' chunks, a row a wavefront, until a draft falls; where there is little to do `weigh` does that beside its own work.
// `weigh` sums what the entries of every chunk weigh in the draw of the last token, `pick` (a workgroup a sequence) finds the
// chunk and in it the token.  Greedy steps need two: the chunks' best entries, then the walk.
// Every sum has one order, so the same inputs give the same tokens.
#include <float.h>

#include "api.h"
#include "common.h"

#define VER_CHUNK 4096
#define VER_THREADS 256
#define VER_WAVES (VER_THREADS / RI_WAVE)
#define VER_PICK_THREADS 1024
#define VER_PICK_EACH (VER_CHUNK / VER_PICK_THREADS)

// With s = log2(e) / T, the exponential of a logit x over that of the largest one m is 2^((x - m) s).
struct ChunkStats { double top, sum; };          // of a chunk of a row: m, the sum over its entries
struct RowStats { double top, inv; };            // of a row: m, 1 / the sum (0 where every entry is masked)
// Where a sequence's walk ended: the row that the last token is drawn from, the draft that fell there (-1: none did, or it
// has a distribution of its own), and the statistics of both distributions.
struct Ending {
    RowStats p, q;
    int row, less, fell, unused;
};

#define VER_MAGIC 6755399441055744.0             // 1.5 * 2^52: a number added to it is rounded to a whole one, in the lowest bits

// 2^f for |f| <= 1/2 times 2^n, n the low 32 bits of `whole`: the polynomial of degree 8 that equals 2^f at the nine Chebyshev
// points of [-1/2, 1/2] (relative error under 1.1e-12); n is added to the exponent, which has to have room for it.
__device__ __forceinline__ double exp2_parts(double f, double whole) {
    double s = 1.3255224878668817e-06;
    s = fma(s, f, 1.5310079402249296e-05);
    s = fma(s, f, 0.00015403455852453838);
    s = fma(s, f, 0.0013333450568000645);
    s = fma(s, f, 0.0096181291594025584);
    s = fma(s, f, 0.055504109412059327);
    s = fma(s, f, 0.24022650695812989);
    s = fma(s, f, 0.69314718054593349);
    s = fma(s, f, 1.0);
    typedef uint32_t __attribute__((ext_vector_type(2))) halves_t;
    halves_t bits = __builtin_bit_cast(halves_t, s);
    bits.y += __builtin_bit_cast(halves_t, whole).x << 20;
    return __builtin_bit_cast(double, bits);
}
// 2^t for t <= 0: t = n + f by adding and taking off 1.5 * 2^52.  t is held to -1000 (NaN with it), where 2^t is 1e-301, nothing
// beside a sum of at least 1.
__device__ __forceinline__ double exp2_nonpositive(double t) {
    t = fmin(fmax(t, -1000.0), 0.0);
    const double y = t + VER_MAGIC;
    return exp2_parts(t - (y - VER_MAGIC), y);
}

// The exponentials of a row's (or a chunk's) entries over that of its largest one.  Ordinary temperatures: with M the whole
// number next to m s, 2^(x s - M) takes eleven float64 instructions, a conversion, a clamp and an addition to the exponent, since
// x s + (1.5 * 2^52 - M) has the whole part in place at once, and x is held in float32 to what the exponent has room for: lo, where the result is 2^-1000 up to the
// rounding of lo, which is that of a normal number (2^-24, some 2^3 exponents) where |M| is below 2^27, lo in float32's range and s below
// 2^80 (lo, where it is not 0, is a whole number of 1 / s); `plain` does without.  NaN and what lies at lo or below is a masked entry, an
// infinite logit the largest finite number.
struct Scale { double s, inv; };                 // log2(e) / T and its inverse
struct Exps {
    double s, c, back;           // log2(e) / T; 1.5 * 2^52 - M; 2^(M - m s)
    float top, lo;
    bool plain;
};
__device__ __forceinline__ Exps exps_below(double m, Scale by) {
    Exps r;
    const double whole = rint(m * by.s);
    r.s = by.s;
    r.top = (float)m;
    const double lo = (whole - 1000.0) * by.inv;
    r.plain = !(fabs(whole) < 134217728.0 && lo >= -FLT_MAX && by.s < 1.2089258196146292e24);
    r.c = VER_MAGIC - whole;
    r.lo = (float)lo;
    r.back = r.plain ? 1.0 : exp2_parts(fma(-m, by.s, whole), 0.0);
    return r;
}
// What `back` times it is the exponential of x.
template <bool PLAIN>
__device__ __forceinline__ double term(const Exps& r, float x) {
    if (PLAIN) return exp2_nonpositive(((double)x - (double)r.top) * r.s);
    const double d = __builtin_amdgcn_fmed3f(x, r.lo, r.top);           // (with a NaN the least of the others)
    const double y = fma(d, r.s, r.c);
    return exp2_parts(fma(d, r.s, r.c - y), y);
}
// The same with 0 for a masked entry, where it matters whether an entry weighs anything at all.
template <bool PLAIN>
__device__ __forceinline__ double term_or_zero(const Exps& r, float x) {
    const double e = term<PLAIN>(r, x);
    const bool some = PLAIN ? ((double)x - (double)r.top) * r.s > -1000.0 || x > r.top : x > r.lo;
    return some ? e : 0.0;
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int m = RI_WAVE / 2; m > 0; m >>= 1) v += __shfl_xor(v, m, RI_WAVE);
    return v;
}
__device__ __forceinline__ double wave_max_d(double v) {
#pragma unroll
    for (int m = RI_WAVE / 2; m > 0; m >>= 1) v = fmax(v, __shfl_xor(v, m, RI_WAVE));
    return v;
}

// A thread's entries of a chunk of n entries; those that are not there are masked.  WIDE: the row starts on a 16-byte
// boundary and its length is a multiple of 4.
template <bool WIDE, int EACH>
__device__ __forceinline__ void load_chunk(float (&v)[EACH], const float* __restrict__ x, int n) {
    constexpr int THREADS = VER_CHUNK / EACH;
    if (n == VER_CHUNK) {                                     // (all chunks but a row's last: no looks at the end)
        if (WIDE) {
#pragma unroll
            for (int u = 0; u < EACH / 4; ++u) {
                const float4 w = *reinterpret_cast<const float4*>(x + 4 * (u * THREADS + threadIdx.x));
                v[4 * u] = w.x, v[4 * u + 1] = w.y, v[4 * u + 2] = w.z, v[4 * u + 3] = w.w;
            }
        } else {
#pragma unroll
            for (int u = 0; u < EACH; ++u) v[u] = x[u * THREADS + threadIdx.x];
        }
        return;
    }
    if (WIDE) {
#pragma unroll
        for (int u = 0; u < EACH / 4; ++u) {
            const int i = 4 * (u * THREADS + threadIdx.x);
            const float4 w = *reinterpret_cast<const float4*>(x + min(i, n - 4));
            v[4 * u] = i < n ? w.x : -INFINITY;
            v[4 * u + 1] = i < n ? w.y : -INFINITY;
            v[4 * u + 2] = i < n ? w.z : -INFINITY;
            v[4 * u + 3] = i < n ? w.w : -INFINITY;
        }
    } else {
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const int i = u * THREADS + threadIdx.x;
            const float w = x[min(i, n - 1)];
            v[u] = i < n ? w : -INFINITY;
        }
    }
}
// The place in its chunk of a thread's entry e.
template <bool WIDE, int EACH>
__device__ __forceinline__ int place_of(int e) {
    constexpr int THREADS = VER_CHUNK / EACH;
    return WIDE ? 4 * ((e / 4) * THREADS + threadIdx.x) + e % 4 : e * THREADS + threadIdx.x;
}

// The rows of a sequence, held to the rows there are.
__device__ __forceinline__ void rows_of(const int32_t* __restrict__ cu, int b, int rows, int& r0, int& r1) {
    r0 = min(max(cu[b], 0), rows);
    r1 = min(max(cu[b + 1], r0), rows);
}

// Whether a row belongs to a sequence, and whether it is not the first of its own (then its token is a draft).  Asked by a
// whole wavefront, a lane a sequence.
__device__ __forceinline__ void place_of_row(const int32_t* __restrict__ cu, int seqs, int rows, int row, bool& within, bool& drafted) {
    int in = 0, first = 0;
    for (int b = threadIdx.x & (RI_WAVE - 1); b < seqs; b += RI_WAVE) {
        int r0, r1;
        rows_of(cu, b, rows, r0, r1);
        in |= row >= r0 && row < r1;
        first |= row == r0 && row < r1;
    }
    within = __any(in);
    drafted = within && !__any(first);
}

// A chunk a wavefront, 64 entries a lane: what is done once a wavefront (place, reductions) is a fifth of its instructions so, a
// third with 32.  The vector unit bounds this pass nearly as the memory does (320 rows x 151,936 and 256 of drafts, 350 MB: 63 to 69 us, 5.1 to
// 5.6 TB/s; with the 64 rows of draft logits that are no draft's read too 70.5 where it is 69).
template <bool WIDE>
__global__ __launch_bounds__(RI_WAVE) void verify_stats(ChunkStats* __restrict__ stats, const float* __restrict__ logits,
                                                        const float* __restrict__ draft, const int32_t* __restrict__ cu, int seqs,
                                                        int rows, int vocab, int chunks, Scale scale) {
    constexpr int EACH = VER_CHUNK / RI_WAVE;
    const int chunk = blockIdx.x, row = blockIdx.y;
    const bool of_draft = blockIdx.z == 1;
    const int at = chunk * VER_CHUNK, n = min(VER_CHUNK, vocab - at);
    float v[EACH];
    bool within, drafted;
    if (of_draft) {                                           // (a row of every sequence is no draft's: not read)
        place_of_row(cu, seqs, rows, row, within, drafted);
        if (!drafted) return;
    }
    load_chunk<WIDE>(v, (of_draft ? draft : logits) + (size_t)row * vocab + at, n);
    if (!of_draft) {                                          // (nearly every row is a sequence's: read beside the question)
        place_of_row(cu, seqs, rows, row, within, drafted);
        if (!within) return;
    }
    float top = -INFINITY;                                    // (the larger of a number and NaN is the number)
#pragma unroll
    for (int e = 0; e < EACH; ++e) top = fmaxf(top, v[e]);
    top = wave_max(top);
    const double m = fminf(top, FLT_MAX);
    const Exps r = exps_below(m, scale);
    double sum = 0.0, more = 0.0;
    if (r.plain) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) sum += term<true>(r, v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < EACH; e += 2) {
            sum += term<false>(r, v[e]);
            more += term<false>(r, v[e + 1]);
        }
    }
    sum = wave_sum_d(sum + more) * r.back;
    if (threadIdx.x == 0) stats[((size_t)blockIdx.z * rows + row) * chunks + chunk] = {m, top > -INFINITY ? sum : 0.0};
}

// A row's chunks joined, by a wavefront, in an order that the number of chunks alone decides.
__device__ __forceinline__ RowStats join_row(const ChunkStats* __restrict__ c, int chunks, Scale scale) {
    const int lane = threadIdx.x & (RI_WAVE - 1);
    double m = -INFINITY;
    for (int i = lane; i < chunks; i += RI_WAVE) m = fmax(m, c[i].top);
    m = wave_max_d(m);
    double s = 0.0;
    for (int i = lane; i < chunks; i += RI_WAVE) s += c[i].sum * exp2_nonpositive((c[i].top - m) * scale.s);
    s = wave_sum_d(s);
    return {m, s > 0.0 ? 1.0 / s : 0.0};
}

__device__ __forceinline__ double probability(const RowStats s, float x, Scale scale) {
    const Exps r = exps_below(s.top, scale);
    return (r.plain ? term_or_zero<true>(r, x) : term_or_zero<false>(r, x)) * r.back * s.inv;
}

// What an entry weighs in the last draw: first in the distribution that is left, second in p itself (taken where nothing is
// left, as when p and q are equal up to their rounding).
struct Weights { double left, whole; };
struct Weigher {
    Exps p, q;
    double p_inv, q_inv;
    int less;                    // the entry that a fallen draft without a distribution takes out, -1: none
    bool has_q, plain;           // plain: one of the two wants it, both are taken so
};
__device__ __forceinline__ Weigher weigher(const Ending& e, bool with_draft, Scale scale) {
    Weigher w;
    w.has_q = with_draft && e.fell;
    w.p = exps_below(e.p.top, scale);
    w.q = exps_below(w.has_q ? e.q.top : e.p.top, scale);
    w.plain = w.p.plain || w.q.plain;
    w.p_inv = w.plain ? e.p.inv : w.p.back * e.p.inv;
    w.q_inv = w.plain ? e.q.inv : w.q.back * e.q.inv;
    w.less = e.fell && !with_draft ? e.less : -1;
    return w;
}
template <bool PLAIN, bool HAS_Q>
__device__ __forceinline__ Weights weigh_entry(const Weigher& w, float x, float qx, int id) {
    const double p = term_or_zero<PLAIN>(w.p, x) * w.p_inv;
    if (HAS_Q) return {fmax(fma(-w.q_inv, term_or_zero<PLAIN>(w.q, qx), p), 0.0), p};
    return {id == w.less ? 0.0 : p, p};
}

// Where a sequence's walk ends, by a workgroup: four rows at a time, a wavefront each, until one ends it; the last row always does.
__device__ __forceinline__ Ending ending_of(const ChunkStats* __restrict__ stats, const float* __restrict__ logits,
                                            const float* __restrict__ draft, const int32_t* __restrict__ tokens,
                                            const float* __restrict__ uniform, int r0, int r1, int rows, int vocab, int chunks, Scale scale) {
    const int lane = threadIdx.x & (RI_WAVE - 1), wave = threadIdx.x / RI_WAVE;
    __shared__ Ending tried[VER_WAVES];
    for (int base = r0;; base += VER_WAVES) {
        const int row = base + wave;
        Ending mine = {{0.0, 0.0}, {0.0, 0.0}, -1, -1, 0, 0};
        if (row < r1) {
            const bool last = row == r1 - 1;
            const int d = last ? -1 : tokens[row + 1];
            const bool known = d >= 0 && d < vocab;           // a draft that is no token of the vocabulary falls
            const float x = logits[(size_t)row * vocab + (known ? d : 0)];
            float qx = 0.f;
            if (draft && !last) {
                qx = draft[(size_t)(row + 1) * vocab + (known ? d : 0)];
                mine.q = join_row(stats + ((size_t)rows + row + 1) * chunks, chunks, scale);
            }
            mine.p = join_row(stats + (size_t)row * chunks, chunks, scale);
            const double p = known ? probability(mine.p, x, scale) : 0.0;
            const double q = !known ? 0.0 : draft ? probability(mine.q, qx, scale) : 1.0;
            const bool stands = (double)uniform[row] * q < p;
            if (last || !stands) {
                mine.row = row;
                mine.less = d;
                mine.fell = !last;
            }
        }
        if (lane == 0) tried[wave] = mine;
        __syncthreads();
        int first = -1;
        for (int w = VER_WAVES - 1; w >= 0; --w)
            if (tried[w].row >= 0) first = w;
        if (first >= 0) return tried[first];
        __syncthreads();
    }
}

template <bool PLAIN, bool HAS_Q, bool WIDE, int EACH>
__device__ __forceinline__ Weights sum_weights(const Weigher& by, const float (&x)[EACH], const float (&qx)[EACH], int at) {
    Weights sum = {0.0, 0.0};
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const Weights w = weigh_entry<PLAIN, HAS_Q>(by, x[e], qx[e], at + place_of<WIDE, EACH>(e));
        sum.left += w.left;
        sum.whole += w.whole;
    }
    return sum;
}

__global__ __launch_bounds__(VER_THREADS) void verify_end(Ending* __restrict__ endings, const ChunkStats* __restrict__ stats,
                                                          const float* __restrict__ logits, const float* __restrict__ draft,
                                                          const int32_t* __restrict__ tokens, const int32_t* __restrict__ cu,
                                                          const float* __restrict__ uniform, int rows, int vocab, int chunks, Scale scale) {
    int r0, r1;
    rows_of(cu, blockIdx.x, rows, r0, r1);
    if (r0 == r1) return;
    const Ending end = ending_of(stats, logits, draft, tokens, uniform, r0, r1, rows, vocab, chunks, scale);
    if (threadIdx.x == 0) endings[blockIdx.x] = end;
}

// ENDS: every workgroup finds its sequence's ending for itself, the first chunk's leaves it for `pick`.
template <bool WIDE, bool ENDS>
__global__ __launch_bounds__(VER_THREADS) void verify_weigh(Weights* __restrict__ masses, Ending* __restrict__ endings,
                                                            const ChunkStats* __restrict__ stats, const float* __restrict__ logits,
                                                            const float* __restrict__ draft, const int32_t* __restrict__ tokens,
                                                            const int32_t* __restrict__ cu, const float* __restrict__ uniform, int rows,
                                                            int vocab, int chunks, Scale scale) {
    constexpr int EACH = VER_CHUNK / VER_THREADS;
    const int chunk = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & (RI_WAVE - 1), wave = threadIdx.x / RI_WAVE;
    __shared__ Weights sums[VER_WAVES];
    int r0, r1;
    rows_of(cu, b, rows, r0, r1);
    if (r0 == r1) return;
    const Ending end = ENDS ? ending_of(stats, logits, draft, tokens, uniform, r0, r1, rows, vocab, chunks, scale) : endings[b];
    if (ENDS && chunk == 0 && threadIdx.x == 0) endings[b] = end;
    const int at = chunk * VER_CHUNK, n = min(VER_CHUNK, vocab - at);
    const Weigher by = weigher(end, draft != nullptr, scale);
    float x[EACH], qx[EACH];
    load_chunk<WIDE>(x, logits + (size_t)end.row * vocab + at, n);
    Weights sum;
    if (by.has_q) {
        load_chunk<WIDE>(qx, draft + (size_t)(end.row + 1) * vocab + at, n);
        sum = by.plain ? sum_weights<true, true, WIDE>(by, x, qx, at) : sum_weights<false, true, WIDE>(by, x, qx, at);
    } else {
        sum = by.plain ? sum_weights<true, false, WIDE>(by, x, x, at) : sum_weights<false, false, WIDE>(by, x, x, at);
    }
    sum.left = wave_sum_d(sum.left);
    sum.whole = wave_sum_d(sum.whole);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < VER_WAVES; ++w) {
            sum.left += sums[w].left;
            sum.whole += sums[w].whole;
        }
        masses[(size_t)b * chunks + chunk] = sum;
    }
}

// What a sequence puts out: the drafts that stand, the token after them, -1 behind it; the rows that are no sequence's, by
// the first workgroup.
__device__ __forceinline__ void put_out(int32_t* __restrict__ accepted, int32_t* __restrict__ out, const int32_t* __restrict__ tokens,
                                        const int32_t* __restrict__ cu, int seqs, int rows, int b, int r0, int r1, int stop, int token) {
    for (int r = r0 + threadIdx.x; r < r1; r += blockDim.x) out[r] = r < stop ? tokens[r + 1] : r == stop ? token : -1;
    if (threadIdx.x == 0) accepted[b] = r1 > r0 ? stop - r0 : 0;
    if (b == 0) {
        const int first = min(max(cu[0], 0), rows), last = min(max(cu[seqs], first), rows);
        for (int r = threadIdx.x; r < first; r += blockDim.x) out[r] = -1;
        for (int r = last + threadIdx.x; r < rows; r += blockDim.x) out[r] = -1;
    }
}

// A wavefront's values with all lanes' before them added, in the order that the steps fix.
__device__ __forceinline__ double wave_upto(double v) {
    const int lane = threadIdx.x & (RI_WAVE - 1);
#pragma unroll
    for (int d = 1; d < RI_WAVE; d *= 2) {
        const double o = __shfl(v, max(lane - d, 0), RI_WAVE);
        v += lane >= d ? o : 0.0;
    }
    return v;
}

// Where the draw falls among a sequence's chunks: the first whose running weight passes the target, else the last that weighs
// anything; what the chunks before it weigh.  By a wavefront, a lane a chunk.
struct Drawn { double target, before; int chunk, whole; };
__device__ __forceinline__ Drawn draw_chunk(const Weights* __restrict__ mine, int chunks, double u) {
    const int lane = threadIdx.x & (RI_WAVE - 1);
    const Weights first = lane < chunks ? mine[lane] : Weights{0.0, 0.0};
    const Weights first_upto = {wave_upto(first.left), wave_upto(first.whole)};
    double left = __shfl(first_upto.left, RI_WAVE - 1, RI_WAVE), whole = __shfl(first_upto.whole, RI_WAVE - 1, RI_WAVE);       // of all chunks
    for (int c0 = RI_WAVE; c0 < chunks; c0 += RI_WAVE) {
        const Weights w = c0 + lane < chunks ? mine[c0 + lane] : Weights{0.0, 0.0};
        left += __shfl(wave_upto(w.left), RI_WAVE - 1, RI_WAVE);
        whole += __shfl(wave_upto(w.whole), RI_WAVE - 1, RI_WAVE);
    }
    Drawn d;
    d.whole = !(left > 0.0);
    d.target = u * (d.whole ? whole : left);
    d.before = 0.0;
    d.chunk = 0;
    double carried = 0.0;
    for (int c0 = 0; c0 < chunks; c0 += RI_WAVE) {
        double own = d.whole ? first.whole : first.left, upto = d.whole ? first_upto.whole : first_upto.left;
        if (c0 > 0) {
            const Weights w = c0 + lane < chunks ? mine[c0 + lane] : Weights{0.0, 0.0};
            own = d.whole ? w.whole : w.left;
            upto = carried + wave_upto(own);
        }
        const unsigned long long some = __ballot(own > 0.0), past = __ballot(own > 0.0 && upto > d.target);
        const unsigned long long take = past ? past & (0ull - past) : some;       // the first past the target, else the last of some
        if (take) {
            const int who = 63 - __clzll((long long)take);
            d.chunk = c0 + who;
            d.before = who > 0 ? __shfl(upto, max(who - 1, 0), RI_WAVE) : carried;
        }
        if (past) break;
        carried = __shfl(upto, RI_WAVE - 1, RI_WAVE);
    }
    return d;
}

__global__ __launch_bounds__(VER_PICK_THREADS) void verify_pick(int32_t* __restrict__ accepted, int32_t* __restrict__ out,
                                                                const Weights* __restrict__ masses, const Ending* __restrict__ endings,
                                                                const float* __restrict__ logits, const float* __restrict__ draft,
                                                                const int32_t* __restrict__ tokens, const int32_t* __restrict__ cu,
                                                                const float* __restrict__ uniform, int seqs, int rows, int vocab,
                                                                int chunks, Scale scale) {
    constexpr int WAVES = VER_PICK_THREADS / RI_WAVE;
    const int b = blockIdx.x, lane = threadIdx.x & (RI_WAVE - 1), wave = threadIdx.x / RI_WAVE;
    __shared__ double of_wave[WAVES];
    __shared__ int first_past[WAVES], last_some[WAVES];
    int r0, r1;
    rows_of(cu, b, rows, r0, r1);
    if (r0 == r1) {
        put_out(accepted, out, tokens, cu, seqs, rows, b, r0, r1, r0, -1);
        return;
    }
    const Ending end = endings[b];
    const Drawn d = draw_chunk(masses + (size_t)b * chunks, chunks, uniform[r1 - 1]);       // (every wavefront for itself)
    const int at = d.chunk * VER_CHUNK, n = min(VER_CHUNK, vocab - at), first = threadIdx.x * VER_PICK_EACH;
    const Weigher by = weigher(end, draft != nullptr, scale);
    double w[VER_PICK_EACH], sum = 0.0;
#pragma unroll
    for (int e = 0; e < VER_PICK_EACH; ++e) {
        const int i = first + e, id = at + min(i, n - 1);
        const float x = logits[(size_t)end.row * vocab + id];
        const float qx = by.has_q ? draft[(size_t)(end.row + 1) * vocab + id] : 0.f;
        const Weights ws = by.has_q ? by.plain ? weigh_entry<true, true>(by, x, qx, id) : weigh_entry<false, true>(by, x, qx, id)
                                    : by.plain ? weigh_entry<true, false>(by, x, qx, id) : weigh_entry<false, false>(by, x, qx, id);
        w[e] = i < n ? (d.whole ? ws.whole : ws.left) : 0.0;
        sum += w[e];
    }
    const double upto = wave_upto(sum);
    if (lane == RI_WAVE - 1) of_wave[wave] = upto;
    __syncthreads();
    double run = d.before;
    for (int v = 0; v < wave; ++v) run += of_wave[v];
    run += upto - sum;
    int past = -1, some = -1;                                 // of this thread's entries
#pragma unroll
    for (int e = VER_PICK_EACH - 1; e >= 0; --e)
        if (w[e] > 0.0 && some < 0) some = first + e;
#pragma unroll
    for (int e = 0; e < VER_PICK_EACH; ++e) {
        run += w[e];
        if (w[e] > 0.0 && run > d.target && past < 0) past = first + e;
    }
    const unsigned long long pasts = __ballot(past >= 0), somes = __ballot(some >= 0);
    if (pasts ? lane == __builtin_ctzll(pasts) : lane == 0) first_past[wave] = past;
    if (somes ? lane == 63 - __clzll((long long)somes) : lane == 0) last_some[wave] = some;
    __syncthreads();
    // (the chunk's sum and its entries' running sum are added up in another order: a target within their rounding of the
    // chunk's end falls to its last entry that weighs anything)
    int place = 0;
    for (int v = 0; v < WAVES; ++v)
        if (last_some[v] >= 0) place = last_some[v];
    for (int v = WAVES - 1; v >= 0; --v)
        if (first_past[v] >= 0) place = first_past[v];
    put_out(accepted, out, tokens, cu, seqs, rows, b, r0, r1, end.row, at + place);
}

// ---- greedy: the best entry of every chunk, then the walk (192 rows x 151,936: 19.5 us, 6 TB/s, and 3.8)
struct Best { float value; int id; };
__device__ __forceinline__ Best better(const Best a, const Best b) {
    return b.value > a.value || (b.value == a.value && b.id < a.id) ? b : a;
}
__device__ __forceinline__ Best wave_best(Best v) {
#pragma unroll
    for (int m = RI_WAVE / 2; m > 0; m >>= 1) {
        const Best o = {__shfl_xor(v.value, m, RI_WAVE), __shfl_xor(v.id, m, RI_WAVE)};
        v = better(v, o);
    }
    return v;
}

template <bool WIDE>
__global__ __launch_bounds__(VER_THREADS) void verify_best(Best* __restrict__ bests, const float* __restrict__ logits, int vocab, int chunks) {
    const int chunk = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & (RI_WAVE - 1), wave = threadIdx.x / RI_WAVE;
    __shared__ Best shared[VER_WAVES];
    const int at = chunk * VER_CHUNK, n = min(VER_CHUNK, vocab - at);
    constexpr int EACH = VER_CHUNK / VER_THREADS;
    float v[EACH];
    load_chunk<WIDE>(v, logits + (size_t)row * vocab + at, n);
    Best best = {-INFINITY, at};                              // (a chunk of masked entries names its first)
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const float x = v[e] > FLT_MAX ? FLT_MAX : v[e];      // (an infinity is the largest number; a NaN stays one)
        if (x > best.value) best = {x, at + place_of<WIDE, EACH>(e)};            // (by rising place; NaN is above nothing)
    }
    best = wave_best(best);
    if (lane == 0) shared[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < VER_WAVES; ++w) best = better(best, shared[w]);
        bests[(size_t)row * chunks + chunk] = best;
    }
}

__global__ __launch_bounds__(VER_THREADS) void verify_walk(int32_t* __restrict__ accepted, int32_t* __restrict__ out,
                                                           const Best* __restrict__ bests, const int32_t* __restrict__ tokens,
                                                           const int32_t* __restrict__ cu, int seqs, int rows, int chunks) {
    const int b = blockIdx.x, lane = threadIdx.x & (RI_WAVE - 1), wave = threadIdx.x / RI_WAVE;
    __shared__ int tried[VER_WAVES];
    int r0, r1;
    rows_of(cu, b, rows, r0, r1);
    int stop = r0, token = -1;
    for (int base = r0; base < r1; base += VER_WAVES) {
        const int row = base + wave;
        int ends = -1;                                        // the best token of a row that ends the walk
        if (row < r1) {
            Best best = {-INFINITY, 0};
            for (int c = lane; c < chunks; c += RI_WAVE) best = better(best, bests[(size_t)row * chunks + c]);
            best = wave_best(best);
            if (row == r1 - 1 || tokens[row + 1] != best.id || best.value == -INFINITY) ends = best.id;      // (a row that masks everything: 0)
        }
        if (lane == 0) tried[wave] = ends;
        __syncthreads();
        int first = -1;
        for (int w = VER_WAVES - 1; w >= 0; --w)
            if (tried[w] >= 0) first = w;
        if (first >= 0) {
            stop = base + first;
            token = tried[first];
            break;
        }
        __syncthreads();
    }
    put_out(accepted, out, tokens, cu, seqs, rows, b, r0, r1, stop, token);
}

static inline int verify_chunks(int vocab) { return (vocab + VER_CHUNK - 1) / VER_CHUNK; }

// Numbers of 8 bytes; 0: such a call is refused (or its workspace would pass 16 GB).
extern "C" int ri_verify_drafts_workspace_words(int seqs, int rows, int vocab, int with_draft) {
    if (seqs < 1 || rows < 1 || vocab < 1 || vocab > 0x7fffffff - VER_CHUNK) return 0;
    const long chunks = verify_chunks(vocab);
    const long bytes = (with_draft ? 2L : 1L) * rows * chunks * (long)sizeof(ChunkStats) + seqs * chunks * (long)sizeof(Weights) +
                       seqs * (long)sizeof(Ending);
    return bytes / 8 <= 0x7fffffffL ? (int)(bytes / 8) : 0;
}

extern "C" int ri_verify_drafts(int32_t* accepted, int32_t* out, const float* logits, const float* draft_logits, const int32_t* tokens,
                                const int32_t* cu_seqlens, const float* uniform, void* workspace, int seqs, int rows, int vocab,
                                double temperature, void* stream) {
    RI_REQUIRE(seqs >= 1 && rows >= 1 && vocab >= 1, "verify_drafts: %d sequences, %d rows, a vocabulary of %d", seqs, rows, vocab);
    RI_REQUIRE(rows <= 65535 && seqs <= 65535, "verify_drafts: %d rows of %d sequences, at most 65535 go in one call", rows, seqs);
    RI_REQUIRE(ri_verify_drafts_workspace_words(seqs, rows, vocab, draft_logits != nullptr) > 0,
               "verify_drafts: %d rows of a vocabulary of %d are too much for one call", rows, vocab);
    RI_REQUIRE(accepted && out && logits && tokens && cu_seqlens && workspace, "verify_drafts: an operand is missing");
    RI_REQUIRE(temperature < INFINITY, "verify_drafts: the temperature is no finite number");      // (nor is NaN)
    const hipStream_t s = (hipStream_t)stream;
    const int chunks = verify_chunks(vocab);
    const bool wide = vocab % 4 == 0 && (uintptr_t)logits % 16 == 0 && (uintptr_t)draft_logits % 16 == 0;
    if (temperature <= 0.0) {
        Best* bests = (Best*)workspace;
        const dim3 grid(chunks, rows);
        if (wide) verify_best<true><<<grid, VER_THREADS, 0, s>>>(bests, logits, vocab, chunks);
        else verify_best<false><<<grid, VER_THREADS, 0, s>>>(bests, logits, vocab, chunks);
        verify_walk<<<seqs, VER_THREADS, 0, s>>>(accepted, out, bests, tokens, cu_seqlens, seqs, rows, chunks);
        RI_LAUNCH_CHECK("verify_drafts");
        return 0;
    }
    RI_REQUIRE(uniform, "verify_drafts: a temperature above 0 wants the random numbers");
    ChunkStats* stats = (ChunkStats*)workspace;
    Weights* masses = (Weights*)(stats + (draft_logits ? 2L : 1L) * rows * chunks);
    Ending* endings = (Ending*)(masses + (long)seqs * chunks);
    const double by = fmin(1.4426950408889634074 / temperature, 1e200);       // (a difference of logits times it stays finite)
    const Scale scale = {by, 1.0 / by};
    const dim3 grid(chunks, rows, draft_logits ? 2 : 1), grid2(chunks, seqs);
    if (wide) verify_stats<true><<<grid, RI_WAVE, 0, s>>>(stats, logits, draft_logits, cu_seqlens, seqs, rows, vocab, chunks, scale);
    else verify_stats<false><<<grid, RI_WAVE, 0, s>>>(stats, logits, draft_logits, cu_seqlens, seqs, rows, vocab, chunks, scale);
#define VERIFY_WEIGH(WIDE, ENDS)                                                                                              \
    verify_weigh<WIDE, ENDS><<<grid2, VER_THREADS, 0, s>>>(masses, endings, stats, logits, draft_logits, tokens, cu_seqlens, uniform, \
                                                           rows, vocab, chunks, scale)
    // Few chunks: a launch less (one sequence of 5 rows x 151,936: 23 us, with `end` 26; 64 of them: 113 and 109).
    if ((long)chunks * seqs <= 2L * ri_compute_units()) {
        if (wide) VERIFY_WEIGH(true, true);
        else VERIFY_WEIGH(false, true);
    } else {
        verify_end<<<seqs, VER_THREADS, 0, s>>>(endings, stats, logits, draft_logits, tokens, cu_seqlens, uniform, rows, vocab, chunks, scale);
        if (wide) VERIFY_WEIGH(true, false);
        else VERIFY_WEIGH(false, false);
    }
#undef VERIFY_WEIGH
    verify_pick<<<seqs, VER_PICK_THREADS, 0, s>>>(accepted, out, masses, endings, logits, draft_logits, tokens, cu_seqlens, uniform, seqs,
                                                  rows, vocab, chunks, scale);
    RI_LAUNCH_CHECK("verify_drafts");
    return 0;
}
