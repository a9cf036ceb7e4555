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
// Everything that is compared is held in 64 bits: a token is the answer to "on which side of a border does u lie", a
// vocabulary has 10^5 borders, and float32 weights put one draw in 10^3 to 10^5 on the wrong side.  The vector unit takes
// float64 at the rate of float32, so it is the polynomial of exp2_nonpositive, 17 instructions an entry, that stands beside
// the 4 bytes of it.
//
// Three launches.  `stats` cuts every row that is asked about into chunks of 4,096 entries, a workgroup each, and leaves a
// chunk's largest logit and its sum of exponentials: the one pass over the logits.  `weigh` (a workgroup a chunk of the
// vocabulary and sequence) joins the rows' chunks in order until a draft falls, which every workgroup of a sequence does
// for itself (a few kilobytes), and sums its chunk of the row that the last token is drawn from.  `pick` (a workgroup a
// sequence) finds the chunk and in it the token.  Greedy steps need two: the chunks' best entries, then the walk.
// Every sum has one order, so the same inputs give the same tokens.
#include <float.h>

#include "api.h"
#include "common.h"

#define VER_CHUNK 4096
#define VER_THREADS 256
#define VER_WAVES (VER_THREADS / RI_WAVE)
#define VER_EACH (VER_CHUNK / VER_THREADS)
#define VER_PICK_THREADS 1024
#define VER_PICK_EACH (VER_CHUNK / VER_PICK_THREADS)

struct ChunkStats { double top, sum; };          // of a chunk of a row: its largest logit, the sum of exp((x - top) / T)
struct RowStats { double top, inv; };            // of a row: its largest logit, 1 / the sum (0 where every entry is masked)
// Where a sequence's walk ended: the row that the last token is drawn from, the draft that fell there (-1: none did, or it
// has a distribution of its own), and the statistics of both distributions.
struct Ending {
    RowStats p, q;
    int row, less, fell, unused;
};

// 2^t for t <= 0 (t NaN: 0), relative error under 3e-13: t = n + f with |f| <= 1/2, the Taylor sum of e^(f ln 2) up to the
// tenth power (the next term is 0.3466^11 / 11! = 2.2e-13), times 2^n.
__device__ __forceinline__ double exp2_nonpositive(double t) {
    t = fmax(t, -1100.0);
    const double n = rint(t), z = (t - n) * 0.69314718055994530942;
    double s = 1.0 / 3628800.0;
    s = fma(s, z, 1.0 / 362880.0);
    s = fma(s, z, 1.0 / 40320.0);
    s = fma(s, z, 1.0 / 5040.0);
    s = fma(s, z, 1.0 / 720.0);
    s = fma(s, z, 1.0 / 120.0);
    s = fma(s, z, 1.0 / 24.0);
    s = fma(s, z, 1.0 / 6.0);
    s = fma(s, z, 0.5);
    s = fma(s, z, 1.0);
    s = fma(s, z, 1.0);
    return ldexp(s, (int)n);
}

// A logit as the sampled forms take it: NaN is a masked entry, an infinite one the largest finite number.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

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
template <bool WIDE>
__device__ __forceinline__ void load_chunk(float (&v)[VER_EACH], const float* __restrict__ x, int n) {
    if (WIDE) {
#pragma unroll
        for (int u = 0; u < VER_EACH / 4; ++u) {
            const int i = 4 * (u * VER_THREADS + threadIdx.x);
            const float4 w = *reinterpret_cast<const float4*>(x + min(i, n - 4));
            v[4 * u] = i < n ? w.x : -INFINITY;
            v[4 * u + 1] = i < n ? w.y : -INFINITY;
            v[4 * u + 2] = i < n ? w.z : -INFINITY;
            v[4 * u + 3] = i < n ? w.w : -INFINITY;
        }
    } else {
#pragma unroll
        for (int u = 0; u < VER_EACH; ++u) {
            const int i = u * VER_THREADS + threadIdx.x;
            const float w = x[min(i, n - 1)];
            v[u] = i < n ? w : -INFINITY;
        }
    }
}
// The place in its chunk of a thread's entry e.
template <bool WIDE>
__device__ __forceinline__ int place_of(int e) {
    return WIDE ? 4 * ((e / 4) * VER_THREADS + threadIdx.x) + e % 4 : e * VER_THREADS + threadIdx.x;
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

template <bool WIDE>
__global__ __launch_bounds__(VER_THREADS) void verify_stats(ChunkStats* __restrict__ stats, const float* __restrict__ logits,
                                                            const float* __restrict__ draft, const int32_t* __restrict__ cu,
                                                            int seqs, int rows, int vocab, int chunks, double scale) {
    const int chunk = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & (RI_WAVE - 1), wave = threadIdx.x / RI_WAVE;
    const bool of_draft = blockIdx.z == 1;
    __shared__ double shared[2 * VER_WAVES];
    const int at = chunk * VER_CHUNK, n = min(VER_CHUNK, vocab - at);
    float v[VER_EACH];
    load_chunk<WIDE>(v, (of_draft ? draft : logits) + (size_t)row * vocab + at, n);
    bool within, drafted;
    place_of_row(cu, seqs, rows, row, within, drafted);
    if (of_draft ? !drafted : !within) return;                // the whole workgroup: nobody asks about this row
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < VER_EACH; ++e) {
        v[e] = clean(v[e]);
        top = fmaxf(top, v[e]);
    }
    top = wave_max(top);
    if (lane == 0) shared[wave] = top;
    __syncthreads();
    double m = shared[0];
#pragma unroll
    for (int w = 1; w < VER_WAVES; ++w) m = fmax(m, shared[w]);
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < VER_EACH; ++e) sum += exp2_nonpositive(((double)v[e] - m) * scale);
    sum = wave_sum_d(sum);
    if (lane == 0) shared[VER_WAVES + wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = shared[VER_WAVES];
#pragma unroll
        for (int w = 1; w < VER_WAVES; ++w) s += shared[VER_WAVES + w];
        stats[((size_t)blockIdx.z * rows + row) * chunks + chunk] = {m, s};
    }
}

// A row's chunks joined, by a wavefront, in an order that the number of chunks alone decides.
__device__ __forceinline__ RowStats join_row(const ChunkStats* __restrict__ c, int chunks, double scale) {
    const int lane = threadIdx.x & (RI_WAVE - 1);
    double m = -INFINITY;
    for (int i = lane; i < chunks; i += RI_WAVE) m = fmax(m, c[i].top);
    m = wave_max_d(m);
    double s = 0.0;
    for (int i = lane; i < chunks; i += RI_WAVE) s += c[i].sum * exp2_nonpositive((c[i].top - m) * scale);
    s = wave_sum_d(s);
    return {m, s > 0.0 ? 1.0 / s : 0.0};
}

__device__ __forceinline__ double probability(const RowStats s, float x, double scale) {
    return exp2_nonpositive(((double)clean(x) - s.top) * scale) * s.inv;
}

// What an entry weighs in the last draw: first in the distribution that is left, second in p itself (taken where nothing is
// left, as when p and q are equal up to their rounding).
struct Weights { double left, whole; };
__device__ __forceinline__ Weights weigh_entry(const Ending& e, float x, float qx, bool has_q, int id, double scale) {
    const double p = probability(e.p, x, scale);
    double left = p;
    if (e.fell) left = has_q ? fmax(p - probability(e.q, qx, scale), 0.0) : id == e.less ? 0.0 : p;
    return {left, p};
}

template <bool WIDE>
__global__ __launch_bounds__(VER_THREADS) void verify_weigh(Weights* __restrict__ masses, Ending* __restrict__ endings,
                                                            const ChunkStats* __restrict__ stats, const float* __restrict__ logits,
                                                            const float* __restrict__ draft, const int32_t* __restrict__ tokens,
                                                            const int32_t* __restrict__ cu, const float* __restrict__ uniform,
                                                            int rows, int vocab, int chunks, double scale) {
    const int chunk = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & (RI_WAVE - 1), wave = threadIdx.x / RI_WAVE;
    __shared__ Ending tried[VER_WAVES];
    __shared__ Weights sums[VER_WAVES];
    int r0, r1;
    rows_of(cu, b, rows, r0, r1);
    if (r0 == r1) return;
    // four rows at a time, a wavefront each, until one ends the walk; the last row always does
    Ending end;
    for (int base = r0;; base += VER_WAVES) {
        const int row = base + wave;
        Ending mine = {{0.0, 0.0}, {0.0, 0.0}, -1, -1, 0, 0};
        if (row < r1) {
            mine.p = join_row(stats + (size_t)row * chunks, chunks, scale);
            if (row == r1 - 1) {
                mine.row = row;
            } else {
                const int d = tokens[row + 1];
                const bool known = d >= 0 && d < vocab;       // a draft that is no token of the vocabulary falls
                double q = 1.0;
                if (draft) {
                    mine.q = join_row(stats + ((size_t)rows + row + 1) * chunks, chunks, scale);
                    q = known ? probability(mine.q, draft[(size_t)(row + 1) * vocab + d], scale) : 0.0;
                }
                const double p = known ? probability(mine.p, logits[(size_t)row * vocab + d], scale) : 0.0;
                if (!((double)uniform[row] * q < p)) {
                    mine.row = row;
                    mine.less = d;
                    mine.fell = 1;
                }
            }
        }
        if (lane == 0) tried[wave] = mine;
        __syncthreads();
        int first = -1;
        for (int w = VER_WAVES - 1; w >= 0; --w)
            if (tried[w].row >= 0) first = w;
        if (first >= 0) {
            end = tried[first];
            break;
        }
        __syncthreads();
    }
    if (chunk == 0 && threadIdx.x == 0) endings[b] = end;
    const int at = chunk * VER_CHUNK, n = min(VER_CHUNK, vocab - at);
    const bool has_q = draft != nullptr;
    float x[VER_EACH], qx[VER_EACH];
    load_chunk<WIDE>(x, logits + (size_t)end.row * vocab + at, n);
    if (has_q && end.fell) load_chunk<WIDE>(qx, draft + (size_t)(end.row + 1) * vocab + at, n);
    Weights sum = {0.0, 0.0};
#pragma unroll
    for (int e = 0; e < VER_EACH; ++e) {
        const Weights w = weigh_entry(end, x[e], qx[e], has_q, at + place_of<WIDE>(e), scale);
        sum.left += w.left;
        sum.whole += w.whole;
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

__global__ __launch_bounds__(VER_PICK_THREADS) void verify_pick(int32_t* __restrict__ accepted, int32_t* __restrict__ out,
                                                                const Weights* __restrict__ masses, const Ending* __restrict__ endings,
                                                                const float* __restrict__ logits, const float* __restrict__ draft,
                                                                const int32_t* __restrict__ tokens, const int32_t* __restrict__ cu,
                                                                const float* __restrict__ uniform, int seqs, int rows, int vocab,
                                                                int chunks, double scale) {
    const int b = blockIdx.x, lane = threadIdx.x & (RI_WAVE - 1), wave = threadIdx.x / RI_WAVE;
    __shared__ double upto_wave[VER_PICK_THREADS / RI_WAVE];
    __shared__ double before_chunk;
    __shared__ int chosen, whole, found, last_some;
    int r0, r1;
    rows_of(cu, b, rows, r0, r1);
    if (r0 == r1) {
        put_out(accepted, out, tokens, cu, seqs, rows, b, r0, r1, r0, -1);
        return;
    }
    const Ending end = endings[b];
    const Weights* mine = masses + (size_t)b * chunks;
    const double u = uniform[r1 - 1];
    if (threadIdx.x == 0) {
        double left = 0.0, all = 0.0;
        for (int c = 0; c < chunks; ++c) {
            left += mine[c].left;
            all += mine[c].whole;
        }
        const int take_all = !(left > 0.0);
        const double target = u * (take_all ? all : left);
        double upto = 0.0, before = 0.0, before_some = 0.0;
        int at = -1, some = 0;
        for (int c = 0; c < chunks; ++c) {
            const double w = take_all ? mine[c].whole : mine[c].left;
            if (w > 0.0) {
                some = c;
                before_some = upto;
            }
            upto += w;
            if (upto > target) {
                at = c;
                before = before_some;
                break;
            }
        }
        chosen = at < 0 ? some : at;                          // (nothing passes: u is not below 1)
        before_chunk = at < 0 ? before_some : before;
        whole = take_all;
        found = VER_CHUNK;
        last_some = -1;
        upto_wave[0] = target;
    }
    __syncthreads();
    const double target = upto_wave[0];
    const int at = chosen * VER_CHUNK, n = min(VER_CHUNK, vocab - at), first = threadIdx.x * VER_PICK_EACH;
    const bool has_q = draft != nullptr;
    double w[VER_PICK_EACH], sum = 0.0;
#pragma unroll
    for (int e = 0; e < VER_PICK_EACH; ++e) {
        const int i = first + e, id = at + min(i, n - 1);
        const float x = logits[(size_t)end.row * vocab + id];
        const float qx = has_q && end.fell ? draft[(size_t)(end.row + 1) * vocab + id] : 0.f;
        const Weights ws = weigh_entry(end, x, qx, has_q, id, scale);
        w[e] = i < n ? (whole ? ws.whole : ws.left) : 0.0;
        sum += w[e];
    }
    double upto = sum;                                        // of the lanes up to this one
#pragma unroll
    for (int d = 1; d < RI_WAVE; d *= 2) {
        const double o = __shfl(upto, max(lane - d, 0), RI_WAVE);
        upto += lane >= d ? o : 0.0;
    }
    __syncthreads();                                          // everybody has read the target
    if (lane == RI_WAVE - 1) upto_wave[wave] = upto;
    __syncthreads();
    double before = before_chunk;
    for (int v = 0; v < wave; ++v) before += upto_wave[v];
    double run = before + (upto - sum);
#pragma unroll
    for (int e = 0; e < VER_PICK_EACH; ++e) {
        run += w[e];
        if (w[e] > 0.0) atomicMax(&last_some, first + e);     // (whole numbers: the order of the lanes changes nothing)
        if (w[e] > 0.0 && run > target) {
            atomicMax(&found, VER_CHUNK * 2 - (first + e));   // the first such place, counted from behind
            break;
        }
    }
    __syncthreads();
    // (the chunk's sum and its entries' running sum are added up in another order: a target within their rounding of the
    // chunk's end falls to its last entry that weighs anything)
    const int place = found > VER_CHUNK ? VER_CHUNK * 2 - found : max(last_some, 0);
    put_out(accepted, out, tokens, cu, seqs, rows, b, r0, r1, end.row, at + place);
}

// ---- greedy: the best entry of every chunk, then the walk
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
    float v[VER_EACH];
    load_chunk<WIDE>(v, logits + (size_t)row * vocab + at, n);
    Best best = {-INFINITY, at};                              // (a chunk of masked entries names its first)
#pragma unroll
    for (int e = 0; e < VER_EACH; ++e)
        if (v[e] > best.value) best = {v[e], at + place_of<WIDE>(e)};      // (by rising place; NaN is above nothing)
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
            if (row == r1 - 1 || tokens[row + 1] != best.id) ends = best.id;
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

extern "C" long ri_verify_drafts_workspace_bytes(int seqs, int rows, int vocab) {
    if (seqs < 1 || rows < 1 || vocab < 1) return 0;
    const long chunks = verify_chunks(vocab);
    return 2L * rows * chunks * (long)sizeof(ChunkStats) + seqs * chunks * (long)sizeof(Weights) + seqs * (long)sizeof(Ending);
}

extern "C" int ri_verify_drafts(int32_t* accepted, int32_t* out, const float* logits, const float* draft_logits, const int32_t* tokens,
                                const int32_t* cu_seqlens, const float* uniform, void* workspace, int seqs, int rows, int vocab,
                                double temperature, void* stream) {
    RI_REQUIRE(seqs >= 1 && rows >= 1 && vocab >= 1, "verify_drafts: %d sequences, %d rows, a vocabulary of %d", seqs, rows, vocab);
    RI_REQUIRE(rows <= 65535 && seqs <= 65535, "verify_drafts: %d rows of %d sequences, at most 65535 go in one call", rows, seqs);
    RI_REQUIRE(vocab <= 0x7fffffff - VER_CHUNK, "verify_drafts: a vocabulary of %d is too large", vocab);
    RI_REQUIRE(accepted && out && logits && tokens && cu_seqlens && workspace, "verify_drafts: an operand is missing");
    RI_REQUIRE(temperature == temperature, "verify_drafts: the temperature is no number");
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
    Weights* masses = (Weights*)(stats + 2L * rows * chunks);
    Ending* endings = (Ending*)(masses + (long)seqs * chunks);
    const double scale = fmin(1.4426950408889634074 / temperature, 1e300);       // (finite: 0 times it is 0)
    const dim3 grid(chunks, rows, draft_logits ? 2 : 1), grid2(chunks, seqs);
    if (wide) {
        verify_stats<true><<<grid, VER_THREADS, 0, s>>>(stats, logits, draft_logits, cu_seqlens, seqs, rows, vocab, chunks, scale);
        verify_weigh<true><<<grid2, VER_THREADS, 0, s>>>(masses, endings, stats, logits, draft_logits, tokens, cu_seqlens, uniform, rows,
                                                         vocab, chunks, scale);
    } else {
        verify_stats<false><<<grid, VER_THREADS, 0, s>>>(stats, logits, draft_logits, cu_seqlens, seqs, rows, vocab, chunks, scale);
        verify_weigh<false><<<grid2, VER_THREADS, 0, s>>>(masses, endings, stats, logits, draft_logits, tokens, cu_seqlens, uniform, rows,
                                                          vocab, chunks, scale);
    }
    verify_pick<<<seqs, VER_PICK_THREADS, 0, s>>>(accepted, out, masses, endings, logits, draft_logits, tokens, cu_seqlens, uniform, seqs,
                                                  rows, vocab, chunks, scale);
    RI_LAUNCH_CHECK("verify_drafts");
    return 0;
}
