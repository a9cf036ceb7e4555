// Attention of new tokens whose sequences begin with the same pages: bfloat16, pages of 32 tokens, heads of 32, 64 and 128.
//
// A batch behind one long prompt reads that prompt's keys and values once a sequence in the ordinary decode attention.
// Here the queries of all tokens are columns of one product over the shared pages: column r of a key head is query head
// r % group of token r / group, as in attention_mfma.h, whose page of arithmetic this is (scores, running maximum and
// sum, weighted values).  What a token sees beyond the shared pages is its own sequence's, by position.
//
// A workgroup takes a tile of columns over a run of pages and leaves, for every column, the largest score m, the sum l of
// exp2(s - m) and the sum of exp2(s - m) v; the shared pages are cut into runs, every sequence's own pages into chunks, and
// a second kernel joins a token's runs and chunks in order:
//     out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i,  M the largest m_i.
// Statistics and sums are float32; the weights enter the second product rounded to bfloat16, as the matrix cores take it and as in the
// other attentions here (products of float32 weights would be eight times the instructions); l is taken before the rounding.  A weight is
// off by 2^-8 of itself at most, one way or the other, so that most of it goes out in the sum: a result's distance from 64 bits grows from
// 0.0017 of it, its own rounding, to 0.0019 to 0.0021.
//
// Keys and values behind a sequence's largest position, or from max_len on, are whatever the page held before: they are taken as zeros, so
// that an infinity or NaN there reaches nothing.
#include <float.h>

#include "attention_mfma.h"

#define SH_OWN_PAGES 16          // pages of a chunk of a sequence's own keys: this many, or half where that leaves compute units empty

struct SharedArgs {
    float* sums;                 // [slots][tokens][heads][dim]
    float2* stats;               // [slots][tokens][heads]: m and l
    const bf16_t* q;
    const bf16_t* k_pages;
    const bf16_t* v_pages;
    const int32_t* cu_seqlens;
    const int32_t* tok_pos;
    const int32_t* page_table;
    int q_stride, table_width, num_pages, tokens, seqs, heads, kv_heads, shared_pages;
    int max_len;                 // of any sequence: keys from there on are not seen
    int splits, pages_per_split, tiles, own_tiles, own_chunks, own_pages;
    float scale_log2;
};

// Key rows, and value columns, behind the last key (counted from the page's first) as zeros.
template <int DH>
__device__ __forceinline__ void drop_keys(Frag (&kf)[2][DH / 32], int last, int lane) {
    const int i = lane & 15;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
        if ((i >> 2) * 8 + kt * 4 + (i & 3) > last) {
#pragma unroll
            for (int ks = 0; ks < DH / 32; ++ks) kf[kt][ks].u = make_uint4(0, 0, 0, 0);
        }
}
template <int DH>
__device__ __forceinline__ void drop_values(Frag (&vf)[DH / 16], int last, int lane) {
    const int jg = lane >> 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int key = jg * 8 + 2 * e;
        const uint32_t mask = key > last ? 0u : key + 1 > last ? 0x0000FFFFu : 0xFFFFFFFFu;
#pragma unroll
        for (int dt = 0; dt < DH / 16; ++dt) vf[dt].w[e] &= mask;
    }
}

// W: wavefronts of a workgroup; SLOTS: pairs of pages of keys, and of values, that LDS holds (0: none, few columns only).
template <int DH, int W, int SLOTS>
struct SharedLds {
    static constexpr int LD = DH + 4;                        // a column's stride, floats
    union {
        struct { bf16_t k[SLOTS ? SLOTS : 1][2][SLOTS ? PAGE * DH : 1], v[SLOTS ? SLOTS : 1][2][SLOTS ? PAGE * DH : 1]; } pages;
        struct { float o[W][16 * LD], m[W][16], l[W][16]; } meet;
    };
};

// Column `col` of the tokens first_token ..: its token and query head.
struct Place { int token, head; };
__device__ __forceinline__ Place place_of(const SharedArgs& a, int first_token, int kvh, int col) {
    const int group = a.heads / a.kv_heads, t = col / group;
    return {first_token + t, kvh * group + col - t * group};
}
__device__ __forceinline__ size_t result_at(const SharedArgs& a, int slot, Place p) {
    return ((size_t)slot * a.tokens + p.token) * a.heads + p.head;
}

// Where the first 64 pages from page0 on that a wavefront takes lie, a lane each (behind the last page there may be: the last).
template <int W>
__device__ __forceinline__ int first_ids(const int32_t* table, int page0, int pages) {
    return table[min(page0 + (int)(threadIdx.x >> 6) + (int)(threadIdx.x & 63) * W, pages - 1)];
}

// Few columns: a tile of 16 NT over the pages page0 .. page1, which the wavefronts take in turn; they meet in LDS.  Bound by memory
// (own keys of 64 sequences, 204 MB: 39 us, 5.2 TB/s), a short chunk by its chain of loads: place, keys, values.
template <int DH, int NT, int W, int SLOTS>
__device__ __forceinline__ void few_columns(const SharedArgs& a, SharedLds<DH, W, SLOTS>& lds, const int32_t* table, int kvh, int slot,
                                            int first_token, int col0, int cols, int page0, int page1, int last_key, int ids, int thread) {
    constexpr int LD = SharedLds<DH, W, SLOTS>::LD;
    const int lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6), i = lane & 15, jg = lane >> 4;
    Columns<DH, NT> c;
    init_columns<DH, NT>(c);
    Place place[NT];
    int min_qpos = last_key;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        place[n] = place_of(a, first_token, kvh, min(col0 + 16 * n + i, cols - 1));
        c.qpos[n] = min(a.tok_pos[place[n].token], last_key);
        min_qpos = min(min_qpos, c.qpos[n]);
        const bf16_t* q = a.q + (size_t)place[n].token * a.q_stride + place[n].head * DH + jg * 8;
#pragma unroll
        for (int ks = 0; ks < DH / 32; ++ks) c.q[n][ks].u = *reinterpret_cast<const uint4*>(q + 32 * ks);
    }
    // The next page's keys are asked for when this one's are used up, its values likewise: a page is on its way all the time.
    // (Behind the last page: a line of it.)
    Frag kf[2][DH / 32], vf[DH / 16];
    // A lane holds the place of one of the wavefront's next 64 pages (the caller has the first 64): a load a page would stand behind
    // the values in the queue.
    int held = 0;
    auto phys_of = [&](int page) -> long {
        const int at = (page - page0) / W;
        if (at >> 6 != held) {
            held = at >> 6;
            ids = table[min(page0 + wave + (64 * held + lane) * W, page1 - 1)];
            ma_here(ids);
        }
        return min(max(__builtin_amdgcn_readlane(ids, at & 63), 0), a.num_pages - 1);
    };
    auto load_keys = [&](long phys, bool wanted) {
        const int w = wanted ? 1 : 0, r = i * w, g = jg * w;
        const bf16_t* from = a.k_pages + (phys * a.kv_heads + kvh) * (long)(PAGE * DH);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int ks = 0; ks < DH / 32; ++ks)
                // (not marked as read once: a load takes 64 bytes of each of 16 rows, the next one the other half of those lines; marked,
                // 64 sequences' own keys took 47 us, so 39)
                kf[kt][ks].u = *reinterpret_cast<const uint4*>(from + ((r >> 2) * 8 + (kt * 4 + (r & 3)) * w) * DH + (ks * 32) * w + g * 8);
    };
    auto load_values = [&](long phys, bool wanted) {
        const int w = wanted ? 1 : 0, r = i * w, g = jg * w;
        const bf16_t* from = a.v_pages + (phys * a.kv_heads + kvh) * (long)(PAGE * DH);
#pragma unroll
        for (int dt = 0; dt < DH / 16; ++dt) vf[dt].u = load_stream16(from + (dt * 16 * w + r) * PAGE + g * 8);
    };
    int page = page0 + wave;
    if (page < page1) {
        {
            const long phys = phys_of(page);
            load_keys(phys, true);
            load_values(phys, true);
        }
        for (; page < page1; page += W) {
            const int last = last_key - page * PAGE;
            const bool more = page + W < page1;
            Frag p[NT];
            if (last < PAGE - 1) drop_keys<DH>(kf, last, lane);
            scores_and_weights<DH, NT>(c, kf, p, page, lane, a.scale_log2, !__any(min_qpos < page * PAGE + PAGE - 1));
            const long next = phys_of(page + W);
            load_keys(next, more);
            if (last < PAGE - 1) drop_values<DH>(vf, last, lane);
            weighted_values<DH, NT>(c, vf, p);
            load_values(next, more);
        }
    }
    finish_columns<DH, NT>(c);
    auto& meet = lds.meet;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (jg == 0) {
            meet.m[wave][i] = c.m[n];
            meet.l[wave][i] = c.l[n];
        }
        __syncthreads();
        float m = meet.m[0][i], l = 0.f;
#pragma unroll
        for (int w = 1; w < W; ++w) m = fmaxf(m, meet.m[w][i]);
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int w = 0; w < W; ++w) l += __builtin_amdgcn_exp2f(meet.m[w][i] - ref) * meet.l[w][i];
        const float mine = __builtin_amdgcn_exp2f(c.m[n] - ref);
#pragma unroll
        for (int dt = 0; dt < DH / 16; ++dt)
            *reinterpret_cast<float4*>(&meet.o[wave][i * LD + dt * 16 + jg * 4]) =
                make_float4(c.o[n][dt][0] * mine, c.o[n][dt][1] * mine, c.o[n][dt][2] * mine, c.o[n][dt][3] * mine);
        if (wave == 0 && jg == 0 && col0 + 16 * n + i < cols) a.stats[result_at(a, slot, place[n])] = make_float2(m, l);
        __syncthreads();
        for (int at = thread; at < 16 * DH / 4; at += W * 64) {
            const int r = at / (DH / 4), d = at % (DH / 4) * 4, col = col0 + 16 * n + r;
            if (col >= cols) break;
            float4 o = *reinterpret_cast<const float4*>(&meet.o[0][r * LD + d]);
#pragma unroll
            for (int w = 1; w < W; ++w) {
                const float4 more = *reinterpret_cast<const float4*>(&meet.o[w][r * LD + d]);
                o = make_float4(o.x + more.x, o.y + more.y, o.z + more.z, o.w + more.w);
            }
            *reinterpret_cast<float4*>(a.sums + result_at(a, slot, place_of(a, first_token, kvh, col)) * DH + d) = o;
        }
        if (n + 1 < NT) __syncthreads();                      // (the next sixteen meet in the same place)
    }
}

// Many columns: a wavefront takes 16 NT of them and walks all pages page0 .. page1, two at a time (a pair that ends behind page1 takes
// its last page twice, the second time masked); the pages are copied into LDS once for all wavefronts, one place a turn where they
// meet.  SLOTS - 1 turns hide a copy's way from memory.  Bound by what it issues, products and exponentials in turn (256 columns a key
// head over 131,072 keys of 8 heads of 128: 187 to 193 us, 0.72 PFLOP/s; products and exponentials alone 110 to 150, copies 115).
template <int DH, int NT, int W, int SLOTS>
__device__ __forceinline__ void many_columns(const SharedArgs& a, SharedLds<DH, W, SLOTS>& lds, int kvh, int slot, int col0, int cols, int page0, int page1) {
    typedef CopiedPage<DH> Copied;
    constexpr int HALVES = 8 / W, MINE = HALVES * Copied::MINE;         // half pages, and copies, of a wavefront for a pair
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, jg = lane >> 4;
    const int last_key = min(page1 * PAGE, a.max_len) - 1, u_last = (page1 - page0 - 1) / 2;
    auto& k_lds = lds.pages.k;
    auto& v_lds = lds.pages.v;
    int ids = a.page_table[min(page0 + lane, page1 - 1)];
    Columns<DH, NT> c;
    init_columns<DH, NT>(c);
    int min_qpos = last_key;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int col = min(col0 + (wave * NT + j) * 16 + i, cols - 1);         // (columns behind the last repeat it and are not stored)
        const Place p = place_of(a, 0, kvh, col);
        c.qpos[j] = min(a.tok_pos[p.token], last_key);
        min_qpos = min(min_qpos, c.qpos[j]);
        const bf16_t* q = a.q + (size_t)p.token * a.q_stride + p.head * DH + jg * 8;
#pragma unroll
        for (int ks = 0; ks < DH / 32; ++ks) c.q[j][ks].u = *reinterpret_cast<const uint4*>(q + 32 * ks);
    }
    const bool all_seen = !__any(min_qpos < page1 * PAGE - 1);
    // the queries are here before the first copy starts: a wait for them behind it would be one for all copies
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int ks = 0; ks < DH / 32; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) ma_here(c.q[j][ks].w[e]);
    auto page_of = [&](int u) { return page0 + 2 * u; };
    auto open = [&](int u) { return all_seen && page_of(u) + 1 < page1; };
    // The first half of the wavefronts copies keys, the other values: the same halves of one page, or of both, in every turn.
    const bool of_values = wave >= W / 2;
    uint32_t off[Copied::MINE];
    Copied::offsets(off, (of_values ? 2 : 0) + (wave & 1), lane);
    const bf16_t* pages = of_values ? a.v_pages : a.k_pages;
    // Where the pages lie: a lane holds the place of one of 64 neighbouring pages.  (A load a turn would be counted among the copies
    // under way; this one is waited for where it is made, once in 32 turns.)
    int held = 0;
    auto look = [&](int u, int n) -> int {                   // of the n-th page that this wavefront copies of pair u (behind the last: of it)
        const int at = min(2 * min(u, u_last) + (HALVES == 2 ? n : wave >> 1 & 1), page1 - page0 - 1);
        if (at >> 6 != held) {
            held = at >> 6;
            ids = a.page_table[min(page0 + 64 * held + lane, page1 - 1)];
            ma_here(ids);
        }
        return min(max(__builtin_amdgcn_readlane(ids, at & 63), 0), a.num_pages - 1);
    };
    auto fetch = [&](int u, const int (&at)[HALVES]) {
#pragma unroll
        for (int n = 0; n < HALVES; ++n) {
            const int h = HALVES == 2 ? n : wave >> 1 & 1;
            const ma_lds_t to = of_values ? ma_lds(v_lds[(unsigned)u % SLOTS][h]) : ma_lds(k_lds[(unsigned)u % SLOTS][h]);
            Copied::copy(to, off, pages + ((long)at[n] * a.kv_heads + kvh) * (PAGE * DH), wave & 1);
        }
    };
    auto scores = [&](float (&s)[NT][2][8], int u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            Frag kf[2][DH / 32];
            Copied::keys(kf, k_lds[(unsigned)u % SLOTS][h], lane);
            float one[NT][8];
            scores_of<DH, NT>(c, kf, one, 0, lane);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[j][h][e] = one[j][e];
        }
    };
    auto mask = [&](float (&s)[NT][2][8], int u) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if ((page_of(u) + e / 8) * PAGE + jg * 8 + e % 8 > c.qpos[j]) s[j][e / 8][e % 8] = -INFINITY;
    };
    auto maxima = [&](const float (&s)[NT][2][8], float (&m_new)[NT]) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float mx = s[j][0][0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[j][e / 8][e % 8]);
            m_new[j] = fmaxf(c.m[j], column_max<(NT >= 2 || DH < 128)>(mx) * a.scale_log2);
        }
    };
    float s_cur[NT][2][8], ref[NT], m_new[NT];
    const int ahead = of_values ? SLOTS - 1 : SLOTS;         // turn u starts the copies of pair u + ahead
    int next[HALVES];
    for (int u = 0; u < ahead; ++u) {
#pragma unroll
        for (int n = 0; n < HALVES; ++n) next[n] = look(u, n);
        fetch(u, next);
    }
#pragma unroll
    for (int n = 0; n < HALVES; ++n) next[n] = look(ahead, n);
    ma_wait_copies<(SLOTS - 1) * MINE>();                     // the keys of pair 0 are there (the values: as many copies, one pair less)
    ma_meet();
    scores(s_cur, 0);
    if (!open(0)) mask(s_cur, 0);
    maxima(s_cur, m_new);
    move_reference<DH, NT>(c, m_new, ref);
    auto weights = [&](Frag (&w)[NT], int h) {
        float one[NT][8];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) one[j][e] = s_cur[j][h][e];
        weights_of<DH, NT>(c, one, ref, w, a.scale_log2);
    };
    auto values = [&](const Frag (&w)[NT], int u, int h) {
        Frag vf[DH / 16];
        Copied::values(vf, v_lds[(unsigned)u % SLOTS][h], lane);
        weighted_values<DH, NT>(c, vf, w);
    };
    auto turn = [&](int u, auto masked) {                    // u: the pair whose weights are due
        ma_wait_copies<(SLOTS - 2) * MINE>();                 // the keys of pair u + 1 and the values of pair u are there,
        ma_wait_lds();                                        // the keys of pair u and the values of pair u - 1 read
        ma_meet();
        fetch(u + ahead, next);
#pragma unroll
        for (int n = 0; n < HALVES; ++n) next[n] = look(u + ahead + 1, n);
        Frag w[2][NT];
        float s_next[NT][2][8];
        scores(s_next, u + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) weights(w[h], h);
        if (decltype(masked)::value) mask(s_next, u + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) values(w[h], u, h);
        maxima(s_next, m_new);
        move_reference<DH, NT>(c, m_new, ref);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) s_cur[j][e / 8][e % 8] = s_next[j][e / 8][e % 8];
    };
    int u = 0;
    for (; u < u_last && open(u + 1); ++u) turn(u, std::false_type());
    for (; u < u_last; ++u) turn(u, std::true_type());
    ma_wait_copies<0>();                                      // (also what was copied for nobody: it must not arrive in another workgroup's LDS)
    ma_meet();
#pragma unroll
    for (int h = 0; h < 2; ++h) {                            // the last pair's weights and value products
        Frag w[NT];
        weights(w, h);
        values(w, u_last, h);
    }
    finish_columns<DH, NT>(c);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int col = col0 + (wave * NT + j) * 16 + i;
        if (col >= cols) continue;
        const size_t at = result_at(a, slot, place_of(a, 0, kvh, col));
        if (jg == 0) a.stats[at] = make_float2(c.m[j], c.l[j]);
#pragma unroll
        for (int dt = 0; dt < DH / 16; ++dt)
            *reinterpret_cast<float4*>(a.sums + at * DH + dt * 16 + jg * 4) = make_float4(c.o[j][dt][0], c.o[j][dt][1], c.o[j][dt][2], c.o[j][dt][3]);
    }
}

// The largest position of a sequence's new tokens, which as a rule is the last one's; a lane a token.
__device__ __forceinline__ int last_position(const SharedArgs& a, int first, int behind) {
    int last = a.tok_pos[min(first + (int)(threadIdx.x & 63), behind - 1)];
    for (int at = first + 64; at < behind; at += 64) last = max(last, a.tok_pos[min(at + (int)(threadIdx.x & 63), behind - 1)]);
    for (int m = 1; m < min(behind - first, 64); m *= 2) last = max(last, __shfl_xor(last, m, 64));
    return __builtin_amdgcn_readfirstlane(last);
}

// A sequence's own chunk, by its number among all (key heads fastest, then tiles, chunks, sequences).
template <int DH, int NT, int W>
__device__ __forceinline__ void own_chunk(const SharedArgs& a, SharedLds<DH, W, 0>& lds, int item) {
    const int kvh = item % a.kv_heads;
    item /= a.kv_heads;
    const int seq = item / (a.own_tiles * a.own_chunks);
    item -= seq * a.own_tiles * a.own_chunks;
    const int chunk = item / a.own_tiles, tile = item - chunk * a.own_tiles, page0 = a.shared_pages + chunk * a.own_pages;
    const int32_t* table = a.page_table + (size_t)seq * a.table_width;
    // (asked for before the sequence's length is known: the loads of a chunk are a chain, and most of its time its first)
    const int ids = first_ids<W>(table, page0, a.table_width);
    const int first = min(max(a.cu_seqlens[seq], 0), a.tokens), behind = min(max(a.cu_seqlens[seq + 1], first), a.tokens);
    const int cols = (behind - first) * (a.heads / a.kv_heads);
    if (tile * 16 * NT >= cols) return;
    const int last_key = min(last_position(a, first, behind), a.max_len - 1);
    const int page1 = min(page0 + a.own_pages, last_key / PAGE + 1);
    if (page0 >= page1) return;
    // One tile, unless the sequence brings more tokens than max_new said.  (The compiler is not to know that a thread has the same number in
    // every turn: what it would keep from one to the next does not fit the registers.)
    for (int col0 = tile * 16 * NT; col0 < cols; col0 += a.own_tiles * 16 * NT) {
        int thread = threadIdx.x;
        ma_here(thread);
        few_columns<DH, NT>(a, lds, table, kvh, a.splits + chunk, first, col0, cols, page0, page1, last_key, ids, thread);
        __syncthreads();
    }
}

// Few columns in all: the runs of the shared pages and the sequences' own chunks, a workgroup each; with more (ALL false) the own
// chunks alone.
template <int DH, bool ALL, int NT, int W>
__global__ void __launch_bounds__(W * 64, NT == 1 ? 3 : 2) attn_shared_few_kernel(const SharedArgs a) {
    __shared__ __attribute__((aligned(16))) SharedLds<DH, W, 0> lds;
    const int of_tile = a.splits * a.kv_heads, shared_items = ALL ? of_tile * a.tiles : 0;
    int item = blockIdx.x;
    if (item >= shared_items) {
        own_chunk<DH, NT>(a, lds, item - shared_items);
        return;
    }
    const int tile = item / of_tile;
    item -= tile * of_tile;
    const int slot = item / a.kv_heads, kvh = item - slot * a.kv_heads, page0 = slot * a.pages_per_split;
    few_columns<DH, NT>(a, lds, a.page_table, kvh, slot, 0, tile * 16 * NT, a.tokens * (a.heads / a.kv_heads), page0,
                    min(page0 + a.pages_per_split, a.shared_pages), min(a.shared_pages * PAGE, a.max_len) - 1,
                    first_ids<W>(a.page_table, page0, a.shared_pages), threadIdx.x);
}

// The shared pages' runs for many columns; by rising number a tile after the other, so that tiles that read the same pages lie a multiple
// of eight apart and meet in one XCD's L2.
template <int DH, int NT, int W, int SLOTS>
__global__ void __launch_bounds__(W * 64, 2) attn_shared_kernel(const SharedArgs a) {
    __shared__ __attribute__((aligned(16))) SharedLds<DH, W, SLOTS> lds;
    const int of_tile = a.splits * a.kv_heads, tile = blockIdx.x / of_tile, item = blockIdx.x - tile * of_tile;
    const int slot = item / a.kv_heads, kvh = item - slot * a.kv_heads, page0 = slot * a.pages_per_split;
    many_columns<DH, NT>(a, lds, kvh, slot, tile * 16 * W * NT, a.tokens * (a.heads / a.kv_heads), page0,
                         min(page0 + a.pages_per_split, a.shared_pages));
}

// A token's runs and chunks joined, a workgroup a (head, token): DH / 4 neighbouring threads read a run's sums of it, 1,024 / DH
// such groups take the runs in turn and meet in LDS in their order (64 tokens x 32 heads of 128, 16 runs and up to 3 chunks: 6.2 us).
// Tokens that are no sequence's get zeros.
#define SH_JOIN 256
template <int DH>
__global__ void __launch_bounds__(SH_JOIN) attn_shared_join_kernel(bf16_t* __restrict__ out, const SharedArgs a) {
    constexpr int LANES = DH / 4, GROUPS = SH_JOIN / LANES;
    __shared__ __attribute__((aligned(16))) float4 sums[SH_JOIN];
    __shared__ float2 stats[GROUPS];
    const int head = blockIdx.x, token = blockIdx.y, lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const int first = a.cu_seqlens[0], behind = a.cu_seqlens[a.seqs];
    uint2* to = reinterpret_cast<uint2*>(out + ((size_t)token * a.heads + head) * DH) + lane;
    if (token < first || token >= behind) {
        if (group == 0) *to = uint2{0u, 0u};
        return;
    }
    const int own = min(a.tok_pos[token], a.max_len - 1) + 1 - a.shared_pages * PAGE;      // own keys that it sees
    const int chunks = own > 0 ? min((own + a.own_pages * PAGE - 1) / (a.own_pages * PAGE), a.own_chunks) : 0;
    const int slots = a.splits + chunks;
    const size_t at = (size_t)token * a.heads + head, step = (size_t)a.tokens * a.heads;
    // a group's runs, its own running maximum and sums
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = group; s < slots; s += GROUPS) {
        const float2 st = a.stats[s * step + at];
        const float4 v = *reinterpret_cast<const float4*>(a.sums + (s * step + at) * DH + 4 * lane);
        const float m_new = fmaxf(m, st.x), ref = m_new == -INFINITY ? 0.f : m_new;
        const float before = __builtin_amdgcn_exp2f(m - ref), now = __builtin_amdgcn_exp2f(st.x - ref);
        l = l * before + st.y * now;
        o = make_float4(o.x * before + v.x * now, o.y * before + v.y * now, o.z * before + v.z * now, o.w * before + v.w * now);
        m = m_new;
    }
    if (lane == 0) stats[group] = make_float2(m, l);
    sums[threadIdx.x] = o;
    __syncthreads();
    if (group > 0) return;
    m = -INFINITY;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) m = fmaxf(m, stats[g].x);
    const float ref = m == -INFINITY ? 0.f : m;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        const float w = __builtin_amdgcn_exp2f(stats[g].x - ref);
        const float4 v = sums[g * LANES + lane];
        l += w * stats[g].y;
        o = make_float4(o.x + w * v.x, o.y + w * v.y, o.z + w * v.z, o.w + w * v.w);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    *to = uint2{pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv)};
}

struct SharedPlan { int nt, few, waves, splits, pages_per_split, tiles, own_tiles, own_chunks, own_pages; };

// A sequence that brings more than 16 columns takes them 32 a workgroup, with fewer wavefronts a compute unit, so that its own keys are read
// half as often: 16 sequences of up to 5 tokens of 4 heads a key head, 20 to 900 own keys, 14.0 us (tiles of 16: 15.7).
// More than 32 columns a key head take the form of many columns: workgroups of four wavefronts with a tile of 64 or, from 65 columns on,
// 128; from 129 columns on, where a run is longer than SH_SHORT_PAGES, of eight with 256, whose copies
// have three turns to arrive instead of one.  us with four : eight wavefronts, up to 32 own keys: 32 sequences of 64 heads behind 131,072
// tokens (runs of 128 pages) 209 : 189, 64 of 32 heads behind 8,192 (16 and 8 pages) 32.3 : 38.5, 52 of 32 heads behind 4,096 (8 pages)
// 27.0 : 31.5.
// The shared pages are cut into as many runs as give every compute unit a workgroup, of eight pages at least: every run costs its columns'
// sums, written and read again.  Twice as many, us: 64 sequences of 32 heads behind 8,192 34.4 : 31.7, 24 behind 16,384 31.6 : 28.6, 8
// behind 32,768 44 : 34.5.  Where workgroups of four wavefronts would walk more than SH_LONG_PAGES two stand beside one another (24 sequences
// of 32 heads behind 131,072 127 : 123).
#define SH_SHORT_PAGES 16
#define SH_LONG_PAGES 128
static SharedPlan shared_plan(int tokens, int seqs, int max_new, int shared_pages, int max_len, int heads, int kv_heads) {
    SharedPlan p;
    const int group = heads / kv_heads;
    const long cols = (long)tokens * group;
    p.nt = cols <= 32 ? 0 : cols <= 64 ? 1 : 2;
    p.few = (long)max_new * group <= 16 ? 1 : 2;
    p.own_tiles = (int)(((long)max_new * group + 16 * p.few - 1) / (16 * p.few));
    const long own = max_len - (long)shared_pages * PAGE;
    p.own_pages = (long)seqs * kv_heads * p.own_tiles <= ri_compute_units() ? SH_OWN_PAGES / 2 : SH_OWN_PAGES;      // (max_len changes no sum)
    p.own_chunks = own > 0 ? (int)((own + p.own_pages * PAGE - 1) / (p.own_pages * PAGE)) : 0;
    for (p.waves = cols <= 128 ? 4 : 8;; p.waves = 4) {
        const int of_wg = p.nt == 0 ? 16 * p.few : 16 * p.waves * p.nt;
        p.tiles = (int)((cols + of_wg - 1) / of_wg);
        const long items = (long)p.tiles * kv_heads;
        long runs = ri_compute_units() / items;
        if (p.waves == 4 && shared_pages > SH_LONG_PAGES * runs) runs = 2L * ri_compute_units() / items;
        if (runs < 1) runs = 1;
        p.pages_per_split = (int)((shared_pages + runs - 1) / runs);
        p.pages_per_split += p.pages_per_split & 1;
        if (p.pages_per_split < 8) p.pages_per_split = 8;
        if (p.waves == 4 || p.pages_per_split > SH_SHORT_PAGES) break;
    }
    p.splits = (shared_pages + p.pages_per_split - 1) / p.pages_per_split;
    return p;
}

extern "C" int ri_attention_shared_slots(int tokens, int seqs, int max_new, int shared_pages, int max_len, int heads, int kv_heads) {
    if (tokens < 1 || seqs < 1 || max_new < 1 || shared_pages < 0 || max_len < 1 || kv_heads < 1 || heads < kv_heads) return 0;
    const SharedPlan p = shared_plan(tokens, seqs, max_new, shared_pages, max_len, heads, kv_heads);
    return p.splits + p.own_chunks;
}

extern "C" int ri_attention_shared_bf16(void* out, void* workspace, const void* q, int q_stride, const void* k_pages, const void* v_pages,
                                        const int32_t* cu_seqlens, const int32_t* tok_pos, const int32_t* page_table, int table_width,
                                        int num_pages, int tokens, int seqs, int max_new, int shared_pages, int max_len, int heads,
                                        int kv_heads, int head_dim, int page_size, float scale, void* stream) {
    RI_REQUIRE(tokens >= 1 && seqs >= 1 && max_new >= 1, "attention_shared: %d tokens of %d sequences, %d at most each", tokens, seqs, max_new);
    RI_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "attention_shared: heads %d, kv heads %d", heads, kv_heads);
    RI_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, "attention_shared: head_dim %d (this kernel is built for 32, 64 and 128)", head_dim);
    RI_REQUIRE(page_size == PAGE, "attention_shared: pages of %d tokens (this kernel takes %d)", page_size, PAGE);
    RI_REQUIRE(q_stride >= heads * head_dim && q_stride % 8 == 0 && (uintptr_t)q % 16 == 0, "attention_shared: q row stride %d, or q off a 16-byte boundary", q_stride);
    RI_REQUIRE((uintptr_t)k_pages % 16 == 0 && (uintptr_t)v_pages % 16 == 0, "attention_shared: pages off a 16-byte boundary");
    RI_REQUIRE(table_width > 0 && num_pages > 0, "attention_shared: page table width %d, %d pages", table_width, num_pages);
    RI_REQUIRE(shared_pages >= 0 && shared_pages <= table_width, "attention_shared: %d shared pages, tables of %d", shared_pages, table_width);
    RI_REQUIRE(max_len >= 1 && max_len <= (long)table_width * PAGE, "attention_shared: sequences of up to %d tokens, tables of %d pages", max_len, table_width);
    RI_REQUIRE(kv_heads <= 65535 && tokens <= 65535 && heads <= 65535, "attention_shared: %d tokens, %d heads exceed one launch", tokens, heads);
    // (a token's own keys and a chunk of them are added up in 32 bits)
    RI_REQUIRE((long)table_width * PAGE <= 0x7fffffff - SH_OWN_PAGES * PAGE, "attention_shared: page table width %d", table_width);
    const float scale_log2 = scale * 1.44269504088896341f;
    RI_REQUIRE(scale > 0.f && scale_log2 <= FLT_MAX, "attention_shared: scale %g is not positive, or log2(e) times it no number", (double)scale);
    RI_REQUIRE(out && workspace && q && k_pages && v_pages && cu_seqlens && tok_pos && page_table, "attention_shared: an operand is missing");
    const SharedPlan p = shared_plan(tokens, seqs, max_new, shared_pages, max_len, heads, kv_heads);
    const long of_shared = (long)p.splits * p.tiles * kv_heads, of_own = (long)p.own_chunks * p.own_tiles * seqs * kv_heads;
    RI_REQUIRE(of_shared + of_own <= 0x7fffffff / 512, "attention_shared: %ld workgroups exceed one launch", of_shared + of_own);
    const size_t rows = (size_t)(p.splits + p.own_chunks) * tokens * heads;
    const SharedArgs a = {(float*)workspace, (float2*)((float*)workspace + rows * head_dim), (const bf16_t*)q, (const bf16_t*)k_pages,
                          (const bf16_t*)v_pages, cu_seqlens, tok_pos, page_table, q_stride, table_width, num_pages, tokens, seqs, heads,
                          kv_heads, shared_pages, max_len, p.splits, p.pages_per_split, p.tiles, p.own_tiles, p.own_chunks, p.own_pages,
                          scale_log2};
    const hipStream_t s = (hipStream_t)stream;
    const unsigned own = (unsigned)of_own, shared = (unsigned)of_shared;
    const dim3 join(heads, tokens);
#define SH_FEW(DH, ALL, GRID)                                                                           \
    do {                                                                                                \
        if (p.few == 1) attn_shared_few_kernel<DH, ALL, 1, 4><<<GRID, 256, 0, s>>>(a);                   \
        else attn_shared_few_kernel<DH, ALL, 2, 4><<<GRID, 256, 0, s>>>(a);                              \
    } while (0)
#define SH_LAUNCH(DH)                                                                                   \
    do {                                                                                                \
        if (p.nt == 0) {                                                                                \
            if (own + shared) SH_FEW(DH, true, own + shared);                                           \
        } else {                                                                                        \
            if (own) SH_FEW(DH, false, own);                                                            \
            if (shared == 0) {                                                                          \
            } else if (p.nt == 1) attn_shared_kernel<DH, 1, 4, 2><<<shared, 256, 0, s>>>(a);            \
            else if (p.waves == 4) attn_shared_kernel<DH, 2, 4, 2><<<shared, 256, 0, s>>>(a);           \
            else attn_shared_kernel<DH, 2, 8, 4><<<shared, 512, 0, s>>>(a);                             \
        }                                                                                               \
        attn_shared_join_kernel<DH><<<join, SH_JOIN, 0, s>>>((bf16_t*)out, a);                          \
    } while (0)
    if (head_dim == 128) SH_LAUNCH(128);
    else if (head_dim == 64) SH_LAUNCH(64);
    else SH_LAUNCH(32);
#undef SH_LAUNCH
#undef SH_FEW
    RI_LAUNCH_CHECK("attention_shared");
    return 0;
}
