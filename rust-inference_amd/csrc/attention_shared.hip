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
// Statistics and sums are float32; the weights enter the second product rounded to bfloat16, l is taken before the rounding.
//
// Keys and values behind a sequence's last token are whatever the page held before: they are taken as zeros, so that an
// infinity or NaN there reaches nothing.
#include "attention_mfma.h"

#define SH_WAVES 4
#define SH_OWN_PAGES 16          // pages of a chunk of a sequence's own keys

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
    int splits, pages_per_split, tiles, own_tiles, own_chunks;
    float scale_log2;
};

// Key rows and value columns behind the last key (counted from the page's first) as zeros.
template <int DH>
__device__ __forceinline__ void drop_behind(PageFrags<DH>& f, int last, int lane) {
    const int i = lane & 15, jg = lane >> 4;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
        if ((i >> 2) * 8 + kt * 4 + (i & 3) > last) {
#pragma unroll
            for (int ks = 0; ks < DH / 32; ++ks) f.k[kt][ks].u = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int key = jg * 8 + 2 * e;
        const uint32_t mask = key > last ? 0u : key + 1 > last ? 0x0000FFFFu : 0xFFFFFFFFu;
#pragma unroll
        for (int dt = 0; dt < DH / 16; ++dt) f.v[dt].w[e] &= mask;
    }
}

// A tile of 16 columns over a run of pages, the pages in turn among the wavefronts.
template <int DH>
__global__ void __launch_bounds__(SH_WAVES * 64) attn_shared_kernel(const SharedArgs a) {
    constexpr int LD = DH + 4;
    __shared__ __attribute__((aligned(16))) float o_lds[SH_WAVES][16 * LD];
    __shared__ float m_lds[SH_WAVES][16], l_lds[SH_WAVES][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, jg = lane >> 4;
    const int kvh = blockIdx.y, group = a.heads / a.kv_heads;
    const int shared_items = a.splits * a.tiles;
    int slot, col0, cols, first_token, page0, page1, last_key;
    const int32_t* table = a.page_table;
    if ((int)blockIdx.x < shared_items) {
        slot = blockIdx.x / a.tiles;
        first_token = 0;
        cols = a.tokens * group;
        col0 = (blockIdx.x % a.tiles) * 16;
        page0 = slot * a.pages_per_split;
        page1 = min(page0 + a.pages_per_split, a.shared_pages);
        last_key = a.shared_pages * PAGE - 1;
    } else {
        int item = blockIdx.x - shared_items;
        const int chunk = item % a.own_chunks;
        item /= a.own_chunks;
        const int seq = item / a.own_tiles;
        slot = a.splits + chunk;
        first_token = min(max(a.cu_seqlens[seq], 0), a.tokens);
        const int behind = min(max(a.cu_seqlens[seq + 1], first_token), a.tokens);
        cols = (behind - first_token) * group;
        col0 = (item % a.own_tiles) * 16;
        if (col0 >= cols) return;
        last_key = min(a.tok_pos[behind - 1], a.table_width * PAGE - 1);
        page0 = a.shared_pages + chunk * SH_OWN_PAGES;
        page1 = min(page0 + SH_OWN_PAGES, last_key / PAGE + 1);
        if (page0 >= page1) return;
        table += (size_t)seq * a.table_width;
    }
    Columns<DH, 1> c;
    init_columns<DH, 1>(c);
    const int col = col0 + i, token = first_token + col / group, head = kvh * group + col % group;
    if (col < cols) {
        c.qpos[0] = min(a.tok_pos[token], last_key);
        const bf16_t* q = a.q + (size_t)token * a.q_stride + head * DH + jg * 8;
#pragma unroll
        for (int ks = 0; ks < DH / 32; ++ks) c.q[0][ks].u = *reinterpret_cast<const uint4*>(q + 32 * ks);
    }
    for (int page = page0 + wave; page < page1; page += SH_WAVES) {
        const long phys = min(max(table[page], 0), a.num_pages - 1);
        PageFrags<DH> f;
        load_page<DH>(f, a.k_pages, a.v_pages, phys, a.kv_heads, kvh, lane);
        const int last = last_key - page * PAGE;
        if (last < PAGE - 1) drop_behind<DH>(f, last, lane);
        const bool open = !__any(col < cols && c.qpos[0] < page * PAGE + PAGE - 1);
        process_page<DH, 1>(c, f, page, lane, a.scale_log2, open);
    }
    finish_columns<DH, 1>(c);
    if (jg == 0) {
        m_lds[wave][i] = c.m[0];
        l_lds[wave][i] = c.l[0];
    }
    __syncthreads();
    float m = m_lds[0][i], l = 0.f;
#pragma unroll
    for (int w = 1; w < SH_WAVES; ++w) m = fmaxf(m, m_lds[w][i]);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < SH_WAVES; ++w) l += __builtin_amdgcn_exp2f(m_lds[w][i] - ref) * l_lds[w][i];
    const float mine = __builtin_amdgcn_exp2f(c.m[0] - ref);
#pragma unroll
    for (int dt = 0; dt < DH / 16; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o_lds[wave][i * LD + dt * 16 + jg * 4 + e] = c.o[0][dt][e] * mine;
    if (wave == 0 && jg == 0 && col < cols) a.stats[((size_t)slot * a.tokens + token) * a.heads + head] = make_float2(m, l);
    __syncthreads();
    for (int at = threadIdx.x; at < 16 * DH; at += SH_WAVES * 64) {
        const int r = at / DH, d = at % DH, cc = col0 + r;
        if (cc >= cols) break;
        float o = o_lds[0][r * LD + d];
#pragma unroll
        for (int w = 1; w < SH_WAVES; ++w) o += o_lds[w][r * LD + d];
        a.sums[(((size_t)slot * a.tokens + first_token + cc / group) * a.heads + kvh * group + cc % group) * DH + d] = o;
    }
}

// A token's runs and chunks joined, a workgroup a (head, token); tokens that are no sequence's get zeros.
template <int DH>
__global__ void __launch_bounds__(DH) attn_shared_join_kernel(bf16_t* __restrict__ out, const SharedArgs a) {
    const int head = blockIdx.x, token = blockIdx.y, d = threadIdx.x;
    const int first = a.cu_seqlens[0], behind = a.cu_seqlens[a.seqs];
    bf16_t* to = out + ((size_t)token * a.heads + head) * DH + d;
    if (token < first || token >= behind) {
        *to = 0;
        return;
    }
    const int own = min(a.tok_pos[token], a.table_width * PAGE - 1) + 1 - a.shared_pages * PAGE;      // own keys that it sees
    const int chunks = own > 0 ? min((own + SH_OWN_PAGES * PAGE - 1) / (SH_OWN_PAGES * PAGE), a.own_chunks) : 0;
    const int slots = a.splits + chunks;
    const size_t at = (size_t)token * a.heads + head, step = (size_t)a.tokens * a.heads;
    float m = -INFINITY;
    for (int s = 0; s < slots; ++s) m = fmaxf(m, a.stats[s * step + at].x);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f, o = 0.f;
    for (int s = 0; s < slots; ++s) {
        const float2 st = a.stats[s * step + at];
        const float w = __builtin_amdgcn_exp2f(st.x - ref);
        l += w * st.y;
        o += w * a.sums[(s * step + at) * DH + d];
    }
    *to = f32_to_bf16(l > 0.f ? o / l : 0.f);
}

struct SharedPlan { int splits, pages_per_split, tiles, own_tiles, own_chunks; };

// Runs of the shared pages: four workgroups a compute unit, eight pages a run at least (two a wavefront).
static SharedPlan shared_plan(int tokens, int seqs, int max_new, int shared_pages, int max_len, int heads, int kv_heads) {
    SharedPlan p;
    const int group = heads / kv_heads;
    p.tiles = (int)(((long)tokens * group + 15) / 16);
    p.own_tiles = (int)(((long)max_new * group + 15) / 16);
    const int own = max_len - shared_pages * PAGE;
    p.own_chunks = own > 0 ? (own + SH_OWN_PAGES * PAGE - 1) / (SH_OWN_PAGES * PAGE) : 0;
    const long wanted = 4L * ri_compute_units() / ((long)p.tiles * kv_heads) + 1;
    p.pages_per_split = shared_pages ? (int)((shared_pages + wanted - 1) / wanted) : 1;
    if (p.pages_per_split < 8) p.pages_per_split = 8;
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
    RI_REQUIRE(table_width > 0 && num_pages > 0, "attention_shared: page table width %d, %d pages", table_width, num_pages);
    RI_REQUIRE(shared_pages >= 0 && shared_pages <= table_width, "attention_shared: %d shared pages, tables of %d", shared_pages, table_width);
    RI_REQUIRE(max_len >= 1 && max_len <= (long)table_width * PAGE, "attention_shared: sequences of up to %d tokens, tables of %d pages", max_len, table_width);
    RI_REQUIRE(kv_heads <= 65535 && tokens <= 65535 && heads <= 65535, "attention_shared: %d tokens, %d heads exceed one launch", tokens, heads);
    RI_REQUIRE((long)table_width * PAGE < 0x7fffffff, "attention_shared: page table width %d", table_width);
    RI_REQUIRE(scale > 0.f, "attention_shared: scale %g is not positive", (double)scale);
    RI_REQUIRE(out && workspace && q && k_pages && v_pages && cu_seqlens && tok_pos && page_table, "attention_shared: an operand is missing");
    const SharedPlan p = shared_plan(tokens, seqs, max_new, shared_pages, max_len, heads, kv_heads);
    const long items = (long)p.splits * p.tiles + (long)p.own_chunks * p.own_tiles * seqs;
    RI_REQUIRE(items <= 0x7fffffff, "attention_shared: %ld workgroups exceed one launch", items);
    const size_t rows = (size_t)(p.splits + p.own_chunks) * tokens * heads;
    const SharedArgs a = {(float*)workspace, (float2*)((float*)workspace + rows * head_dim), (const bf16_t*)q, (const bf16_t*)k_pages,
                          (const bf16_t*)v_pages, cu_seqlens, tok_pos, page_table, q_stride, table_width, num_pages, tokens, seqs, heads,
                          kv_heads, shared_pages, p.splits, p.pages_per_split, p.tiles, p.own_tiles, p.own_chunks,
                          scale * 1.44269504088896341f};
    const hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)items, kv_heads), join(heads, tokens);
#define SH_LAUNCH(DH)                                                             \
    do {                                                                          \
        if (items) attn_shared_kernel<DH><<<grid, SH_WAVES * 64, 0, s>>>(a);      \
        attn_shared_join_kernel<DH><<<join, DH, 0, s>>>((bf16_t*)out, a);         \
    } while (0)
    if (head_dim == 128) SH_LAUNCH(128);
    else if (head_dim == 64) SH_LAUNCH(64);
    else SH_LAUNCH(32);
#undef SH_LAUNCH
    RI_LAUNCH_CHECK("attention_shared");
    return 0;
}
