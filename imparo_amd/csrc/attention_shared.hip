// Decode attention for rows in groups that share a prefix: the keys and values that all rows of a group have in the same pages are
// read once for all of them, the keys behind are each row's own.
//
// The result is the softmax over all keys a row sees, taken in parts: a part p of the keys leaves its reference m_p, l_p = sum 2^(s - m_p)
// and O_p = sum 2^(s - m_p) v (s: scaled scores times log2(e)), and with M = max m_p the output is sum 2^(m_p - M) O_p / sum 2^(m_p - M) l_p.
// One launch makes all parts: blocks for the groups' shared keys, whose queries are those of all rows of the group side by side, and blocks
// for each row's own keys; a second launch adds the parts up.
//
// A wave walks over tiles of 32 keys with the 32x32x16 product, arranged so that nothing moves between lanes:
//   S^T[key][query] = K Q^T     lane: column query lane % 32, rows 8 (r / 4) + 4 (lane / 32) + r % 4 for r of 16
//   O^T[dim][query] += V^T P^T  the operand P^T wants keys 16 u + 8 (lane / 32) + j in lane's slots j of product u
// Which key a row of the first product stands for is free to choose: row 16 u + 8 a + 4 h + t is key 16 u + 8 h + 4 a + t (two bits
// change places), so that the lane's results 8 u + j are exactly the keys its operand of the second product wants.
#include "common.h"
#include "api.h"

#define SHARED_WAVES 4
#define SHARED_MIN_SPLIT 256       // keys a part has at least

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
union SharedFrag {
    u32x4 u;
    bf16x8 v;
};
// a piece of values at keys key .. key + 7 with those outside [lo, hi] zeroed, whatever stands there
__device__ __forceinline__ u32x4 only_between(u32x4 v, int key, int lo, int hi) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = key + 2 * j;
        v[j] &= (k >= lo && k <= hi ? 0xFFFFu : 0u) | (k + 1 >= lo && k + 1 <= hi ? 0xFFFF0000u : 0u);
    }
    return v;
}
__device__ __forceinline__ u32x4 load16(const bf16_t* p) { return *reinterpret_cast<const u32x4*>(p); }

struct SharedArgs {
    const bf16_t* __restrict__ q;
    const bf16_t* __restrict__ k;
    const bf16_t* __restrict__ v;
    bf16_t* __restrict__ out;
    float* __restrict__ part_o;      // [listed rows, heads, parts, D]
    float* __restrict__ part_ml;     // [listed rows, heads, parts, 2]
    const int32_t* __restrict__ rows;
    const int32_t* __restrict__ group_start;
    const int32_t* __restrict__ shared;
    const int32_t* __restrict__ seg_start;
    const int32_t* __restrict__ positions;
    const int32_t* __restrict__ table;
    int n_rows, n_groups, stride, page_shift, heads, kv_heads, n_pages, window;
    int n_pre, pre_split, n_own, own_split;      // parts and keys a part: of the shared keys, of a row's own
    int pre_tiles;                               // tiles of queries a group's kv head has at most
    float scale;                                 // its size, times log2(e)
    uint32_t flip;                               // its sign, for two bfloat16 of a query at once
};

// The group a listed row is in (its keys up to `shared` are the group's), or -1. All lanes ask for the same row.
__device__ __forceinline__ int group_of(const SharedArgs& a, int i) {
    const int lane = threadIdx.x & (WAVE - 1);
    for (int g0 = 0; g0 < a.n_groups; g0 += WAVE) {
        const int g = g0 + lane;
        const bool here = g < a.n_groups && a.group_start[g] <= i && i < a.group_start[g + 1];
        const unsigned long long who = __ballot(here);
        if (who) return g0 + __ffsll((long long)who) - 1;
    }
    return -1;
}
// 16 bytes of a query, its sign turned where the scale is negative: the largest score is then that of the largest product
__device__ __forceinline__ u32x4 query_piece(const SharedArgs& a, const bf16_t* q, bool valid) {
    return valid ? load16(q) ^ a.flip : u32x4{0u, 0u, 0u, 0u};
}
// how many keys a group's rows share, inside what a table can name
__device__ __forceinline__ int shared_keys(const SharedArgs& a, int g) {
    return g < 0 ? 0 : (int)min((long long)max(a.shared[g], 0), (long long)a.stride << a.page_shift);
}

template <int ND>
struct SharedTile {
    static constexpr int DT = (ND + 1) / 2;
    SharedFrag k[ND];        // key (row) lane % 32 permuted, dims 16 ks + 8 h + j
    SharedFrag v[2][DT];     // dim 32 dt + lane % 32, keys 16 u + 8 h + j
};

// The pages of a tile of 32 keys, asked for a tile ahead: one for its first 16 keys and one for the others, the same where pages hold
// 32 keys or more (PAGED). [lo, hi] are the keys that any query reads: pages are looked up inside it only.
template <bool PAGED>
struct TilePages {
    int page[PAGED ? 1 : 2];
    __device__ __forceinline__ void ask(const SharedArgs& a, const int32_t* __restrict__ table, int key0, int lo, int hi) {
#pragma unroll
        for (int u = 0; u < (PAGED ? 1 : 2); ++u) page[u] = table[min(max(key0 + 16 * u, lo & ~15), hi & ~15) >> a.page_shift];
    }
    // where a head's part of the page begins, and where in the page the 16 keys do (the same for the whole wave)
    __device__ __forceinline__ size_t head(const SharedArgs& a, int u, int kvh) const {
        const int p = __builtin_amdgcn_readfirstlane(page[PAGED ? 0 : u]);
        return ((size_t)min(max(p, 0), a.n_pages - 1) * a.kv_heads + kvh) << a.page_shift;
    }
    __device__ __forceinline__ int slot(const SharedArgs& a, int u, int key0) const { return (key0 + 16 * u) & ((1 << a.page_shift) - 1); }
};

// Asks for the tile of keys key0 .. key0 + 31, whose pages are there. What a page holds outside [lo, hi] is read with it and masked later.
template <int ND, bool PAGED>
__device__ __forceinline__ void shared_load(SharedTile<ND>& t, const SharedArgs& a, const TilePages<PAGED>& pages, int kvh, int key0, int lane) {
    constexpr int D = ND * 16, DT = (ND + 1) / 2;
    const int c = lane & 31, h = lane >> 5, page_size = 1 << a.page_shift;
    const int key = (c & 16) | (c & 4) << 1 | (c & 8) >> 1 | (c & 3);
    if constexpr (PAGED) {
        const size_t head = pages.head(a, 0, kvh);
        const int slot = pages.slot(a, 0, key0);
        const bf16_t *k = a.k + (head + slot) * D, *v = a.v + head * D + slot;
#pragma unroll
        for (int ks = 0; ks < ND; ++ks) t.k[ks].u = load16(k + (key * D + 8 * h + 16 * ks));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int d = min(32 * dt + c, D - 1);           // (dims past the head: the last again, never written out)
#pragma unroll
            for (int u = 0; u < 2; ++u) t.v[u][dt].u = load16(v + ((d << a.page_shift) + 8 * h + 16 * u));
        }
    } else {
        const size_t head0 = pages.head(a, 0, kvh), head1 = pages.head(a, 1, kvh);
        const int slot0 = pages.slot(a, 0, key0), slot1 = pages.slot(a, 1, key0);
        const bf16_t* k = a.k + (key & 16 ? (head1 + slot1) * D : (head0 + slot0) * D) + ((key & 15) * D + 8 * h);
#pragma unroll
        for (int ks = 0; ks < ND; ++ks) t.k[ks].u = load16(k + 16 * ks);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int d = min(32 * dt + c, D - 1);
            t.v[0][dt].u = load16(a.v + head0 * D + slot0 + (d * page_size + 8 * h));
            t.v[1][dt].u = load16(a.v + head1 * D + slot1 + (d * page_size + 8 * h));
        }
    }
}

template <int ND, int MT>
struct SharedState {
    static constexpr int DT = (ND + 1) / 2;
    SharedFrag q[MT][ND];
    f32x16 o[MT][DT];
    float m[MT], l[MT];      // reference of the exponentials (one for both halves of the wave), this lane's share of their sum
    int lo[MT], hi[MT];      // keys this lane's query sees
};

// One tile: scores, exponentials, weighted values. The reference of a query's exponentials moves only when a score passes it by 8 or more (a
// power of two of 8, harmless to float32 sums and to the rounding of the weights): most tiles then multiply no accumulator.
// Weights are rounded to bfloat16 for the second product, half a step of 2^-8 each and of either sign; the sum takes them as they were.
// EDGE: some key of the tile is outside some query's range. What is outside every query's range may be anything: such values are zeroed.
template <int ND, int MT, bool EDGE>
__device__ __forceinline__ void shared_tile(SharedState<ND, MT>& st, const SharedTile<ND>& t, int key0, int lo, int hi, float scale,
                                            int lane) {
    constexpr int DT = (ND + 1) / 2;
    const int h = lane >> 5;
    SharedFrag p[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < ND; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(t.k[ks].v, st.q[mt][ks].v, s, 0, 0, 0);
        if (EDGE) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = key0 + 16 * (r >> 3) + 8 * h + (r & 7);
                s[r] = key >= st.lo[mt] && key <= st.hi[mt] ? s[r] : -INFINITY;
            }
        }
        float mx = fmaxf(s[0], s[1]);
#pragma unroll
        for (int r = 2; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
        mx *= scale;
        if (__any(mx > st.m[mt] + 8.f)) {
            const float m_new = fmaxf(st.m[mt], fmaxf(mx, lane_xor<32>(mx)));
            const float corr = st.m[mt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m[mt] - m_new);
            st.m[mt] = m_new;
            st.l[mt] *= corr;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) st.o[mt][dt][r] *= corr;
        }
        const float m = st.m[mt] == -INFINITY ? 0.f : st.m[mt];
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], scale, -m));
            sum += s[r];
        }
        st.l[mt] += sum;
#pragma unroll
        for (int u = 0; u < 2; ++u)
            p[mt][u].u = u32x4{f32x2_to_bf16x2(s[8 * u], s[8 * u + 1]), f32x2_to_bf16x2(s[8 * u + 2], s[8 * u + 3]),
                               f32x2_to_bf16x2(s[8 * u + 4], s[8 * u + 5]), f32x2_to_bf16x2(s[8 * u + 6], s[8 * u + 7])};
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            SharedFrag a = t.v[u][dt];
            if (EDGE) a.u = only_between(a.u, key0 + 16 * u + 8 * h, lo, hi);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                st.o[mt][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, p[mt][u].v, st.o[mt][dt], 0, 0, 0);
        }
}

// One block's part: the queries `first_query` .. of the rows from `first_row` on (query x is row x / per, head x % per of the kv head), over the
// keys [begin, end) of the table, each query inside what it sees; the four waves take tiles in turn, meet in LDS, and leave one part.
template <int ND, int MT, bool PAGED>
__device__ __forceinline__ void shared_part(const SharedArgs& a, int first_row, int n_queries, int first_query, int per, int kvh,
                                            const int32_t* __restrict__ table, int begin, int end, int part, float* lds) {
    constexpr int D = ND * 16, DT = (ND + 1) / 2;
    const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int c = lane & 31, h = lane >> 5;
    SharedState<ND, MT> st;
    size_t place[MT];
    int lo_all = INT32_MAX, hi_all = -1, lo_in = 0, hi_in = INT32_MAX;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int x = first_query + 32 * mt + c;
        const bool valid = x < n_queries;
        const int i = first_row + (valid ? x / per : 0), head = kvh * per + (valid ? x % per : 0);
        const int t = a.seg_start[a.rows[i]];
        const int pos = (int)min((long long)a.positions[t], ((long long)a.stride << a.page_shift) - 1);
        const bf16_t* qrow = a.q + ((size_t)t * a.heads + head) * D + 8 * h;
#pragma unroll
        for (int ks = 0; ks < ND; ++ks)
            st.q[mt][ks].u = query_piece(a, qrow + 16 * ks, valid);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) st.o[mt][dt][r] = 0.f;
        st.m[mt] = -INFINITY;
        st.l[mt] = 0.f;
        st.lo[mt] = max(begin, pos < 0 ? 0 : first_seen(pos, a.window));
        st.hi[mt] = min(end - 1, pos);
        const bool sees = valid && st.lo[mt] <= st.hi[mt];
        if (!sees) st.lo[mt] = INT32_MAX, st.hi[mt] = -1;
        // the widest and the narrowest range; a lane without a query asks for nothing and leaves the narrowest as it is
        lo_all = min(lo_all, st.lo[mt]);
        hi_all = max(hi_all, st.hi[mt]);
        if (valid) {
            lo_in = max(lo_in, st.lo[mt]);
            hi_in = min(hi_in, st.hi[mt]);
        }
        place[mt] = valid ? ((size_t)i * a.heads + head) * (a.n_pre + a.n_own) + part : (size_t)-1;
    }
#pragma unroll
    for (int n = 1; n < 32; n <<= 1) {
        lo_all = min(lo_all, __shfl_xor(lo_all, n, WAVE));
        hi_all = max(hi_all, __shfl_xor(hi_all, n, WAVE));
        lo_in = max(lo_in, __shfl_xor(lo_in, n, WAVE));
        hi_in = min(hi_in, __shfl_xor(hi_in, n, WAVE));
    }
    lo_all = __builtin_amdgcn_readfirstlane(lo_all);
    hi_all = __builtin_amdgcn_readfirstlane(hi_all);
    lo_in = __builtin_amdgcn_readfirstlane(lo_in);
    hi_in = __builtin_amdgcn_readfirstlane(hi_in);

    if (lo_all <= hi_all) {
        constexpr int STEP = 32 * SHARED_WAVES;
        int key0 = (lo_all & ~31) + 32 * wave;
        auto step = [&](const SharedTile<ND>& t, int key) __attribute__((always_inline)) {
            if (key >= lo_in && key + 31 <= hi_in) shared_tile<ND, MT, false>(st, t, key, lo_all, hi_all, a.scale, lane);
            else shared_tile<ND, MT, true>(st, t, key, lo_all, hi_all, a.scale, lane);
        };
        SharedTile<ND> even, odd;
        TilePages<PAGED> pages;
        auto ask = [&](SharedTile<ND>& t, int key) __attribute__((always_inline)) {
            shared_load<ND, PAGED>(t, a, pages, kvh, key, lane);
            pages.ask(a, table, key + STEP, lo_all, hi_all);
        };
        if (key0 <= hi_all) {
            pages.ask(a, table, key0, lo_all, hi_all);
            ask(even, key0);
        }
        while (key0 <= hi_all) {
            if (key0 + STEP <= hi_all) ask(odd, key0 + STEP);
            step(even, key0);
            key0 += STEP;
            if (key0 > hi_all) break;
            if (key0 + STEP <= hi_all) ask(even, key0 + STEP);
            step(odd, key0);
            key0 += STEP;
        }
    }

    // ---- the waves meet: references first, then sums and accumulators of waves 2 and 3 onto 0 and 1, and 1 onto 0
    float* ml = lds + 2 * DT * 16 * WAVE;                          // [MT][4 waves][32]
    float f[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        st.l[mt] += lane_xor<32>(st.l[mt]);
        if (h == 0) ml[(mt * SHARED_WAVES + wave) * 32 + c] = st.m[mt];
    }
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < SHARED_WAVES; ++w) m = fmaxf(m, ml[(mt * SHARED_WAVES + w) * 32 + c]);
        f[mt] = st.m[mt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m[mt] - m);
        st.m[mt] = m;
        st.l[mt] *= f[mt];
    }
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
        if (h == 0) ml[(mt * SHARED_WAVES + wave) * 32 + c] = st.l[mt];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) st.o[mt][dt][r] = f[mt] > 0.f ? st.o[mt][dt][r] * f[mt] : 0.f;
        for (int from = 2; from >= 1; --from) {                    // (waves 2, 3 first; then wave 1)
            if (wave >= from && wave < 2 * from)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) lds[(((wave - from) * DT + dt) * 16 + r) * WAVE + lane] = st.o[mt][dt][r];
            __syncthreads();
            if (wave < from)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) st.o[mt][dt][r] += lds[((wave * DT + dt) * 16 + r) * WAVE + lane];
            __syncthreads();
        }
        if (wave == 0 && place[mt] != (size_t)-1) {
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < SHARED_WAVES; ++w) l += ml[(mt * SHARED_WAVES + w) * 32 + c];
            if (h == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * place[mt]) = make_float2(st.m[mt], l);
            float* o = a.part_o + place[mt] * D;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int d = 32 * dt + 8 * b + 4 * h;
                    if (d < D)
                        *reinterpret_cast<float4*>(o + d) = make_float4(st.o[mt][dt][4 * b], st.o[mt][dt][4 * b + 1],
                                                                        st.o[mt][dt][4 * b + 2], st.o[mt][dt][4 * b + 3]);
                }
        }
    }
}

template <int ND, int MT, bool PAGED>
__global__ __launch_bounds__(SHARED_WAVES * WAVE, ND * MT > 4 ? 1 : 2) void k_attn_shared(SharedArgs a) {
    constexpr int DT = (ND + 1) / 2;
    __shared__ __attribute__((aligned(16))) float lds[2 * DT * 16 * WAVE + MT * SHARED_WAVES * 32];
    const int per = a.heads / a.kv_heads, b = blockIdx.x;
    // the tiles of queries that read the same keys follow one another eight blocks apart: on one XCD, whose L2 has them
    const int tile = (b / 8) % a.pre_tiles, unit = b / (8 * a.pre_tiles) * 8 + b % 8;
    const int part = unit % a.n_pre, kvh = unit / a.n_pre % a.kv_heads, g = unit / (a.n_pre * a.kv_heads);
    if (g >= a.n_groups) return;
    const int first = max(a.group_start[g], 0), n = min(a.group_start[g + 1], a.n_rows) - first;
    const int keys = shared_keys(a, g), begin = part * a.pre_split, end = min(begin + a.pre_split, keys);
    const int first_query = tile * 32 * MT;
    if (first_query >= n * per || begin >= keys) return;
    shared_part<ND, MT, PAGED>(a, first, n * per, first_query, per, kvh, a.table + (size_t)a.rows[first] * a.stride, begin, end, part, lds);
}

// ---- shared keys of many queries
// With more than 64 queries a kv head a block's four waves take 32 queries each and walk over the same keys, 64 at a time, which the block keeps
// in LDS twice: one tile is multiplied while the next one's loads are on their way in registers. Rows are padded by 16 bytes, an odd
// number of 16-byte pieces, so that operand reads of neighbouring rows fall on different banks. Bound by the exponentials: 16 a lane and 32
// keys, a quarter of a lane's rate each, against ND + ND products.
#define MANY_KEYS 64

template <int ND, bool PAGED>
__global__ __launch_bounds__(SHARED_WAVES * WAVE, 2) void k_attn_shared_many(SharedArgs a) {
    constexpr int D = ND * 16, DT = (ND + 1) / 2, THREADS = SHARED_WAVES * WAVE;
    constexpr int LDK = D + 8, LDV = MANY_KEYS + 8, CH = D / 8;                   // CH: 16-byte pieces of a key
    constexpr int K_PIECES = MANY_KEYS * CH, V_PIECES = D * (MANY_KEYS / 8);
    constexpr int K_PER = (K_PIECES + THREADS - 1) / THREADS, V_PER = (V_PIECES + THREADS - 1) / THREADS;
    __shared__ __attribute__((aligned(16))) bf16_t ks[2][MANY_KEYS * LDK], vs[2][DT * 32 * LDV];
    __shared__ int ranges[2][SHARED_WAVES];
    const int per = a.heads / a.kv_heads, b = blockIdx.x, tid = threadIdx.x;
    const int lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE), c = lane & 31, h = lane >> 5;
    const int block = (b / 8) % a.pre_tiles, unit = b / (8 * a.pre_tiles) * 8 + b % 8;
    const int part = unit % a.n_pre, kvh = unit / a.n_pre % a.kv_heads, g = unit / (a.n_pre * a.kv_heads);
    if (g >= a.n_groups) return;
    const int first_row = max(a.group_start[g], 0), n_queries = (min(a.group_start[g + 1], a.n_rows) - first_row) * per;
    const int keys = shared_keys(a, g), begin = part * a.pre_split, end = min(begin + a.pre_split, keys);
    if (block * 32 * SHARED_WAVES >= n_queries || begin >= keys) return;
    const int32_t* __restrict__ table = a.table + (size_t)a.rows[first_row] * a.stride;

    // ---- this wave's queries
    const int x = (block * SHARED_WAVES + wave) * 32 + c;
    const bool valid = x < n_queries;
    const int i = first_row + (valid ? x / per : 0), head = kvh * per + (valid ? x % per : 0);
    const int t = a.seg_start[a.rows[i]];
    const int pos = (int)min((long long)a.positions[t], ((long long)a.stride << a.page_shift) - 1);
    SharedFrag q[ND];
    const bf16_t* qrow = a.q + ((size_t)t * a.heads + head) * D + 8 * h;
#pragma unroll
    for (int k = 0; k < ND; ++k) q[k].u = query_piece(a, qrow + 16 * k, valid);
    int lo = max(begin, pos < 0 ? 0 : first_seen(pos, a.window)), hi = min(end - 1, pos);
    if (!valid || lo > hi) lo = INT32_MAX, hi = -1;
    int lo_w = lo, hi_w = hi, lo_in = valid ? lo : 0, hi_in = valid ? hi : INT32_MAX;
#pragma unroll
    for (int n = 1; n < 32; n <<= 1) {
        lo_w = min(lo_w, __shfl_xor(lo_w, n, WAVE));
        hi_w = max(hi_w, __shfl_xor(hi_w, n, WAVE));
        lo_in = max(lo_in, __shfl_xor(lo_in, n, WAVE));
        hi_in = min(hi_in, __shfl_xor(hi_in, n, WAVE));
    }
    lo_w = __builtin_amdgcn_readfirstlane(lo_w), hi_w = __builtin_amdgcn_readfirstlane(hi_w);
    lo_in = __builtin_amdgcn_readfirstlane(lo_in), hi_in = __builtin_amdgcn_readfirstlane(hi_in);
    if (lane == 0) ranges[0][wave] = lo_w, ranges[1][wave] = hi_w;
    __syncthreads();
    int lo_all = INT32_MAX, hi_all = -1;
#pragma unroll
    for (int w = 0; w < SHARED_WAVES; ++w) lo_all = min(lo_all, ranges[0][w]), hi_all = max(hi_all, ranges[1][w]);

    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
    float m = -INFINITY, l = 0.f;

    if (lo_all <= hi_all) {
        const int page_size = 1 << a.page_shift;
        // a thread's pieces of a tile: keys k_row[j] of K, and of V the eight keys from v_key on (of K_PER and V_PER rows)
        const int v_key = 8 * (tid % (MANY_KEYS / 8));
        // PAGED: a tile lies in one page, and a thread's places in it are always the same
        u32x4 kr[K_PER], vr[V_PER];
        int k_page[PAGED ? 1 : K_PER], v_page = 0;
        auto ask_pages = [&](int key0) __attribute__((always_inline)) {
            if constexpr (PAGED) {
                k_page[0] = table[min(key0, hi_all) >> a.page_shift];
            } else {
#pragma unroll
                for (int j = 0; j < K_PER; ++j)
                    k_page[j] = table[min(max(key0 + min(tid + j * THREADS, K_PIECES - 1) / CH, lo_all), hi_all) >> a.page_shift];
                v_page = table[min(max(key0 + v_key, lo_all & ~7), hi_all & ~7) >> a.page_shift];
            }
        };
        auto ask_tile = [&](int key0) __attribute__((always_inline)) {            // (the pages asked for before)
            if constexpr (PAGED) {
                const size_t page = min(max(__builtin_amdgcn_readfirstlane(k_page[0]), 0), a.n_pages - 1);
                const size_t head = (page * a.kv_heads + kvh) << a.page_shift;
                const int slot = key0 & (page_size - 1);
                const bf16_t *k = a.k + (head + slot) * D, *v = a.v + head * D + slot;
#pragma unroll
                for (int j = 0; j < K_PER; ++j) kr[j] = load16(k + 8 * min(tid + j * THREADS, K_PIECES - 1));
#pragma unroll
                for (int j = 0; j < V_PER; ++j)
                    vr[j] = load16(v + ((min(tid + j * THREADS, V_PIECES - 1) / (MANY_KEYS / 8) << a.page_shift) + v_key));
            } else {
#pragma unroll
                for (int j = 0; j < K_PER; ++j) {
                    const int piece = min(tid + j * THREADS, K_PIECES - 1), key = min(max(key0 + piece / CH, lo_all), hi_all);
                    const size_t page = min(max(k_page[j], 0), a.n_pages - 1);
                    kr[j] = load16(a.k + ((page * a.kv_heads + kvh) * page_size + (key & (page_size - 1))) * D + 8 * (piece % CH));
                }
                const size_t page = min(max(v_page, 0), a.n_pages - 1);
                const int slot = min(max(key0 + v_key, lo_all & ~7), hi_all & ~7) & (page_size - 1);
#pragma unroll
                for (int j = 0; j < V_PER; ++j) {
                    const int d = min(tid + j * THREADS, V_PIECES - 1) / (MANY_KEYS / 8);
                    vr[j] = load16(a.v + ((page * a.kv_heads + kvh) * D + d) * page_size + slot);
                }
            }
        };
        auto keep_tile = [&](int key0, int buf) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < K_PER; ++j) {
                const int piece = tid + j * THREADS;
                if (K_PIECES % THREADS == 0 || piece < K_PIECES)
                    *reinterpret_cast<u32x4*>(&ks[buf][piece / CH * LDK + 8 * (piece % CH)]) = kr[j];
            }
            if (key0 < lo_all || key0 + MANY_KEYS - 1 > hi_all) {                 // values that no query reads may be anything: zeros
#pragma unroll
                for (int j = 0; j < V_PER; ++j) vr[j] = only_between(vr[j], key0 + v_key, lo_all, hi_all);
            }
#pragma unroll
            for (int j = 0; j < V_PER; ++j) {
                const int piece = tid + j * THREADS;
                if (V_PIECES % THREADS == 0 || piece < V_PIECES)
                    *reinterpret_cast<u32x4*>(&vs[buf][piece / (MANY_KEYS / 8) * LDV + v_key]) = vr[j];
            }
        };
        int key0 = lo_all & ~(MANY_KEYS - 1), buf = 0;
        ask_pages(key0);
        ask_tile(key0);
        ask_pages(key0 + MANY_KEYS);
        keep_tile(key0, 0);
        ask_tile(key0 + MANY_KEYS);
        ask_pages(key0 + 2 * MANY_KEYS);
        __syncthreads();
        for (; key0 <= hi_all; key0 += MANY_KEYS, buf ^= 1) {
#pragma unroll
            for (int half = 0; half < MANY_KEYS / 32; ++half) {
                const int key = key0 + 32 * half;
                if (key > hi_w || key + 31 < lo_w) continue;
                const bf16_t* krow = &ks[buf][(32 * half + ((c & 16) | (c & 4) << 1 | (c & 8) >> 1 | (c & 3))) * LDK + 8 * h];
                f32x16 s;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
                for (int k = 0; k < ND; ++k) {
                    SharedFrag f;
                    f.u = load16(krow + 16 * k);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.v, q[k].v, s, 0, 0, 0);
                }
                if (key < lo_in || key + 31 > hi_in) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int at = key + 16 * (r >> 3) + 8 * h + (r & 7);
                        s[r] = at >= lo && at <= hi ? s[r] : -INFINITY;
                    }
                }
                float mx = fmaxf(s[0], s[1]);
#pragma unroll
                for (int r = 2; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
                mx *= a.scale;
                if (__any(mx > m + 8.f)) {
                    const float m_new = fmaxf(m, fmaxf(mx, lane_xor<32>(mx)));
                    const float corr = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
                    m = m_new;
                    l *= corr;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[dt][r] *= corr;
                }
                const float from = m == -INFINITY ? 0.f : m;
                float sum = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale, -from));
                    sum += s[r];
                }
                l += sum;
                SharedFrag p[2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    p[u].u = u32x4{f32x2_to_bf16x2(s[8 * u], s[8 * u + 1]), f32x2_to_bf16x2(s[8 * u + 2], s[8 * u + 3]),
                                   f32x2_to_bf16x2(s[8 * u + 4], s[8 * u + 5]), f32x2_to_bf16x2(s[8 * u + 6], s[8 * u + 7])};
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        SharedFrag f;                                             // (rows past the head: whatever stands there, never written out)
                        f.u = load16(&vs[buf][(32 * dt + c) * LDV + 32 * half + 16 * u + 8 * h]);
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.v, p[u].v, o[dt], 0, 0, 0);
                    }
            }
            if (key0 + MANY_KEYS <= hi_all) {
                keep_tile(key0 + MANY_KEYS, buf ^ 1);
                ask_tile(key0 + 2 * MANY_KEYS);
                ask_pages(key0 + 3 * MANY_KEYS);
            }
            __syncthreads();
        }
    }
    l += lane_xor<32>(l);
    if (!valid) return;
    const size_t place = ((size_t)i * a.heads + head) * (a.n_pre + a.n_own) + part;
    if (h == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * place) = make_float2(m, l);
    float* out = a.part_o + place * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = 32 * dt + 8 * r + 4 * h;
            if (d < D) *reinterpret_cast<float4*>(out + d) = make_float4(o[dt][4 * r], o[dt][4 * r + 1], o[dt][4 * r + 2], o[dt][4 * r + 3]);
        }
}

// ---- a row's own keys
// Few queries (the heads of one kv head) over keys that nobody else reads: bound by memory, so the 16x16x32 product, whose state of 16 queries
// is small, and many waves a SIMD. S^T in two products of 16 keys whose row m is key 8 (m / 4) + 4 t + m % 4 of product t: a lane has
// 8 consecutive keys of query lane % 16 (those from 8 (lane / 16) on), as the second product wants them.
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int ND>
struct OwnTile {
    SharedFrag k[2][(ND + 1) / 2];
    SharedFrag v[ND];
};

template <int ND, bool PAGED>
__device__ __forceinline__ void own_load(OwnTile<ND>& t, const SharedArgs& a, const TilePages<PAGED>& pages, int kvh, int key0, int lane) {
    constexpr int D = ND * 16, NK = (ND + 1) / 2;
    const int c = lane & 15, g = lane >> 4;
    const size_t head0 = pages.head(a, 0, kvh), head1 = PAGED ? head0 : pages.head(a, 1, kvh);
    const int slot0 = pages.slot(a, 0, key0), slot1 = PAGED ? slot0 + 16 : pages.slot(a, 1, key0);
    const bf16_t *k, *v;
    int krow, vcol;
    if constexpr (PAGED) {
        k = a.k + (head0 + slot0) * D, v = a.v + head0 * D + slot0;
        krow = 8 * (c >> 2) + (c & 3), vcol = 8 * g;
    } else {
        k = a.k + (c & 8 ? (head1 + slot1) * D : (head0 + slot0) * D), v = a.v + (g & 2 ? head1 * D + slot1 : head0 * D + slot0);
        krow = 8 * ((c >> 2) & 1) + (c & 3), vcol = 8 * (g & 1);
    }
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int ks = 0; ks < NK; ++ks)                          // (dims past the head: the row's last 8 again, zeroed before use)
            t.k[p][ks].u = load16(k + ((krow + 4 * p) * D + min(32 * ks + 8 * g, D - 8)));
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) t.v[dt].u = load16(v + (((16 * dt + c) << a.page_shift) + vcol));
}

template <int ND>
struct OwnState {
    SharedFrag q[(ND + 1) / 2];
    f32x4 o[ND];
    float m, l;
};

template <int ND>
__device__ __forceinline__ void own_tile(OwnState<ND>& st, const OwnTile<ND>& t, int key0, int lo, int hi, float scale, int lane) {
    constexpr int D = ND * 16, NK = (ND + 1) / 2;
    const int g = lane >> 4, first = key0 + 8 * g;
    f32x4 s[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        s[p] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) {
            SharedFrag k = t.k[p][ks];
            if (32 * ks + 32 > D && 32 * ks + 8 * g >= D) k.u = u32x4{0u, 0u, 0u, 0u};
            s[p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k.v, st.q[ks].v, s[p], 0, 0, 0);
        }
    }
    const bool edge = key0 < lo || key0 + 31 > hi;               // (the same for the whole wave)
    float x[8], mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = s[j >> 2][j & 3];
        if (edge) x[j] = first + j >= lo && first + j <= hi ? x[j] : -INFINITY;
        mx = fmaxf(mx, x[j]);
    }
    mx *= scale;
    if (__any(mx > st.m + 8.f)) {
        const float m_new = fmaxf(st.m, max_16_32(mx));
        const float corr = st.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m - m_new);
        st.m = m_new;
        st.l *= corr;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) st.o[dt] *= corr;
    }
    const float m = st.m == -INFINITY ? 0.f : st.m;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], scale, -m));
        sum += x[j];
    }
    st.l += sum;
    SharedFrag p;
    p.u = u32x4{f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]), f32x2_to_bf16x2(x[4], x[5]), f32x2_to_bf16x2(x[6], x[7])};
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) {
        SharedFrag v = t.v[dt];
        if (edge) v.u = only_between(v.u, first, lo, hi);
        st.o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v.v, p.v, st.o[dt], 0, 0, 0);
    }
}

// A block: one listed row, kv head, 16 of its queries and part of its own keys; four waves take tiles in turn and meet in LDS.
template <int ND, bool PAGED>
__global__ __launch_bounds__(SHARED_WAVES * WAVE, ND > 4 ? 2 : ND > 2 ? 3 : 4) void k_attn_own(SharedArgs a) {
    constexpr int D = ND * 16, NK = (ND + 1) / 2, STEP = 32 * SHARED_WAVES;
    __shared__ __attribute__((aligned(16))) float sums[SHARED_WAVES][ND * 4][WAVE];
    __shared__ float ms[SHARED_WAVES][16], ls[SHARED_WAVES][16];
    const int per = a.heads / a.kv_heads, lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int c = lane & 15, g = lane >> 4;
    const int part = blockIdx.x, kvh = blockIdx.y % a.kv_heads, first_query = blockIdx.y / a.kv_heads * 16, i = blockIdx.z;
    const int row = a.rows[i], t = a.seg_start[row];
    const int keys = shared_keys(a, group_of(a, i));
    const int pos = (int)min((long long)a.positions[t], ((long long)a.stride << a.page_shift) - 1);
    const int begin = (keys & ~31) + part * a.own_split;
    if (begin > pos || keys > pos) return;
    const int lo = max(max(begin, keys), first_seen(pos, a.window)), hi = min(begin + a.own_split - 1, pos);
    const int32_t* table = a.table + (size_t)row * a.stride;
    const bool valid = first_query + c < per;
    const int head = kvh * per + first_query + (valid ? c : 0);
    OwnState<ND> st;
    const bf16_t* qrow = a.q + ((size_t)t * a.heads + head) * D;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks)
        st.q[ks].u = query_piece(a, qrow + 32 * ks + 8 * g, valid && 32 * ks + 8 * g < D);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) st.o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    st.m = -INFINITY;
    st.l = 0.f;
    if (lo <= hi) {
        int key0 = (lo & ~31) + 32 * wave;
        OwnTile<ND> even, odd;
        TilePages<PAGED> pages;
        auto ask = [&](OwnTile<ND>& t, int key) __attribute__((always_inline)) {
            own_load<ND, PAGED>(t, a, pages, kvh, key, lane);
            pages.ask(a, table, key + STEP, lo, hi);
        };
        if (key0 <= hi) {
            pages.ask(a, table, key0, lo, hi);
            ask(even, key0);
        }
        while (key0 <= hi) {
            if (key0 + STEP <= hi) ask(odd, key0 + STEP);
            own_tile<ND>(st, even, key0, lo, hi, a.scale, lane);
            key0 += STEP;
            if (key0 > hi) break;
            if (key0 + STEP <= hi) ask(even, key0 + STEP);
            own_tile<ND>(st, odd, key0, lo, hi, a.scale, lane);
            key0 += STEP;
        }
    }
    st.l = sum_16_32(st.l);
    if (g == 0) {
        ms[wave][c] = st.m;
        ls[wave][c] = st.l;
    }
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[wave][4 * dt + r][lane] = st.o[dt][r];
    __syncthreads();
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < SHARED_WAVES; ++w) m = fmaxf(m, ms[w][c]);
    float f[SHARED_WAVES], l = 0.f;
#pragma unroll
    for (int w = 0; w < SHARED_WAVES; ++w) {
        f[w] = ms[w][c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[w][c] - m);
        l += ls[w][c] * f[w];
    }
    if (!valid) return;
    const size_t place = ((size_t)i * a.heads + head) * (a.n_pre + a.n_own) + a.n_pre + part;
    if (wave == 0 && g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * place) = make_float2(m, l);
    for (int dt = wave; dt < ND; dt += SHARED_WAVES) {            // a wave adds up and writes 16 dims: a lane four neighbours of them
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < SHARED_WAVES; ++w)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += f[w] > 0.f ? sums[w][4 * dt + r][lane] * f[w] : 0.f;
        *reinterpret_cast<float4*>(a.part_o + place * D + 16 * dt + 4 * g) = make_float4(v[0], v[1], v[2], v[3]);
    }
}

// A wave adds up the parts of one row's head: D / 4 lanes a part, several parts side by side, eight loads a lane in flight.
__global__ __launch_bounds__(WAVE) void k_attn_shared_merge(SharedArgs a, int head_dim) {
    constexpr int GROUP = 8;
    const int i = blockIdx.x / a.heads, head = blockIdx.x % a.heads, lane = threadIdx.x;
    const int lanes_a_part = head_dim / 4, side = WAVE / lanes_a_part;
    const int sub = lane / lanes_a_part, d = (lane % lanes_a_part) * 4;
    const bool works = sub < side;
    const int t = a.seg_start[a.rows[i]];
    const int end_all = (int)min((long long)a.positions[t] + 1, (long long)a.stride << a.page_shift);
    const int keys = shared_keys(a, group_of(a, i));
    const int pre = min((keys + a.pre_split - 1) / a.pre_split, a.n_pre);
    const int own = keys < end_all ? min((end_all - (keys & ~31) + a.own_split - 1) / a.own_split, a.n_own) : 0;
    const int n = pre + own;                                     // part k: of the shared keys, then of the row's own
    const size_t base = ((size_t)i * a.heads + head) * (a.n_pre + a.n_own);
    auto at = [&](int k) { return base + (k < pre ? k : a.n_pre + k - pre); };
    float top = -INFINITY;
    for (int k = lane; k < n; k += WAVE) top = fmaxf(top, a.part_ml[2 * at(k)]);
    top = wave_max(top);
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
    for (int k0 = 0; k0 < n; k0 += WAVE) {                       // lane j holds the weight of part k0 + j
        float w = 0.f;
        if (k0 + lane < n) {
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * at(k0 + lane));
            w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
            sum += w > 0.f ? ml.y * w : 0.f;
        }
        const int here = min(WAVE, n - k0);
        for (int j0 = 0; j0 < here; j0 += GROUP * side) {
            float4 v[GROUP];
#pragma unroll
            for (int j = 0; j < GROUP; ++j)
                v[j] = *reinterpret_cast<const float4*>(a.part_o + at(k0 + min(j0 + j * side + min(sub, side - 1), here - 1)) * head_dim + d);
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                const int k = j0 + j * side + sub;
                const float wk = __shfl(w, min(k, WAVE - 1), WAVE);
                const bool on = works && k < here && wk > 0.f;
                acc[0] += on ? v[j].x * wk : 0.f;
                acc[1] += on ? v[j].y * wk : 0.f;
                acc[2] += on ? v[j].z * wk : 0.f;
                acc[3] += on ? v[j].w * wk : 0.f;
            }
        }
    }
    sum = wave_sum(sum);
    float total[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < side; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) total[j] += __shfl(acc[j], lane % lanes_a_part + k * lanes_a_part, WAVE);
    if (sub != 0) return;
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;              // a row that sees nothing is zeros
    uint2 packed;
    packed.x = f32x2_to_bf16x2(total[0] * inv, total[1] * inv);
    packed.y = f32x2_to_bf16x2(total[2] * inv, total[3] * inv);
    *reinterpret_cast<uint2*>(a.out + ((size_t)t * a.heads + head) * head_dim + d) = packed;
}

struct SharedShape {
    int n_pre, pre_split, n_own, own_split, query_tiles, pre_tiles, own_tiles;
};
static int clamped(long long v, long long lo, long long hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }
// How the keys are cut: enough blocks for two a CU, parts of SHARED_MIN_SPLIT keys at least. Depends on sizes alone.
static SharedShape shared_shape(int n_rows, int heads, int kv_heads, int head_dim, int n_groups, int max_group, int max_shared, int max_own) {
    SharedShape s;
    const int per = heads / kv_heads;
    const long long queries = (long long)max_group * per;
    // queries of a block: 32 or 64 whose waves share out the keys, or with more than 64 queries four waves of 32 over the same keys
    s.query_tiles = queries > 64 ? 4 : queries > 32 && head_dim <= 64 ? 2 : 1;
    s.pre_tiles = max_shared > 0 && n_groups > 0 ? (int)((queries + 32 * s.query_tiles - 1) / (32 * s.query_tiles)) : 0;
    s.own_tiles = (per + 15) / 16;
    auto cut = [](long long blocks, long long units, int keys, int& n, int& split) {
        const int most = (keys + SHARED_MIN_SPLIT - 1) / SHARED_MIN_SPLIT;
        n = clamped(blocks / units, 1, most > 0 ? most : 1);
        split = ((keys + n - 1) / n + 127) & ~127;
        if (split < 128) split = 128;
        n = (keys + split - 1) / split;
    };
    if (s.pre_tiles) cut(512, (long long)n_groups * kv_heads * s.pre_tiles, max_shared, s.n_pre, s.pre_split);
    else s.n_pre = 0, s.pre_split = 128;
    // (own keys are counted from a multiple of 32, up to 31 below the first)
    if (max_own > 0) cut(8192, (long long)n_rows * kv_heads * s.own_tiles, max_own + 31, s.n_own, s.own_split);
    else s.n_own = 0, s.own_split = 128;
    return s;
}
static bool shared_sizes_bad(int n_rows, int heads, int kv_heads, int n_groups, int max_group, int max_shared, int max_own) {
    return n_rows < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || n_groups < 0 || max_group < 0 || max_shared < 0 || max_own < 0 ||
           max_shared > 1 << 30 || max_own > 1 << 30 || n_rows > 65535 || n_groups > 1 << 20 || max_group > 1 << 20 || heads > 1 << 16;
}

extern "C" int imparo_attention_shared_parts(int n_rows, int heads, int kv_heads, int head_dim, int n_groups, int max_group, int max_shared, int max_own) {
    if (shared_sizes_bad(n_rows, heads, kv_heads, n_groups, max_group, max_shared, max_own) || n_rows == 0) return 0;
    const SharedShape s = shared_shape(n_rows, heads, kv_heads, head_dim, n_groups, max_group, max_shared, max_own);
    return s.n_pre + s.n_own;
}

extern "C" int imparo_attention_decode_shared(const void* q, const void* k_cache, const void* v_cache, void* out, float* part_o,
                                              float* part_ml, int64_t part_o_floats, int64_t part_ml_floats, const int32_t* rows, int n_rows,
                                              const int32_t* group_start, int n_groups,
                                              const int32_t* shared, const int32_t* seg_start, const int32_t* positions,
                                              const int32_t* block_table, int table_stride, int page_size, int heads, int kv_heads,
                                              int head_dim, int n_pages, float scale, int window, int max_shared, int max_own,
                                              int max_group, imparo_stream stream) {
    if (!q || !k_cache || !v_cache || !out || !rows || !seg_start || !positions || !block_table ||
        shared_sizes_bad(n_rows, heads, kv_heads, n_groups, max_group, max_shared, max_own) || (n_groups && (!group_start || !shared)) ||
        table_stride <= 0 || page_size < 16 || page_size > 1 << 20 || (page_size & (page_size - 1)) || head_dim <= 0 || head_dim > 128 || head_dim % 16 ||
        n_pages <= 0 || window < 0)
        return IMPARO_BAD_ARGUMENT;
    if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)part_o) & 15 || ((uintptr_t)part_ml | (uintptr_t)out) & 7)
        return IMPARO_BAD_ARGUMENT;
    if (n_rows == 0) return IMPARO_OK;
    const SharedShape s = shared_shape(n_rows, heads, kv_heads, head_dim, n_groups, max_group, max_shared, max_own);
    const long long parts = (long long)n_rows * heads * (s.n_pre + s.n_own);
    if (parts && (!part_o || !part_ml)) return IMPARO_BAD_ARGUMENT;
    if (part_o_floats < parts * head_dim || part_ml_floats < parts * 2) return IMPARO_SCRATCH_TOO_SMALL;
    const long long units = (long long)n_groups * kv_heads * s.n_pre;
    const long long pre_blocks = (units + 7) / 8 * 8 * s.pre_tiles, own_blocks = (long long)n_rows * kv_heads * s.own_tiles * s.n_own;
    if (pre_blocks + own_blocks > 1 << 30 || kv_heads * s.own_tiles > 65535 || (long long)n_rows * heads > 1 << 30) return IMPARO_BAD_ARGUMENT;
    const SharedArgs a{(const bf16_t*)q, (const bf16_t*)k_cache, (const bf16_t*)v_cache, (bf16_t*)out, part_o, part_ml, rows, group_start, shared,
                       seg_start, positions, block_table, n_rows, n_groups, table_stride, __builtin_ctz((unsigned)page_size), heads, kv_heads,
                       n_pages, window, s.n_pre, s.pre_split, s.n_own, s.own_split, s.pre_tiles,
                       fmaxf(fabsf(scale) * 1.44269504088896340736f, 1.0e-37f), scale < 0.f ? 0x80008000u : 0u};
    hipStream_t st = (hipStream_t)stream;
    const int threads = SHARED_WAVES * WAVE;
    const dim3 own_grid(s.n_own, kv_heads * s.own_tiles, n_rows);
    // (a tile of 32 keys, or of 64, in one page: a thread's places in it are then always the same)
#define SHARED_GO(ND)                                                                                             \
    case ND:                                                                                                      \
        if (pre_blocks && s.query_tiles == 4) {                                                                   \
            if (page_size >= MANY_KEYS) k_attn_shared_many<ND, true><<<(int)pre_blocks, threads, 0, st>>>(a);     \
            else k_attn_shared_many<ND, false><<<(int)pre_blocks, threads, 0, st>>>(a);                           \
        } else if (pre_blocks) {                                                                                  \
            constexpr int MT = ND <= 4 ? 2 : 1;                                                                   \
            if (s.query_tiles == 2 && page_size >= 32) k_attn_shared<ND, MT, true><<<(int)pre_blocks, threads, 0, st>>>(a); \
            else if (s.query_tiles == 2) k_attn_shared<ND, MT, false><<<(int)pre_blocks, threads, 0, st>>>(a);    \
            else if (page_size >= 32) k_attn_shared<ND, 1, true><<<(int)pre_blocks, threads, 0, st>>>(a);         \
            else k_attn_shared<ND, 1, false><<<(int)pre_blocks, threads, 0, st>>>(a);                             \
        }                                                                                                         \
        if (s.n_own) {                                                                                            \
            if (page_size >= 32) k_attn_own<ND, true><<<own_grid, threads, 0, st>>>(a);                           \
            else k_attn_own<ND, false><<<own_grid, threads, 0, st>>>(a);                                          \
        }                                                                                                         \
        break;
    switch (head_dim / 16) {
        SHARED_GO(1) SHARED_GO(2) SHARED_GO(3) SHARED_GO(4) SHARED_GO(5) SHARED_GO(6) SHARED_GO(7) SHARED_GO(8)
    }
#undef SHARED_GO
    if (launch_status()) return IMPARO_LAUNCH_FAILED;
    k_attn_shared_merge<<<n_rows * heads, WAVE, 0, st>>>(a, head_dim);
    return launch_status();
}

int imparo_load_code_attention_shared() {
    hipFuncAttributes attributes;
    return hipFuncGetAttributes(&attributes, reinterpret_cast<const void*>(&k_attn_shared_merge)) == hipSuccess ? IMPARO_OK
                                                                                                    : IMPARO_LAUNCH_FAILED;
}
