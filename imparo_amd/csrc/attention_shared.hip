// Decode attention for rows in groups that share a prefix: the keys and values that all rows of a group have in the same pages are
// read once for all of them, the keys behind are each row's own.
//
// The result is the softmax over all keys a row sees, taken in parts: a part p of the keys leaves its reference m_p, l_p = sum 2^(s - m_p)
// and O_p = sum 2^(s - m_p) v (s: scaled scores times log2(e)), and with M = max m_p the output is sum 2^(m_p - M) O_p / sum 2^(m_p - M) l_p.
// One launch makes all parts: blocks for the groups' shared keys, whose queries are those of all rows of the group side by side (bound by the
// exponentials where they are many), and waves for each row's own keys (bound by memory), on the same CUs at the same time; a second launch adds the
// parts up.
//
// Both kinds keep a tile of keys in LDS: whole lines are loaded, neighbouring lanes neighbouring 16 bytes, which fragments for the matrix cores
// read straight from memory are not (16 lanes, 16 lines: 3.6 TB/s of own keys, where a plain read reaches 6). Rows in LDS are padded by 16 bytes, an odd
// number of 16-byte pieces, so that the operand reads of neighbouring rows fall on different banks. The next tile's loads are on their way in
// registers while one is multiplied, and its pages' numbers are there a tile earlier still.
//
// The products are arranged so that nothing moves between lanes:
//   S^T[key][query] = K Q^T         a lane ends up with scores of one query
//   O^T[dim][query] += V^T P^T      whose operand P^T wants eight consecutive keys of one query in a lane (the cache keeps V transposed in its pages)
// and which key a row of the first product stands for is free to choose, so that the scores a lane has are the ones it then needs: for
// 32x32x16, whose results are rows 8 (r / 4) + 4 h + r % 4 (h = lane / 32), row 16 u + 8 a + 4 h + t is key 16 u + 8 h + 4 a + t; for two products
// 16x16x32, row m of product p is key 8 (m / 4) + 4 p + m % 4.
#include "common.h"
#include "api.h"

#define SHARED_WAVES 4
#define SHARED_KEYS 64             // shared keys of a tile
#define SHARED_MIN_SPLIT 256       // and of a part at least, of so many keys that these make many parts
#define SHARED_FEW_SPLIT 128       // and else (448 keys in parts of 128 | 256: 10.7 | 11.7 us; 4,096: 19.9 | 18.3, with twice the parts to add up)
#define SHARED_SPLIT 1024          // and of a part where there is a block a CU
#define SHARED_BLOCKS 512          // blocks that shared keys are cut for at most, two a CU
#define OWN_KEYS 32                // a row's own keys of a tile
#define OWN_MIN_SPLIT 64           // and of a part at least
#define OWN_WAVES (12 * 256)       // waves that own keys are cut for, twelve a CU

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
union SharedFrag {
    u32x4 u;
    bf16x8 v;
};
__device__ __forceinline__ u32x4 load16(const bf16_t* p) { return *reinterpret_cast<const u32x4*>(p); }
// the same of lines that are read once and whole by one instruction: they need not stay in a cache
__device__ __forceinline__ u32x4 load16_once(const bf16_t* p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)); }
// a piece of values at keys key .. key + 7 with those outside [lo, hi] zeroed, whatever stands there
__device__ __forceinline__ u32x4 only_between(u32x4 v, int key, int lo, int hi) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = key + 2 * j;
        v[j] &= (k >= lo && k <= hi ? 0xFFFFu : 0u) | (k + 1 >= lo && k + 1 <= hi ? 0xFFFF0000u : 0u);
    }
    return v;
}

// Eight weights added up as they go into the product with the values, two an instruction: the denominator has the same roundings in it. (The
// instruction rounds a sum of three by up to 1.5e-7 of it, measured.)
__device__ __forceinline__ float weights_sum(u32x4 p) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 ones = {(__bf16)1.f, (__bf16)1.f};
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t two = p[j];                                // (a cast of the element itself takes the vector's first)
        sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), ones, sum, false);
    }
    return sum;
}

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
    int n_rows, n_groups, stride, page_shift, heads, kv_heads, per, n_pages, window;      // per: heads a kv head
    int n_pre, pre_split, n_own, own_split;      // parts and keys a part: of the shared keys, of a row's own
    int pre_tiles, own_tiles;                    // blocks' shares of a group's queries of a kv head, and 16 queries of a row's
    int pre_queries;                             // queries of a kv head that those blocks have room for
    int pre_blocks;                              // blocks for shared keys: the first ones
    float scale;                                 // its size, times log2(e)
    uint32_t flip;                               // its sign, for two bfloat16 of a query at once
};

// The group a listed row is in (its keys up to `shared` are the group's), or -1, and its first row. All lanes ask for the same row.
struct RowGroup {
    int g, first;
};
__device__ __forceinline__ RowGroup group_of(const SharedArgs& a, int i) {
    const int lane = threadIdx.x & (WAVE - 1);
    for (int g0 = 0; g0 < a.n_groups; g0 += WAVE) {
        const int g = g0 + lane, first = g < a.n_groups ? a.group_start[g] : INT32_MAX;
        const bool here = first <= i && i < a.group_start[min(g, a.n_groups - 1) + 1];
        const unsigned long long who = __ballot(here);
        if (who) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll((long long)who) - 1);
            return RowGroup{g0 + at, __builtin_amdgcn_readlane(first, at)};
        }
    }
    return RowGroup{-1, 0};
}
// 16 bytes of a query, its sign turned where the scale is negative: the largest score is then that of the largest product
__device__ __forceinline__ u32x4 query_piece(const SharedArgs& a, const bf16_t* q, bool valid) {
    return valid ? load16(q) ^ a.flip : u32x4{0u, 0u, 0u, 0u};
}
__device__ __forceinline__ int keys_of_table(const SharedArgs& a) { return (int)min((long long)a.stride << a.page_shift, (long long)INT32_MAX); }
// how many keys a group's rows share, inside what a table can name
__device__ __forceinline__ int shared_keys(const SharedArgs& a, int g) { return g < 0 ? 0 : min(max(a.shared[g], 0), keys_of_table(a)); }
// the page itself, whatever the table says
__device__ __forceinline__ size_t a_page(const SharedArgs& a, int page) { return (size_t)min(max(page, 0), a.n_pages - 1); }

// The reference of a query's exponentials moves only when a score passes it by 8 or more (a power of two of 8, harmless to float32 sums and to the
// rounding of the weights): most tiles then multiply no accumulator. Says whether this tile, with `mx` the largest score a lane has (of any
// of the lanes that share a query: `both` brings them together), moves it, and by what factor.
template <typename B>
__device__ __forceinline__ bool moved_reference(float& m, float mx, float& corr, B both) {
    if (!__any(mx > m + 8.f)) return false;
    const float m_new = fmaxf(m, both(mx));
    corr = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    return true;
}

// ---- shared keys
// A block's four waves take QW tiles of 32 queries and, for QW of 2, the two halves of a tile of keys. Bound by the exponentials with many queries (16 a lane
// for 32 keys, a quarter of a lane's rate each, beside 2 ND products), by memory with few. Weights are rounded to bfloat16 for the second product, half a
// step of 2^-8 each and of either sign, and summed as rounded, so that a key with nearly all the weight gives its value and not that off by half a step.
// 32 heads by 8 of 64, 64 rows behind 32,768 keys (256 queries a kv head): 45 to 47 us with the adding up of parts (3 more with the two halves of a tile
// one after the other), 380 TFLOP/s; 24 by 8 of 128, four groups of 16 rows behind 8,192 keys: 39 us without it, 3.3 TB/s, a tile's loads a block on
// their way. Not faster: the sums out of the matrix pipe (one more product a tile where the vector pipe waits as it is), two tiles on their way in
// registers (they did not fit), three blocks a CU (more parts to add up).
template <int ND, int QW, bool PAGED>
struct SharedBlock {
    static constexpr int D = ND * 16, DT = (ND + 1) / 2, THREADS = SHARED_WAVES * WAVE, KW = SHARED_WAVES / QW;
    static constexpr int LDK = D + 8, LDV = SHARED_KEYS + 8, CH = D / 8;           // CH: 16-byte pieces of a key
    static constexpr int K_PIECES = SHARED_KEYS * CH, V_PIECES = D * (SHARED_KEYS / 8);
    static constexpr int K_PER = (K_PIECES + THREADS - 1) / THREADS, V_PER = (V_PIECES + THREADS - 1) / THREADS;
    static constexpr int K_SIZE = SHARED_KEYS * LDK, V_SIZE = DT * 32 * LDV;       // (of one of two buffers, in elements)
    static constexpr int TILES = 2 * (K_SIZE + V_SIZE) * 2, MEETING = KW > 1 ? QW * (DT * 16 + 2) * WAVE * 4 : 0;
    static constexpr int LDS = TILES > MEETING ? TILES : MEETING;

    static __device__ __forceinline__ void run(const SharedArgs& a, char* lds, int b) {
        bf16_t* ks = reinterpret_cast<bf16_t*>(lds);
        bf16_t* vs = ks + 2 * K_SIZE;
        const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE), c = lane & 31, h = lane >> 5;
        const int qw = wave % QW, kw = wave / QW, per = a.per;
        // the blocks that read the same keys follow one another eight blocks apart: on one XCD, whose L2 has them
        const int block = (b / 8) % a.pre_tiles, unit = b / (8 * a.pre_tiles) * 8 + b % 8;
        const int part = unit % a.n_pre, kvh = unit / a.n_pre % a.kv_heads, g = unit / (a.n_pre * a.kv_heads);
        if (g >= a.n_groups) return;
        const int first_row = max(a.group_start[g], 0), n_queries = (min(a.group_start[g + 1], a.n_rows) - first_row) * per;
        const int keys = shared_keys(a, g), begin = part * a.pre_split, end = min(begin + a.pre_split, keys);
        if (block * 32 * QW >= n_queries || begin >= keys) return;
        const int32_t* __restrict__ table = a.table + (size_t)a.rows[first_row] * a.stride;

        const int x = (block * QW + qw) * 32 + c;
        const bool valid = x < n_queries;
        const int i = first_row + (valid ? x / per : 0), head = kvh * per + (valid ? x % per : 0);
        const int row = a.rows[i];

        // ---- tiles: which keys are read at all (under a window only known once the positions are)
        int lo_all = begin, hi_all = end - 1, lo = begin, hi = end - 1, t = 0;
        auto sees = [&]() __attribute__((always_inline)) {
            const int pos = a.positions[t];
            lo = max(begin, pos < 0 ? 0 : first_seen(pos, a.window));
            hi = min(end - 1, pos);
            if (!valid || lo > hi) lo = INT32_MAX, hi = -1;
        };
        if (a.window) {
            t = a.seg_start[row];
            sees();
            int* range = reinterpret_cast<int*>(lds);
            if (tid == 0) range[0] = INT32_MAX, range[1] = -1;
            __syncthreads();
            if (hi >= 0) {
                atomicMin(&range[0], lo);
                atomicMax(&range[1], hi);
            }
            __syncthreads();
            lo_all = __builtin_amdgcn_readfirstlane(range[0]), hi_all = __builtin_amdgcn_readfirstlane(range[1]);
            __syncthreads();
        }
        const int page_size = 1 << a.page_shift;
        const int v_key = 8 * (tid % (SHARED_KEYS / 8));
        u32x4 kr[K_PER], vr[V_PER];
        int k_page[PAGED ? 1 : K_PER], v_page = 0;
        // PAGED: a tile lies in one page, and a thread's places in it are always the same
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
        auto ask_tile = [&](int key0) __attribute__((always_inline)) {
            if constexpr (PAGED) {
                const size_t first = (a_page(a, __builtin_amdgcn_readfirstlane(k_page[0])) * a.kv_heads + kvh) << a.page_shift;
                const int slot = key0 & (page_size - 1);
                const bf16_t *k = a.k + (first + slot) * D, *v = a.v + first * D + slot;
#pragma unroll
                for (int j = 0; j < K_PER; ++j) kr[j] = load16(k + 8 * min(tid + j * THREADS, K_PIECES - 1));
#pragma unroll
                for (int j = 0; j < V_PER; ++j)
                    vr[j] = load16(v + ((min(tid + j * THREADS, V_PIECES - 1) / (SHARED_KEYS / 8) << a.page_shift) + v_key));
            } else {
#pragma unroll
                for (int j = 0; j < K_PER; ++j) {
                    const int piece = min(tid + j * THREADS, K_PIECES - 1), key = min(max(key0 + piece / CH, lo_all), hi_all);
                    kr[j] = load16(a.k + (((a_page(a, k_page[j]) * a.kv_heads + kvh) << a.page_shift) + (key & (page_size - 1))) * D + 8 * (piece % CH));
                }
                const size_t first = ((a_page(a, v_page) * a.kv_heads + kvh) << a.page_shift) * D;
                const int slot = min(max(key0 + v_key, lo_all & ~7), hi_all & ~7) & (page_size - 1);
#pragma unroll
                for (int j = 0; j < V_PER; ++j)
                    vr[j] = load16(a.v + first + ((min(tid + j * THREADS, V_PIECES - 1) / (SHARED_KEYS / 8) << a.page_shift) + slot));
            }
        };
        auto keep_tile = [&](int key0, int buf) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < K_PER; ++j) {
                const int piece = tid + j * THREADS;
                if (K_PIECES % THREADS == 0 || piece < K_PIECES)
                    *reinterpret_cast<u32x4*>(ks + buf * K_SIZE + piece / CH * LDK + 8 * (piece % CH)) = kr[j];
            }
            if (key0 < lo_all || key0 + SHARED_KEYS - 1 > hi_all) {               // values that no query reads may be anything: zeros
#pragma unroll
                for (int j = 0; j < V_PER; ++j) vr[j] = only_between(vr[j], key0 + v_key, lo_all, hi_all);
            }
#pragma unroll
            for (int j = 0; j < V_PER; ++j) {
                const int piece = tid + j * THREADS;
                if (V_PIECES % THREADS == 0 || piece < V_PIECES)
                    *reinterpret_cast<u32x4*>(vs + buf * V_SIZE + piece / (SHARED_KEYS / 8) * LDV + v_key) = vr[j];
            }
        };
        const bool any = lo_all <= hi_all;
        int key0 = lo_all & ~(SHARED_KEYS - 1), buf = 0;
        if (any) ask_pages(key0);
        if (!a.window) t = a.seg_start[row];
        if (any) {
            ask_tile(key0);
            ask_pages(key0 + SHARED_KEYS);
        }
        // ---- this wave's queries
        if (!a.window) sees();
        SharedFrag q[ND];
        const bf16_t* qrow = a.q + ((size_t)t * a.heads + head) * D + 8 * h;
#pragma unroll
        for (int k = 0; k < ND; ++k) q[k].u = query_piece(a, qrow + 16 * k, valid);
        f32x16 o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
        float m = -INFINITY, l = 0.f;                             // (the reference is one for both halves of the wave, the sum a lane's own)
        if (any) {
            keep_tile(key0, 0);
            ask_tile(key0 + SHARED_KEYS);
            ask_pages(key0 + 2 * SHARED_KEYS);
            __syncthreads();
            for (; key0 <= hi_all; key0 += SHARED_KEYS, buf ^= 1) {
                // this wave's keys of the tile: all 64, or its half of them
                constexpr int N = SHARED_KEYS / 32 / KW;
                const int at = KW > 1 ? 32 * kw : 0, key = key0 + at;
                if (__any(key <= hi && key + 32 * N - 1 >= lo)) {
                    f32x16 s[N];
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        const bf16_t* krow = ks + buf * K_SIZE + (at + 32 * n + ((c & 16) | (c & 4) << 1 | (c & 8) >> 1 | (c & 3))) * LDK + 8 * h;
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[n][r] = 0.f;
#pragma unroll
                        for (int k = 0; k < ND; ++k) {
                            SharedFrag f;
                            f.u = load16(krow + 16 * k);
                            s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.v, q[k].v, s[n], 0, 0, 0);
                        }
                    }
                    if (__any(valid && (key < lo || key + 32 * N - 1 > hi))) {
#pragma unroll
                        for (int n = 0; n < N; ++n)
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                const int one = key + 32 * n + 16 * (r >> 3) + 8 * h + (r & 7);
                                s[n][r] = one >= lo && one <= hi ? s[n][r] : -INFINITY;
                            }
                    }
                    float mx = -INFINITY;
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int r = 0; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[n][r]), s[n][r + 1]);
                    float corr;
                    if (moved_reference(m, mx * a.scale, corr, [](float v) { return fmaxf(v, lane_xor<32>(v)); })) {
                        l *= corr;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[dt][r] *= corr;
                    }
                    const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
                    for (int n = 0; n < N; ++n) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[n][r] = __builtin_amdgcn_exp2f(fmaf(s[n][r], a.scale, -from));
                        SharedFrag p[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            p[u].u = u32x4{f32x2_to_bf16x2(s[n][8 * u], s[n][8 * u + 1]), f32x2_to_bf16x2(s[n][8 * u + 2], s[n][8 * u + 3]),
                                           f32x2_to_bf16x2(s[n][8 * u + 4], s[n][8 * u + 5]), f32x2_to_bf16x2(s[n][8 * u + 6], s[n][8 * u + 7])};
                        l += weights_sum(p[0].u) + weights_sum(p[1].u);
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                SharedFrag f;                     // (rows past the head: whatever stands there, never written out)
                                f.u = load16(vs + buf * V_SIZE + (32 * dt + c) * LDV + at + 32 * n + 16 * u + 8 * h);
                                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.v, p[u].v, o[dt], 0, 0, 0);
                            }
                    }
                }
                if (key0 + SHARED_KEYS <= hi_all) {
                    keep_tile(key0 + SHARED_KEYS, buf ^ 1);
                    ask_tile(key0 + 2 * SHARED_KEYS);
                    ask_pages(key0 + 3 * SHARED_KEYS);
                }
                __syncthreads();
            }
        }
        l += lane_xor<32>(l);
        // A value that is infinite or NaN at a key that a query does not see (it lies further back, or ahead of its window) goes into the product
        // with a weight of 0, and makes NaN of the query's sums all the same. That is noticed here, and the sums of such a query are made anew, key by
        // key, out of those that it sees; a query that sees all of the part has its sums from the product, whatever they are. To notice takes 0.3 us of a
        // call of 10 (to look at the values as they are read takes registers that the loop has not got); to make sums anew about a microsecond a key of 64,
        // so that a call under a window that cuts a part of 256 | 1,024 keys takes 0.26 | 2.5 ms while there is such a value in that part
        float zeros = 0.f;                                        // (0 as long as all are finite)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (32 * dt + 8 * (r >> 2) < D) zeros += o[dt][r] * 0.f;
        if (__builtin_expect(valid && (lo > lo_all || hi < hi_all) && zeros != 0.f && fabsf(l) < INFINITY, 0)) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
            const float from = m == -INFINITY ? 0.f : m;
            const bf16_t* one_q = a.q + ((size_t)t * a.heads + head) * D;
            l = 0.f;
            for (int key = lo; key <= hi; ++key) {
                if (KW > 1 && (key >> 5 & 1) != kw) continue;
                const size_t first = ((a_page(a, table[key >> a.page_shift]) * a.kv_heads + kvh) << a.page_shift) * D;
                const int slot = key & (page_size - 1);
                float dot = 0.f;
#pragma unroll 1
                for (int d = 0; d < D; d += 4) {
                    const u32x2 qd = *reinterpret_cast<const u32x2*>(one_q + d), kd = *reinterpret_cast<const u32x2*>(a.k + first + slot * D + d);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        dot = fmaf(__uint_as_float(qd[e] << 16), __uint_as_float(kd[e] << 16), dot);
                        dot = fmaf(__uint_as_float(qd[e] & 0xFFFF0000u), __uint_as_float(kd[e] & 0xFFFF0000u), dot);
                    }
                }
                const bf16_t* values = a.v + first + slot;        // (a page has at most 2^27 elements a kv head)
                const float p = bf16_to_f32(f32_to_bf16(__builtin_amdgcn_exp2f(fmaf(a.flip ? -dot : dot, a.scale, -from))));
                l += p;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int d = 32 * dt + 8 * (r >> 2);
                        if (d < D) o[dt][r] = fmaf(p, bf16_to_f32(values[(d + 4 * h + (r & 3)) << a.page_shift]), o[dt][r]);
                        if ((r & 3) == 3) __builtin_amdgcn_sched_barrier(0);      // (four loads on their way: all of them take registers that the loop above is in need of)
                    }
            }
        }
        if constexpr (KW > 1) {                                   // the waves of the second halves hand over to those of the first
            float* meet = reinterpret_cast<float*>(lds) + qw * (DT * 16 + 2) * WAVE + lane;
            __syncthreads();
            if (kw == 1) {
                meet[0] = m;
                meet[WAVE] = l;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) meet[(2 + dt * 16 + r) * WAVE] = o[dt][r];
            }
            __syncthreads();
            if (kw == 1) return;
            const float m_other = meet[0], top = fmaxf(m, m_other);
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top), f_other = m_other == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_other - top);
            l = l * f + meet[WAVE] * f_other;
            m = top;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] = o[dt][r] * f + meet[(2 + dt * 16 + r) * WAVE] * f_other;
        }
        if (!valid) return;
        const size_t place = ((size_t)i * a.heads + head) * (a.n_pre + a.n_own) + part;
        if (h == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * place) = make_float2(m, l);
        float* out = a.part_o + place * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 32 * dt + 8 * r + 4 * h;
                if (d < D) *reinterpret_cast<f32x4*>(out + d) = f32x4{o[dt][4 * r], o[dt][4 * r + 1], o[dt][4 * r + 2], o[dt][4 * r + 3]};
            }
    }
};

// ---- a row's own keys
// A wave by itself, with a tile of its own in LDS: one listed row, kv head, 16 of its queries (the heads of the kv head) and a part of the row's own keys.
// Bound by memory; what a wave has to find out before its first key (four trips to memory one behind the other) weighs on every part, so parts are long
// where there are waves enough. Keys go past the caches, whose lines they would only push out (a tile's keys are whole lines; its values are half
// lines, whose other half the next tile wants): 256 rows with 1,024 keys each on average, 8 kv heads of 64, 145 us through the caches, 122 so,
// 4.4 TB/s, and 6 with rows of one length; the rest is the longest rows' end. Tiles of 64 keys (whole lines of values too) take the LDS that the
// blocks of shared keys need: 115 us alone, but 64 rows behind 32,768 shared keys 48 -> 66.
template <int ND, bool PAGED>
struct OwnWave {
    static constexpr int D = ND * 16, NK = (ND + 1) / 2, LDK = D + 8, LDV = OWN_KEYS + 8, CH = D / 8;
    static constexpr int K_SIZE = OWN_KEYS * LDK, LDS = (K_SIZE + D * LDV) * 2;    // (in bytes)

    static __device__ __forceinline__ void run(const SharedArgs& a, char* lds, int unit) {
        const int lane = threadIdx.x & (WAVE - 1), c = lane & 15, g = lane >> 4, per = a.per;
        bf16_t* ks = reinterpret_cast<bf16_t*>(lds + threadIdx.x / WAVE * LDS);
        bf16_t* vs = ks + K_SIZE;
        // kv heads first: neighbouring waves find out the same
        const int kvh = unit % a.kv_heads, part = unit / a.kv_heads % a.n_own, rest = unit / (a.kv_heads * a.n_own);
        const int first_query = rest % a.own_tiles * 16, i = rest / a.own_tiles;
        if (i >= a.n_rows) return;
        const int row = a.rows[i], keys = shared_keys(a, group_of(a, i).g), t = a.seg_start[row];
        const int32_t* __restrict__ table = a.table + (size_t)row * a.stride;
        const int begin = (keys & ~(OWN_KEYS - 1)) + part * a.own_split;
        const int pos = min(a.positions[t], keys_of_table(a) - 1);
        if (begin > pos || keys > pos) return;
        const int lo = max(max(begin, keys), first_seen(pos, a.window)), hi = min(begin + a.own_split - 1, pos);
        const bool valid = first_query + c < per;
        const int head = kvh * per + first_query + (valid ? c : 0);
        const bf16_t* qrow = a.q + ((size_t)t * a.heads + head) * D;
        u32x4 kr[ND], vr[ND];
        int page[PAGED ? 1 : 2];
        auto ask_pages = [&](int key0) __attribute__((always_inline)) {           // (of a tile's first 16 keys, and of the others)
#pragma unroll
            for (int u = 0; u < (PAGED ? 1 : 2); ++u) page[u] = table[min(max(key0 + 16 * u, lo & ~15), hi & ~15) >> a.page_shift];
        };
        auto ask_tile = [&](int key0) __attribute__((always_inline)) {
            const int mask = (1 << a.page_shift) - 1;
            if constexpr (PAGED) {
                const size_t first = (a_page(a, __builtin_amdgcn_readfirstlane(page[0])) * a.kv_heads + kvh) << a.page_shift;
                const bf16_t *k = a.k + (first + (key0 & mask)) * D, *v = a.v + first * D + (key0 & mask);
#pragma unroll
                for (int j = 0; j < ND; ++j) kr[j] = load16_once(k + 8 * (lane + j * WAVE));
#pragma unroll
                for (int j = 0; j < ND; ++j) vr[j] = load16(v + (((lane + j * WAVE) / 4 << a.page_shift) + 8 * (lane & 3)));
            } else {
                const size_t first0 = ((a_page(a, __builtin_amdgcn_readfirstlane(page[0])) * a.kv_heads + kvh) << a.page_shift) * D;
                const size_t first1 = ((a_page(a, __builtin_amdgcn_readfirstlane(page[1])) * a.kv_heads + kvh) << a.page_shift) * D;
                const bf16_t *k0 = a.k + first0 + (key0 & mask) * D, *k1 = a.k + first1 + (((key0 + 16) & mask) - 16) * D;
                const bf16_t* v = lane & 2 ? a.v + first1 + ((key0 + 16) & mask) : a.v + first0 + (key0 & mask);
#pragma unroll
                for (int j = 0; j < ND; ++j) kr[j] = load16((lane + j * WAVE < 16 * CH ? k0 : k1) + 8 * (lane + j * WAVE));
#pragma unroll
                for (int j = 0; j < ND; ++j) vr[j] = load16(v + (((lane + j * WAVE) / 4 << a.page_shift) + 8 * (lane & 1)));
            }
        };
        if (lo <= hi) ask_pages(lo & ~(OWN_KEYS - 1));
        SharedFrag q[NK];
#pragma unroll
        for (int k = 0; k < NK; ++k) q[k].u = query_piece(a, qrow + 32 * k + 8 * g, valid && 32 * k + 8 * g < D);
        f32x4 o[ND];
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        if (lo <= hi) {
            int key0 = lo & ~(OWN_KEYS - 1);
            ask_tile(key0);
            ask_pages(key0 + OWN_KEYS);
            for (; key0 <= hi; key0 += OWN_KEYS) {
                const bool edge = key0 < lo || key0 + OWN_KEYS - 1 > hi;          // (the same for the whole wave)
                if (edge) {                                                       // values that no query reads may be anything: zeros
#pragma unroll
                    for (int j = 0; j < ND; ++j) vr[j] = only_between(vr[j], key0 + 8 * (lane & 3), lo, hi);
                }
#pragma unroll
                for (int j = 0; j < ND; ++j) {
                    const int piece = lane + j * WAVE;
                    *reinterpret_cast<u32x4*>(ks + piece / CH * LDK + 8 * (piece % CH)) = kr[j];
                    *reinterpret_cast<u32x4*>(vs + piece / 4 * LDV + 8 * (lane & 3)) = vr[j];
                }
                wave_lds_sync();
                if (key0 + OWN_KEYS <= hi) {
                    ask_tile(key0 + OWN_KEYS);
                    ask_pages(key0 + 2 * OWN_KEYS);
                }
                const int first = key0 + 8 * g;
                float s[8], mx = -INFINITY;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    f32x4 four = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < NK; ++k) {
                        SharedFrag f;                             // (dims past the head: its last 8 again, against zeros of the query)
                        f.u = load16(ks + (8 * (c >> 2) + 4 * p + (c & 3)) * LDK + min(32 * k + 8 * g, D - 8));
                        if (32 * k + 32 > D && 32 * k + 8 * g >= D) f.u = u32x4{0u, 0u, 0u, 0u};
                        four = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.v, q[k].v, four, 0, 0, 0);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int one = first + 4 * p + j;
                        s[4 * p + j] = !edge || (one >= lo && one <= hi) ? four[j] : -INFINITY;
                        mx = fmaxf(mx, s[4 * p + j]);
                    }
                }
                float corr;
                if (moved_reference(m, mx * a.scale, corr, [](float v) { return max_16_32(v); })) {
                    l *= corr;
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt) o[dt] *= corr;
                }
                const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] = __builtin_amdgcn_exp2f(fmaf(s[j], a.scale, -from));
                SharedFrag p;
                p.u = u32x4{f32x2_to_bf16x2(s[0], s[1]), f32x2_to_bf16x2(s[2], s[3]), f32x2_to_bf16x2(s[4], s[5]), f32x2_to_bf16x2(s[6], s[7])};
                l += weights_sum(p.u);
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) {
                    SharedFrag f;
                    f.u = load16(vs + (16 * dt + c) * LDV + 8 * g);
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.v, p.v, o[dt], 0, 0, 0);
                }
                wave_lds_sync();
            }
        }
        l = sum_16_32(l);
        if (!valid) return;
        const size_t place = ((size_t)i * a.heads + head) * (a.n_pre + a.n_own) + a.n_pre + part;
        if (g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * place) = make_float2(m, l);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) *reinterpret_cast<f32x4*>(a.part_o + place * D + 16 * dt + 4 * g) = o[dt];
    }
};

template <int ND, int QW, bool PAGED>
__global__ __launch_bounds__(SHARED_WAVES * WAVE, ND > 4 ? 2 : ND > 2 ? 3 : 4) void k_attn_shared(SharedArgs a) {
    typedef SharedBlock<ND, QW, PAGED> Block;
    typedef OwnWave<ND, PAGED> Own;
    __shared__ __attribute__((aligned(16))) char lds[Block::LDS > SHARED_WAVES * Own::LDS ? Block::LDS : SHARED_WAVES * Own::LDS];
    const int b = blockIdx.x;
    if (b < a.pre_blocks) Block::run(a, lds, b);
    else Own::run(a, lds, __builtin_amdgcn_readfirstlane((b - a.pre_blocks) * SHARED_WAVES + (int)threadIdx.x / WAVE));
}

// A wave adds up the parts of one row's head: D / 4 lanes a part, several parts side by side, eight loads a lane in flight. References and sums of
// all parts, and the values of the first ones, are asked for before it is known which of them there are.
__global__ __launch_bounds__(SHARED_WAVES * WAVE) void k_attn_shared_merge(SharedArgs a, int head_dim) {
    constexpr int GROUP = 8;
    const int unit = __builtin_amdgcn_readfirstlane(blockIdx.x * SHARED_WAVES + threadIdx.x / WAVE), lane = threadIdx.x & (WAVE - 1);
    const int i = unit / a.heads, head = unit % a.heads;
    if (i >= a.n_rows) return;
    const int lanes_a_part = head_dim / 4, side = WAVE / lanes_a_part;
    const int sub = lane / lanes_a_part, d = (lane % lanes_a_part) * 4, parts = a.n_pre + a.n_own;
    const bool works = sub < side;
    const size_t base = (size_t)unit * parts;
    const int row = a.rows[i];
    float2 ml = make_float2(-INFINITY, 0.f);
    f32x4 v[GROUP];
    if (lane < parts) ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (base + lane));
    auto ask = [&](int j0, int n) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < GROUP; ++j)
            v[j] = *reinterpret_cast<const f32x4*>(a.part_o + (base + min(j0 + j * side + min(sub, side - 1), n - 1)) * head_dim + d);
    };
    if (parts) ask(0, parts);
    const int t = a.seg_start[row];
    const RowGroup group = group_of(a, i);
    const int keys = shared_keys(a, group.g);
    const int end_all = (int)min((long long)a.positions[t] + 1, (long long)keys_of_table(a));
    const int pre = min((keys + a.pre_split - 1) / a.pre_split, a.n_pre);
    const int own = keys < end_all ? min((end_all - (keys & ~(OWN_KEYS - 1)) + a.own_split - 1) / a.own_split, a.n_own) : 0;
    // Keys that the launch was not shaped for (a bound of the call's that does not hold for what stands on the device): no block or wave took them, and
    // what stands in place of their parts is another call's. Such a row is NaN
    const bool lost = min(keys, end_all) > a.n_pre * a.pre_split || (keys < end_all && end_all - (keys & ~(OWN_KEYS - 1)) > a.n_own * a.own_split) ||
                      (keys > 0 && (long long)(i + 1 - max(group.first, 0)) * a.per > a.pre_queries);
    auto there = [&](int k) { return k < pre || (k >= a.n_pre && k < a.n_pre + own); };
    // A part in which the row sees nothing is -inf, 0 and zeros; one whose scores are all NaN has no reference either, but a NaN for a sum, and weighs
    // NaN. What a part holds counts even where its weight vanishes beside the others': NaN times 0 is NaN.
    float top = there(lane) ? ml.x : -INFINITY;
    for (int k = lane + WAVE; k < parts; k += WAVE) top = fmaxf(top, there(k) ? a.part_ml[2 * (base + k)] : -INFINITY);
    top = wave_max(top);
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
    for (int k0 = 0; k0 < parts; k0 += WAVE) {                   // lane j holds the weight of part k0 + j
        float w = -1.f;                                           // (no such part: scratch that nobody wrote)
        if (there(k0 + lane)) {
            if (k0) ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (base + k0 + lane));
            w = ml.x == -INFINITY ? ml.y : __builtin_amdgcn_exp2f(ml.x - top);
            sum += ml.y * w;
        }
        const int here = min(WAVE, parts - k0);
        for (int j0 = 0; j0 < here; j0 += GROUP * side) {
            if (k0 + j0) ask(k0 + j0, parts);
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                const int k = j0 + j * side + sub;
                const float wk = __shfl(w, min(k, WAVE - 1), WAVE);
                const bool on = works && k < here && !(wk < 0.f);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] += on ? v[j][e] * wk : 0.f;
            }
        }
    }
    sum = wave_sum(sum);
    float total[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < side; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) total[j] += __shfl(acc[j], lane % lanes_a_part + k * lanes_a_part, WAVE);
    if (sub != 0) return;
    const float inv = lost ? __builtin_nanf("") : sum == 0.f ? 0.f : 1.0f / sum;      // (a row that sees nothing is zeros)
    uint2 packed;
    packed.x = f32x2_to_bf16x2(total[0] * inv, total[1] * inv);
    packed.y = f32x2_to_bf16x2(total[2] * inv, total[3] * inv);
    *reinterpret_cast<uint2*>(a.out + ((size_t)t * a.heads + head) * head_dim + d) = packed;
}

struct SharedShape {
    int n_pre, pre_split, n_own, own_split, query_waves, pre_tiles, own_tiles;
};
static int clamped(long long v, long long lo, long long hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }
// How the keys are cut: for so many blocks or waves as fill the chip, and parts of so many keys at least. Depends on sizes alone.
static SharedShape shared_shape(int n_rows, int heads, int kv_heads, int n_groups, int max_group, int max_shared, int max_own) {
    SharedShape s;
    const int per = heads / kv_heads;
    const long long queries = (long long)max_group * per;
    s.query_waves = queries > 64 ? 4 : 2;
    s.pre_tiles = max_shared > 0 && n_groups > 0 ? (int)((queries + 32 * s.query_waves - 1) / (32 * s.query_waves)) : 0;
    s.own_tiles = (per + 15) / 16;
    auto cut = [](long long pieces, int keys, int least, int step, int& n, int& split) {
        n = clamped(pieces, 1, (keys + least - 1) / least);
        split = ((keys + n - 1) / n + step - 1) / step * step;
        n = (keys + split - 1) / split;
    };
    s.n_pre = s.n_own = 0, s.pre_split = SHARED_KEYS, s.own_split = OWN_KEYS;
    if (s.pre_tiles) {
        // a part costs its results' way to memory and back: from a block a CU on parts are long ones (4,096 keys of 1,024 queries a kv head in parts of
        // 512, 1,024: 151, 134 us beside the own keys; 32,768 keys of 256 queries in parts of 1,024, 2,048: 48, 54)
        const long long units = (long long)n_groups * kv_heads * s.pre_tiles, few = SHARED_BLOCKS / 2 / units, most = SHARED_BLOCKS / units;
        cut(clamped(max_shared / SHARED_SPLIT, few, most), max_shared, max_shared > 8 * SHARED_MIN_SPLIT ? SHARED_MIN_SPLIT : SHARED_FEW_SPLIT, SHARED_KEYS, s.n_pre, s.pre_split);
    }
    // (own keys are counted from a multiple of OWN_KEYS, up to one less below the first)
    if (max_own > 0) cut(OWN_WAVES / ((long long)n_rows * kv_heads * s.own_tiles), max_own + OWN_KEYS - 1, OWN_MIN_SPLIT, OWN_KEYS, s.n_own, s.own_split);
    return s;
}
static bool shared_sizes_bad(int n_rows, int heads, int kv_heads, int n_groups, int max_group, int max_shared, int max_own) {
    return n_rows < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || n_groups < 0 || max_group < 0 || max_shared < 0 || max_own < 0 ||
           max_shared > 1 << 30 || max_own > 1 << 30 || n_rows > 65535 || n_groups > 1 << 20 || max_group > 1 << 20 || heads > 1 << 16 ||
           (long long)max_group * (heads / kv_heads) > 1 << 30;             // (queries of a kv head are numbered in 32 bits)
}

extern "C" int imparo_attention_shared_parts(int n_rows, int heads, int kv_heads, int n_groups, int max_group, int max_shared, int max_own) {
    if (shared_sizes_bad(n_rows, heads, kv_heads, n_groups, max_group, max_shared, max_own) || n_rows == 0) return 0;
    const SharedShape s = shared_shape(n_rows, heads, kv_heads, n_groups, max_group, max_shared, max_own);
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
        n_pages <= 0 || window < 0 || !(fabsf(scale) * 1.44269504088896340736f < INFINITY))
        return IMPARO_BAD_ARGUMENT;
    if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)part_o) & 15 || ((uintptr_t)part_ml | (uintptr_t)out) & 7)
        return IMPARO_BAD_ARGUMENT;
    if (n_rows == 0) return IMPARO_OK;
    const SharedShape s = shared_shape(n_rows, heads, kv_heads, n_groups, max_group, max_shared, max_own);
    const long long parts = (long long)n_rows * heads * (s.n_pre + s.n_own);
    if (parts && (!part_o || !part_ml)) return IMPARO_BAD_ARGUMENT;
    if (part_o_floats < parts * head_dim || part_ml_floats < parts * 2) return IMPARO_SCRATCH_TOO_SMALL;
    const long long units = (long long)n_groups * kv_heads * s.n_pre, own_waves = (long long)n_rows * kv_heads * s.own_tiles * s.n_own;
    const long long pre_blocks = (units + 7) / 8 * 8 * s.pre_tiles, blocks = pre_blocks + (own_waves + SHARED_WAVES - 1) / SHARED_WAVES;
    if (blocks > 1 << 30 || own_waves > 1 << 30 || (long long)n_rows * heads > 1 << 30) return IMPARO_BAD_ARGUMENT;
    const SharedArgs a{(const bf16_t*)q, (const bf16_t*)k_cache, (const bf16_t*)v_cache, (bf16_t*)out, part_o, part_ml, rows, group_start, shared,
                       seg_start, positions, block_table, n_rows, n_groups, table_stride, __builtin_ctz((unsigned)page_size), heads, kv_heads,
                       heads / kv_heads, n_pages, window, s.n_pre, s.pre_split, s.n_own, s.own_split, s.pre_tiles, s.own_tiles, s.pre_tiles * 32 * s.query_waves, (int)pre_blocks,
                       fmaxf(fabsf(scale) * 1.44269504088896340736f, 1.0e-37f), scale < 0.f ? 0x80008000u : 0u};
    hipStream_t st = (hipStream_t)stream;
    if (blocks) {
        // (pages of a tile or more: a thread's places in a tile are then always the same)
        const int kind = (s.query_waves == 4 ? 2 : 0) + (page_size >= SHARED_KEYS);
#define SHARED_GO(ND)                                                                                                     \
    case ND:                                                                                                              \
        if (kind == 0) k_attn_shared<ND, 2, false><<<(int)blocks, SHARED_WAVES * WAVE, 0, st>>>(a);                       \
        else if (kind == 1) k_attn_shared<ND, 2, true><<<(int)blocks, SHARED_WAVES * WAVE, 0, st>>>(a);                   \
        else if (kind == 2) k_attn_shared<ND, 4, false><<<(int)blocks, SHARED_WAVES * WAVE, 0, st>>>(a);                  \
        else k_attn_shared<ND, 4, true><<<(int)blocks, SHARED_WAVES * WAVE, 0, st>>>(a);                                  \
        break;
        switch (head_dim / 16) {
            SHARED_GO(1) SHARED_GO(2) SHARED_GO(3) SHARED_GO(4) SHARED_GO(5) SHARED_GO(6) SHARED_GO(7) SHARED_GO(8)
        }
#undef SHARED_GO
        if (launch_status()) return IMPARO_LAUNCH_FAILED;
    }
    k_attn_shared_merge<<<(n_rows * heads + SHARED_WAVES - 1) / SHARED_WAVES, SHARED_WAVES * WAVE, 0, st>>>(a, head_dim);
    return launch_status();
}

int imparo_load_code_attention_shared() {
    hipFuncAttributes attributes;
    return hipFuncGetAttributes(&attributes, reinterpret_cast<const void*>(&k_attn_shared_merge)) == hipSuccess ? IMPARO_OK
                                                                                                    : IMPARO_LAUNCH_FAILED;
}
