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
union SharedFrag {
    uint4 u;
    bf16x8 v;
    bf16_t h[8];
};

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
    int pre_tiles, own_tiles;                    // tiles of queries a group's kv head has at most, and a row's
    int pre_blocks;                              // blocks for shared keys: the first ones
    float scale;                                 // times log2(e)
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

// Asks for the tile of keys key0 .. key0 + 31; [lo, hi] are the keys that any query reads: pages are looked up inside it only.
// A page holds 16 keys or more, so a tile lies in one page or two.
template <int ND>
__device__ __forceinline__ void shared_load(SharedTile<ND>& t, const SharedArgs& a, const int32_t* __restrict__ table, int kvh,
                                            int key0, int lo, int hi, int lane) {
    constexpr int D = ND * 16, DT = (ND + 1) / 2;
    const int page_size = 1 << a.page_shift, c = lane & 31, h = lane >> 5;
    size_t head[2];
    int slot[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int key = min(max(key0 + 16 * u, lo & ~15), hi & ~15);
        const int page = min(max(table[key >> a.page_shift], 0), a.n_pages - 1);
        head[u] = ((size_t)page * a.kv_heads + kvh) * D;
        slot[u] = key & (page_size - 1);
    }
    const int key = (c & 16) | (c & 4) << 1 | (c & 8) >> 1 | (c & 3);
    const bf16_t* krow = a.k + (key & 16 ? head[1] : head[0]) * page_size + (size_t)((key & 16 ? slot[1] : slot[0]) + (key & 15)) * D + 8 * h;
#pragma unroll
    for (int ks = 0; ks < ND; ++ks) t.k[ks].u = *reinterpret_cast<const uint4*>(krow + 16 * ks);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        const int d = min(32 * dt + c, D - 1);               // (dims past the head: the last again, never written out)
#pragma unroll
        for (int u = 0; u < 2; ++u)
            t.v[u][dt].u = *reinterpret_cast<const uint4*>(a.v + (head[u] + d) * page_size + slot[u] + 8 * h);
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
                s[r] = key >= st.lo[mt] && key <= st.hi[mt] ? s[r] * scale : -INFINITY;
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= scale;
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
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
            s[r] = __builtin_amdgcn_exp2f(s[r] - m);
            sum += s[r];
        }
        st.l[mt] += sum;
#pragma unroll
        for (int u = 0; u < 2; ++u)
            p[mt][u].u = make_uint4(f32x2_to_bf16x2(s[8 * u], s[8 * u + 1]), f32x2_to_bf16x2(s[8 * u + 2], s[8 * u + 3]),
                                    f32x2_to_bf16x2(s[8 * u + 4], s[8 * u + 5]), f32x2_to_bf16x2(s[8 * u + 6], s[8 * u + 7]));
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            SharedFrag a = t.v[u][dt];
            if (EDGE) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = key0 + 16 * u + 8 * h + j;
                    if (key < lo || key > hi) a.h[j] = 0;
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                st.o[mt][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, p[mt][u].v, st.o[mt][dt], 0, 0, 0);
        }
}

// One block's part: the queries `first_query` .. of the rows from `first_row` on (query x is row x / per, head x % per of the kv head), over the
// keys [begin, end) of the table, each query inside what it sees; the four waves take tiles in turn, meet in LDS, and leave one part.
template <int ND, int MT>
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
            st.q[mt][ks].u = valid ? *reinterpret_cast<const uint4*>(qrow + 16 * ks) : make_uint4(0u, 0u, 0u, 0u);
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
        if (key0 <= hi_all) shared_load<ND>(even, a, table, kvh, key0, lo_all, hi_all, lane);
        while (key0 <= hi_all) {
            if (key0 + STEP <= hi_all) shared_load<ND>(odd, a, table, kvh, key0 + STEP, lo_all, hi_all, lane);
            step(even, key0);
            key0 += STEP;
            if (key0 > hi_all) break;
            if (key0 + STEP <= hi_all) shared_load<ND>(even, a, table, kvh, key0 + STEP, lo_all, hi_all, lane);
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

template <int ND, int MT>
__global__ __launch_bounds__(SHARED_WAVES * WAVE, ND * MT > 4 ? 1 : 2) void k_attn_shared(SharedArgs a) {
    constexpr int DT = (ND + 1) / 2;
    __shared__ __attribute__((aligned(16))) float lds[2 * DT * 16 * WAVE + MT * SHARED_WAVES * 32];
    const int per = a.heads / a.kv_heads;
    int b = blockIdx.x;
    if (b < a.pre_blocks) {
        // the tiles of queries that read the same keys follow one another eight blocks apart: on one XCD, whose L2 has them
        const int tile = (b / 8) % a.pre_tiles, unit = b / (8 * a.pre_tiles) * 8 + b % 8;
        const int part = unit % a.n_pre, kvh = unit / a.n_pre % a.kv_heads, g = unit / (a.n_pre * a.kv_heads);
        if (g >= a.n_groups) return;
        const int first = max(a.group_start[g], 0), n = min(a.group_start[g + 1], a.n_rows) - first;
        const int keys = shared_keys(a, g), begin = part * a.pre_split, end = min(begin + a.pre_split, keys);
        const int first_query = tile * 32 * MT;
        if (first_query >= n * per || begin >= keys) return;
        shared_part<ND, MT>(a, first, n * per, first_query, per, kvh, a.table + (size_t)a.rows[first] * a.stride, begin, end, part, lds);
        return;
    }
    b -= a.pre_blocks;
    const int part = b % a.n_own, kvh = b / a.n_own % a.kv_heads, tile = b / (a.n_own * a.kv_heads) % a.own_tiles,
              i = b / (a.n_own * a.kv_heads * a.own_tiles);
    const int keys = shared_keys(a, group_of(a, i));
    const int row = a.rows[i];
    const int end_all = (int)min((long long)a.positions[a.seg_start[row]] + 1, (long long)a.stride << a.page_shift);
    const int begin = (keys & ~31) + part * a.own_split;
    if (begin >= end_all || keys >= end_all) return;
    shared_part<ND, 1>(a, i, per, tile * 32, per, kvh, a.table + (size_t)row * a.stride, max(begin, keys), min(begin + a.own_split, end_all),
                       a.n_pre + part, lds);
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
static SharedShape shared_shape(int n_rows, int heads, int kv_heads, int n_groups, int max_group, int max_shared, int max_own) {
    SharedShape s;
    const int per = heads / kv_heads;
    const long long queries = (long long)max_group * per;
    s.query_tiles = queries > 32 ? 2 : 1;
    s.pre_tiles = max_shared > 0 && n_groups > 0 ? (int)((queries + 32 * s.query_tiles - 1) / (32 * s.query_tiles)) : 0;
    s.own_tiles = (per + 31) / 32;
    auto cut = [](long long units, int keys, int& n, int& split) {
        const int most = (keys + SHARED_MIN_SPLIT - 1) / SHARED_MIN_SPLIT;
        n = clamped(512 / units, 1, most > 0 ? most : 1);
        split = ((keys + n - 1) / n + 127) & ~127;
        if (split < 128) split = 128;
        n = (keys + split - 1) / split;
    };
    if (s.pre_tiles) cut((long long)n_groups * kv_heads * s.pre_tiles, max_shared, s.n_pre, s.pre_split);
    else s.n_pre = 0, s.pre_split = 128;
    // (own keys are counted from a multiple of 32, up to 31 below the first)
    if (max_own > 0) cut((long long)n_rows * kv_heads * s.own_tiles, max_own + 31, s.n_own, s.own_split);
    else s.n_own = 0, s.own_split = 128;
    return s;
}
static bool shared_sizes_bad(int n_rows, int heads, int kv_heads, int n_groups, int max_group, int max_shared, int max_own) {
    return n_rows < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || n_groups < 0 || max_group < 0 || max_shared < 0 || max_own < 0 ||
           max_shared > 1 << 30 || max_own > 1 << 30 || n_rows > 1 << 20 || n_groups > 1 << 20 || max_group > 1 << 20 || heads > 1 << 16;
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
        table_stride <= 0 || page_size < 16 || (page_size & (page_size - 1)) || head_dim <= 0 || head_dim > 128 || head_dim % 16 ||
        n_pages <= 0 || window < 0)
        return IMPARO_BAD_ARGUMENT;
    if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)part_o) & 15 || ((uintptr_t)part_ml | (uintptr_t)out) & 7)
        return IMPARO_BAD_ARGUMENT;
    if (n_rows == 0) return IMPARO_OK;
    const SharedShape s = shared_shape(n_rows, heads, kv_heads, n_groups, max_group, max_shared, max_own);
    const long long parts = (long long)n_rows * heads * (s.n_pre + s.n_own);
    if (parts && (!part_o || !part_ml)) return IMPARO_BAD_ARGUMENT;
    if (part_o_floats < parts * head_dim || part_ml_floats < parts * 2) return IMPARO_SCRATCH_TOO_SMALL;
    const long long units = (long long)n_groups * kv_heads * s.n_pre;
    const long long pre_blocks = (units + 7) / 8 * 8 * s.pre_tiles, own_blocks = (long long)n_rows * kv_heads * s.own_tiles * s.n_own;
    if (pre_blocks + own_blocks > 1 << 30 || (long long)n_rows * heads > 1 << 30) return IMPARO_BAD_ARGUMENT;
    const SharedArgs a{(const bf16_t*)q, (const bf16_t*)k_cache, (const bf16_t*)v_cache, (bf16_t*)out, part_o, part_ml, rows, group_start, shared,
                       seg_start, positions, block_table, n_rows, n_groups, table_stride, __builtin_ctz((unsigned)page_size), heads, kv_heads,
                       n_pages, window, s.n_pre, s.pre_split, s.n_own, s.own_split, s.pre_tiles, s.own_tiles, (int)pre_blocks,
                       scale * 1.44269504088896340736f};
    hipStream_t st = (hipStream_t)stream;
    const int blocks = (int)(pre_blocks + own_blocks);
    if (blocks) {
#define SHARED_GO(ND)                                                                                             \
    case ND:                                                                                                      \
        if (s.query_tiles == 2) k_attn_shared<ND, 2><<<blocks, SHARED_WAVES * WAVE, 0, st>>>(a);                  \
        else k_attn_shared<ND, 1><<<blocks, SHARED_WAVES * WAVE, 0, st>>>(a);                                     \
        break;
        switch (head_dim / 16) {
            SHARED_GO(1) SHARED_GO(2) SHARED_GO(3) SHARED_GO(4) SHARED_GO(5) SHARED_GO(6) SHARED_GO(7) SHARED_GO(8)
        }
#undef SHARED_GO
        if (launch_status()) return IMPARO_LAUNCH_FAILED;
    }
    k_attn_shared_merge<<<n_rows * heads, WAVE, 0, st>>>(a, head_dim);
    return launch_status();
}

int imparo_load_code_attention_shared() {
    hipFuncAttributes attributes;
    return hipFuncGetAttributes(&attributes, reinterpret_cast<const void*>(&k_attn_shared_merge)) == hipSuccess ? IMPARO_OK
                                                                                                    : IMPARO_LAUNCH_FAILED;
}
