// Picking the next token from float32 logits: argmax (smallest index at the
// maximum, NaN never wins) and temperature sampling by inverse CDF.
#include "common.h"
#include "api.h"
#include <float.h>
#include <limits.h>

struct Best {
    float v;
    int i;
};

__device__ __forceinline__ Best better(Best a, Best b) {
    return (b.v > a.v || (b.v == a.v && b.i < a.i)) ? b : a;
}

__device__ __forceinline__ Best block_best(Best b, Best* scratch, int threads) {
    b = better(b, Best{lane_xor<32>(b.v), lane_xor<32>(b.i)});
    b = better(b, Best{lane_xor<16>(b.v), lane_xor<16>(b.i)});
    b = better(b, Best{lane_xor<8>(b.v), lane_xor<8>(b.i)});
    b = better(b, Best{lane_xor<4>(b.v), lane_xor<4>(b.i)});
    b = better(b, Best{lane_xor<2>(b.v), lane_xor<2>(b.i)});
    b = better(b, Best{lane_xor<1>(b.v), lane_xor<1>(b.i)});
    const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
    const int n_waves = (threads + WAVE - 1) / WAVE;
    __syncthreads();
    if (lane == 0) scratch[wave] = b;
    __syncthreads();
    Best r = scratch[0];
    for (int w = 1; w < n_waves; ++w) r = better(r, scratch[w]);
    return r;
}

__device__ __forceinline__ Best row_best(const float* __restrict__ row, int vocab, Best* scratch, int threads) {
    Best b;
    b.v = -INFINITY;
    b.i = INT_MAX;
    if ((vocab & 3) == 0 && (((uintptr_t)row) & 15) == 0) {
        // The maximum first, four values a load and sixteen loads in flight (a row of 65,536 on 1,024 threads is one trip
        // to memory; no load sits under a branch: past the end the row's last piece is read again, which changes no
        // maximum), then its smallest index by the threads that met it, from the run of loads they met it in: a comparison
        // and a choice of index for every value were a third of the time (one row of 65,536 9.0 us, so 6.2).
        const float4* row4 = reinterpret_cast<const float4*>(row);
        const int n4 = vocab >> 2;
        if (n4 <= threads) {
            // one load a thread: the maximum and its index together, one meeting of the block (a row of 1,000 in two 3.8 us)
            const float4 v = row4[min((int)threadIdx.x, n4 - 1)];
            const float vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if ((int)threadIdx.x < n4 && (vs[j] > b.v || (vs[j] == b.v && 4 * (int)threadIdx.x + j < b.i))) {
                    b.v = vs[j];
                    b.i = 4 * (int)threadIdx.x + j;
                }
            b = block_best(b, scratch, threads);
            if (b.i == INT_MAX) b.i = 0;   // every value was NaN
            return b;
        }
        constexpr int DEEP = 16;
        float m = -INFINITY;
        int met = 0;
        for (int first = threadIdx.x; first < n4; first += DEEP * threads) {
            float4 v[DEEP];
#pragma unroll
            for (int k = 0; k < DEEP; ++k) v[k] = row4[min(first + k * threads, n4 - 1)];
            float mm = -INFINITY;
#pragma unroll
            for (int k = 0; k < DEEP; ++k) mm = fmaxf(mm, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
            if (mm > m) {
                m = mm;
                met = first;
            }
        }
        float top = wave_max(m);
        const int n_waves = (threads + WAVE - 1) / WAVE;
        if ((threadIdx.x & (WAVE - 1)) == 0) scratch[threadIdx.x / WAVE].v = top;
        __syncthreads();
        float tops[16];
#pragma unroll
        for (int w = 0; w < 16; ++w) tops[w] = scratch[min(w, n_waves - 1)].v;
#pragma unroll
        for (int w = 0; w < 16; ++w) top = fmaxf(top, tops[w]);
        if (top > -INFINITY) {                       // (nothing but -inf and NaN: value by value below)
            if (m == top) {
                float4 v[DEEP];
#pragma unroll
                for (int k = 0; k < DEEP; ++k) v[k] = row4[min(met + k * threads, n4 - 1)];
#pragma unroll
                for (int k = DEEP - 1; k >= 0; --k) {
                    const int i = min(met + k * threads, n4 - 1);
                    const float vs[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
                    for (int j = 3; j >= 0; --j)
                        if (vs[j] == top) b.i = 4 * i + j;
                }
                b.v = top;
            }
            return block_best(b, scratch, threads);
        }
    }
    for (int i = threadIdx.x; i < vocab; i += threads) {
        const float v = row[i];
        if (v > b.v || (v == b.v && i < b.i)) {
            b.v = v;
            b.i = i;
        }
    }
    b = block_best(b, scratch, threads);
    if (b.i == INT_MAX) b.i = 0;   // every value was NaN
    return b;
}

__global__ void k_argmax_rows(const float* __restrict__ logits, int32_t* __restrict__ out, int vocab) {
    __shared__ Best scratch[16];
    const Best b = row_best(logits + (size_t)blockIdx.x * vocab, vocab, scratch, blockDim.x);
    if (threadIdx.x == 0) out[blockIdx.x] = b.i;
}

extern "C" int imparo_argmax_rows(const float* logits, int32_t* out, int n_rows, int vocab, imparo_stream stream) {
    if (!logits || !out || n_rows < 0 || vocab <= 0) return IMPARO_BAD_ARGUMENT;
    if (n_rows == 0) return IMPARO_OK;
    const int threads = vocab >= 16384 ? 1024 : 256;
    k_argmax_rows<<<n_rows, threads, 0, (hipStream_t)stream>>>(logits, out, vocab);
    return launch_status();
}

// Each thread owns one contiguous piece of the row. Piece sums are scanned in
// thread order, the piece holding u * total is walked element by element: the
// pick is the first index whose running sum exceeds the target.
// The sums' order is part of the result (two machines that draw the same number pick the same token), so the scan
// over the pieces and the walk inside one stay chains of additions; what a chain adds is fetched ahead of it, sixteen
// values a time, and all that is no addition (exponentials, comparisons) is done by the whole block. Measured, 64
// rows of 65,536 logits: 153 us with both chains reading LDS and memory value by value, 38 us so (28 us for rows of 16,384).
#define SAMPLE_THREADS 1024
__device__ __forceinline__ void sample_row(const float* __restrict__ row, float temp, float uniform, int32_t* __restrict__ out,
                                           int vocab, int threads) {
    __shared__ Best scratch[16];
    __shared__ __attribute__((aligned(16))) float sums[SAMPLE_THREADS], before[SAMPLE_THREADS];
    __shared__ int first_past, last_positive, found;
    __shared__ float cum_shared, target_shared;
    const Best top = row_best(row, vocab, scratch, threads);
    if (!(temp > 0.f)) {
        if (threadIdx.x == 0) *out = top.i;
        return;
    }
    const float inv_t = 1.0f / temp;
    const int tid = threadIdx.x;                               // (threads: a multiple of 16)
    const int piece = (vocab + threads - 1) / threads;
    const int begin = min(vocab, tid * piece), end = min(vocab, begin + piece);
    float local = 0.f;
    int i = begin;
    if (piece % 16 == 0 && (((uintptr_t)row) & 15) == 0) {     // whole vectors, sixteen values in flight
        for (; i + 16 <= end; i += 16) {
            float4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float4*>(row + i + 4 * j);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float e = expf((x[k] - top.v) * inv_t);
                    if (e == e) local += e;   // a NaN logit has probability zero
                }
            }
        }
    }
    for (; i < end; ++i) {
        const float e = expf((row[i] - top.v) * inv_t);
        if (e == e) local += e;
    }
    sums[tid] = local;
    if (tid == 0) {
        first_past = INT_MAX;
        last_positive = 0;
        found = -1;
    }
    __syncthreads();
    if (tid == 0) {                                            // what lies before each piece, and the total
        float total = 0.f;
        float4 next[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) next[j] = *reinterpret_cast<const float4*>(&sums[4 * j]);
        for (int t = 0; t < threads; t += 16) {
            float4 now[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                now[j] = next[j];
                next[j] = *reinterpret_cast<const float4*>(&sums[min(t + 16, threads - 16) + 4 * j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float4 b;
                b.x = total, total += now[j].x;
                b.y = total, total += now[j].y;
                b.z = total, total += now[j].z;
                b.w = total, total += now[j].w;
                *reinterpret_cast<float4*>(&before[t + 4 * j]) = b;
            }
        }
        target_shared = uniform * total;
    }
    __syncthreads();
    const float target = target_shared;
    if (local > 0.f) {
        if (before[tid] + local > target) atomicMin(&first_past, tid);
        atomicMax(&last_positive, tid);
    }
    __syncthreads();
    const int owner = first_past != INT_MAX ? first_past : last_positive;   // (rounding can push the target past the total)
    if (tid == 0) cum_shared = before[owner];
    const int own_begin = min(vocab, owner * piece), own_end = min(vocab, own_begin + piece);
    int last = top.i;
    for (int at = own_begin; at < own_end; at += threads) {
        __syncthreads();
        sums[tid] = at + tid < own_end ? expf((row[at + tid] - top.v) * inv_t) : 0.f;
        __syncthreads();
        if (tid == 0) {
            float cum = cum_shared;
            int pick = -1;
            const int n = min(threads, own_end - at);
            for (int t = 0; t < n && pick < 0; t += 16) {
                float4 v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float4*>(&sums[t + 4 * j]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float e[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool on = e[k] > 0.f && pick < 0;
                        if (on) last = at + t + 4 * j + k;
                        cum = on ? cum + e[k] : cum;
                        if (on && cum > target) pick = last;
                    }
                }
            }
            cum_shared = cum;
            found = pick;
        }
        __syncthreads();
        if (found >= 0) break;
    }
    if (tid == 0) *out = found >= 0 ? found : last;
}

__global__ __launch_bounds__(SAMPLE_THREADS) void k_sample_rows(
    const float* __restrict__ logits, const float* __restrict__ temperature, const float* __restrict__ uniform,
    int32_t* __restrict__ out, int vocab) {
    sample_row(logits + (size_t)blockIdx.x * vocab, temperature[blockIdx.x], uniform[blockIdx.x], out + blockIdx.x, vocab, blockDim.x);
}

// (the order of a row's sums depends on it)
__host__ __device__ static inline int sample_threads(int vocab) { return vocab >= 16384 ? SAMPLE_THREADS : 256; }

extern "C" int imparo_sample_rows(const float* logits, const float* temperature, const float* uniform, int32_t* out,
                                  int n_rows, int vocab, imparo_stream stream) {
    if (!logits || !temperature || !uniform || !out || n_rows < 0 || vocab <= 0) return IMPARO_BAD_ARGUMENT;
    if (n_rows == 0) return IMPARO_OK;
    const int threads = sample_threads(vocab);
    k_sample_rows<<<n_rows, threads, 0, (hipStream_t)stream>>>(logits, temperature, uniform, out, vocab);
    return launch_status();
}

// ---------------------------------------------------------------- picks under top-k, top-p and min-p
// With m the row's largest logit, w_i = 2^((x_i - m) log2(e) / T) and tokens in the order "larger logit first, smaller index
// first": top-k keeps the first k, top-p of those the fewest first whose weights reach p of their sum, min-p of those the ones
// with w_i >= min_p. Each keeps a beginning of that order, so what is kept is all above a logit and so many ties with it, the
// ones of the smallest index. The pick is the first token, in the order of indices, whose running sum of kept weights passes u
// times their sum.
// Sums decide here, and which token a sum passes at must not depend on how it was split: a weight is held as the integer
// nearest to w 2^44 (w from a float64 exponential), so sums are exact in any order, over any split, and by atomics. 2^19 logits
// fill 63 bits. A token below 2^-44 of the likeliest is not drawn: all of those together weigh less than 2^-25, under one
// step of a 24-bit u.
// One block a row, and what an instruction a logit costs is what the kernel costs (65,536 logits, 64 lanes a clock: 0.43 us each),
// so the row is read few times (out of L2 after the first) and little is done a logit. First the largest; then how far down anything is
// kept, as a number of bins, 2,048 over the 44 octaves that weigh anything: for min-p its own; for top-k the k-th largest of the threads'
// own maxima, as k logits at least are no smaller; for top-p alone the bin of a histogram of weights, 512 of them as fine as the row allows, where p of them is reached. The
// tokens above that go into a list, four a thread at most, and border, ties and pick are found in the list alone, every
// token compared with every other where they are few, else by histograms over nine bits of keys or indices at a time (list_find). A row
// that keeps more than a few under top-p lists the tokens of the border's bin only, has the sums of the ones above by the runs they are in (every wave has a
// histogram of its run), and picks in the run that u falls in: one exponential a logit, and one for those of that run. What fits neither (large top-k, thousands of ties) is done over the row itself, pass by pass (pick_narrow).
// Measured, a row a block, logits of normal noise: one of 65,536 under top-k (and top-p) 12.0 us, under min-p 9.4 to 10, under top-p (0.95, T = 1) 23 where
// one token is kept (a deviation of 6), 25 with 42 (4), 33 with 3,570 (3), 36 to 39 with more (2.5 and less), of which the largest logit 6, weights and
// their histogram 13, the border's tokens 5 to 9, border and pick 4 to 11; 64 rows under top-k and top-p 13 to 14; 256 rows of 130,001 of all kinds 82, under
// top-k 43, where argmax takes 52.
#define PICK_THREADS 1024          // of short rows too (with 256 threads, when that was tried: 5 of 1,003 under top-k 13.1 us for 9.9, 8 of 16,000 under top-p 53 for 24)
#define PICK_BINS 2048
#define PICK_BITS 9                // bits of a key or an index that a search in the list settles at a time
#define PICK_FEW 256               // tokens that are compared with one another instead
#define PICK_EACH 4                // tokens of the list a thread has at most
#define PICK_CUT 44
#define PICK_RUNS (PICK_THREADS / WAVE)
#define PICK_COARSE (PICK_BINS / 4)
#define PICK_STEPS 512

typedef unsigned long long u64;

// the float's place in the order of floats (-0 and 0 are one), and back
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float float_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

template <int N>
__device__ __forceinline__ u64 lane_xor_u64(u64 v) {
    return ((u64)lane_xor_bits<N>((uint32_t)(v >> 32)) << 32) | lane_xor_bits<N>((uint32_t)v);
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
    v += lane_xor_u64<1>(v);
    v += lane_xor_u64<2>(v);
    v += lane_xor_u64<4>(v);
    v += lane_xor_u64<8>(v);
    v += lane_xor_u64<16>(v);
    v += lane_xor_u64<32>(v);
    return v;
}
// What CTRL moves to this lane, 0 where nothing comes: the steps of a running sum over the lanes
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved(u64 v) {
    return ((u64)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false) << 32) |
           (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ u64 wave_scan(u64 v) {                 // the sum over the lanes up to and with this one
    v += moved<0x111, 0xf>(v);                                    // row_shr:1, 2, 4, 8
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);                                    // lane 15 of a row of 16 to the next row: rows 1 and 3
    v += moved<0x143, 0xc>(v);                                    // lane 31 to rows 2 and 3
    return v;
}

struct PickShared {
    u64 hist[PICK_RUNS * PICK_COARSE];      // (PICK_BINS of them where the runs do not have one each)
    u64 level[2][1 << PICK_BITS];     // used in turn: while one is read the other is cleared
    float list_x[PICK_EACH * PICK_THREADS];
    int list_index[PICK_EACH * PICK_THREADS];
    double table[PICK_STEPS];         // 2^(PICK_CUT + i / PICK_STEPS)
    u64 waves[16], turns[132];
    float tops[16], sums[16];
    u64 few_ord[PICK_FEW], few_weight[PICK_FEW], few_mass[2][PICK_FEW], few_sum[2];
    int few_rank[PICK_FEW];
    u64 above, inside, need;          // of the bin where the sum is reached: what lies above it, what it holds; what is asked for
    int bin, n_list, cut, reached;
    uint32_t low;
    uint32_t key_low, key_high;
};

// 2^(PICK_CUT + i / PICK_STEPS): e^z as its power series up to z^17 / 17!, z < 0.7, below a tenth of a float64's step
struct PickTable {
    double v[PICK_STEPS];
    constexpr PickTable() : v() {
        for (int i = 0; i < PICK_STEPS; ++i) {
            const double z = 0.69314718055994530942 * i / PICK_STEPS;
            double sum = 1.0;
            for (int n = 17; n > 0; --n) sum = 1.0 + sum * z / n;
            v[i] = sum * (double)(1ull << PICK_CUT);
        }
    }
};
static __device__ const PickTable pick_table = PickTable();

// Weights of a row: 2^y 2^44 to the nearest integer, y = (x - top) c1 <= 0, for y above -45 (what is asked about lies in one of the bins).
// y 512 = n + f with n whole, 2^(n / 512) out of a table and an exponent, and 2^(f / 512), |f| <= 1/2, from its power series, cut where the next term
// is below 2^-46; rounded with the addition of 2^52, whose low bits then are the integer.
struct PickWeights {
    static_assert(PICK_STEPS == 1 << 9, "the shift below");
    double top, c;                    // c1 PICK_STEPS
    const double* table;
    __device__ __forceinline__ u64 operator()(float x) const {
        constexpr double MAGIC = 6755399441055744.0, L = 0.69314718055994530942 / PICK_STEPS;
        const double d = (double)x - top, t = fma(d, c, MAGIC), f = fma(d, c, -(t - MAGIC));
        const int n = __double2loint(t);
        double p = fma(f, L * L * L / 6, L * L / 2);
        p = fma(f, p, L);
        p = fma(f, p, 1.0);
        const double step = table[n & (PICK_STEPS - 1)];
        const double v = fma(p, __hiloint2double(__double2hiint(step) + (int)((uint32_t)(n & -PICK_STEPS) << 11), __double2loint(step)), 4503599627370496.0);
        return (u64)__double_as_longlong(v) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ double octaves(float x) const { return ((double)x - top) * c * (1.0 / PICK_STEPS); }
};

// The bin of sh.hist where the running sum reaches what is asked for: `need`, or for share >= 0 that share of all. Leaves bin,
// above, inside and need in LDS; bin is -1 where the sum is never reached. Every thread calls, behind and ahead of a barrier of its own.
__device__ __forceinline__ void pick_bin(PickShared& sh, u64 need, double share) {
    const int threads = blockDim.x, per = PICK_BINS / threads, tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    u64 mine = 0;
    for (int i = 0; i < per; ++i) mine += sh.hist[tid * per + i];
    const u64 upto = wave_scan(mine);
    if (lane == WAVE - 1) sh.waves[wave] = upto;
    if (tid == 0) sh.bin = -1;
    __syncthreads();
    u64 before = 0, total = 0;
    for (int w = 0; w < threads / WAVE; ++w) {
        const u64 v = sh.waves[w];
        before += w < wave ? v : 0;
        total += v;
    }
    if (share >= 0.0) need = max((u64)1, (u64)ceil(share * (double)total));
    u64 at = before + upto - mine;
    if (at < need && need <= at + mine) {
        int b = tid * per;
        u64 v = sh.hist[b];
        while (at + v < need) {
            at += v;
            v = sh.hist[++b];
        }
        sh.bin = b;
        sh.above = at;
        sh.inside = v;
        sh.need = need;
    }
    __syncthreads();
}

// A row's logits, lane by lane: wave w has the values of its own run, 256 a turn, four neighbours a lane. What stands in front of
// the row or behind it inside the 16 aligned bytes that hold its first or last value is read with them (the same 16 bytes of
// memory, so it is there) and counts as NaN, which every comparison passes over.
struct PickRow {
    const float4* base;
    int skew, vocab, turns, first;      // first: index in the row of this lane's first value in turn 0
    int wave_first;                     // the same of the wave's first lane

    __device__ __forceinline__ void open(const float* row, int n) {
        vocab = n;
        skew = (int)(((uintptr_t)row & 15) >> 2);
        base = reinterpret_cast<const float4*>(row - skew);
        const int waves = blockDim.x / WAVE, lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
        turns = (vocab + skew + 4 * WAVE * waves - 1) / (4 * WAVE * waves);
        of_wave(wave);
    }
    __device__ __forceinline__ void of_wave(int wave) {
        wave_first = wave * turns * 4 * WAVE - skew;
        first = wave_first + 4 * ((int)threadIdx.x & (WAVE - 1));
    }
    __device__ __forceinline__ float4 load(int c) const { return base[min(max(first + skew + c * 4 * WAVE, 0), vocab + skew - 1) >> 2]; }
    __device__ __forceinline__ void values(float (&x)[4], const float4& v, int c) const {
        const int i = first + c * 4 * WAVE, w = wave_first + c * 4 * WAVE;
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        if (w < 0 || w + 4 * WAVE > vocab) {                      // (the wave's turn reaches past an end of the row)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = i + j >= 0 && i + j < vocab ? x[j] : __builtin_nanf("");
        }
    }
    // f(values, index of the first of the four), turn after turn, the loads of DEEP turns in flight. Code that a block runs through once
    // comes out of memory too: long bodies are better off in a loop than written out many times.
    template <int DEEP = 4, typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int c0 = 0; c0 < turns; c0 += DEEP) {
            float4 v[DEEP];
#pragma unroll
            for (int c = 0; c < DEEP; ++c) v[c] = load(c0 + c);
#pragma unroll
            for (int c = 0; c < DEEP; ++c) {
                if (c0 + c >= turns) break;
                float x[4];
                values(x, v[c], c0 + c);
                f(x, first + (c0 + c) * 4 * WAVE);
            }
        }
    }
};

// What of a row is kept: keys above `key`, and the key itself up to index `cut`
struct PickSet {
    uint32_t key;
    int cut;
    __device__ __forceinline__ bool has(uint32_t k, int index) const { return k > key || (k == key && index <= cut); }
};

// ---- in the list: a thread's tokens, and for the search at hand what each counts and where it stands in the order
struct PickList {
    float x[PICK_EACH];
    int index[PICK_EACH];
    u64 weight[PICK_EACH], counts[PICK_EACH];
    uint32_t ord[PICK_EACH];
    int n, turn;                       // tokens of this thread; the histogram that is next in turn

    __device__ __forceinline__ void take(const PickShared& sh, const PickWeights& weights, int threads) {
        const int all = sh.n_list;
        n = 0;
#pragma unroll
        for (int e = 0; e < PICK_EACH; ++e) {
            const int at = e * threads + (int)threadIdx.x;
            if (e * threads >= all) break;
            if (at < all) {
                x[e] = sh.list_x[at];
                index[e] = sh.list_index[at];
                weight[e] = weights(x[e]);
                n = e + 1;
            }
        }
    }
};

// Where, among the list's tokens and in the order of `ord` (whole numbers from low to high, the smallest first), the running sum of `counts`
// reaches `need`, or of their sum the part that `asked` says (asked(sum)): sets ord, above and inside of the one that is passed at; false where it is never
// reached. PICK_BITS at a time: a histogram by atomics, and one wave adds its bins up (all of them for themselves would take four times as
// long: a SIMD has four of them).
struct Found {
    uint32_t ord;
    u64 above, inside, need;
};
template <typename A>
__device__ __forceinline__ bool list_find(PickShared& sh, PickList& list, uint32_t low, uint32_t high, Found& found, A asked) {
    constexpr int BINS = 1 << PICK_BITS, PER = BINS / WAVE;
    const int tid = threadIdx.x, lane = tid & (WAVE - 1);
    u64 above = 0, need = 0;
    auto slot = [](uint32_t b) { return b % PER * WAVE + b / PER; };      // (a lane adds up PER neighbours: apart by as many as there are lanes, no two meet on a bank)
    for (bool first = true;; first = false) {
        const int bits = low == high ? 0 : 32 - __clz((int)(high - low)), shift = max(0, bits - PICK_BITS);
        u64* hist = sh.level[list.turn];
        list.turn ^= 1;
#pragma unroll
        for (int e = 0; e < PICK_EACH; ++e)
            if (e < list.n && list.counts[e] && list.ord[e] >= low && list.ord[e] <= high)
                atomicAdd(&hist[slot((list.ord[e] - low) >> shift)], list.counts[e]);
        __syncthreads();
        if (tid >= WAVE) {
            for (int b = tid - WAVE; b < BINS; b += (int)blockDim.x - WAVE) sh.level[list.turn][b] = 0;
        } else {
            u64 bin[PER], mine = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                bin[i] = hist[i * WAVE + lane];
                mine += bin[i];
            }
            const u64 upto = wave_scan(mine);
            if (first) need = asked(((u64)(uint32_t)__builtin_amdgcn_readlane((int)(upto >> 32), WAVE - 1) << 32) |
                                    (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)upto, WAVE - 1));
            u64 at = upto - mine + above;
            const bool here = at < need && need <= at + mine;
            if (lane == 0 && !__any(here)) sh.reached = 0;
            if (here) {
                int b = 0;
                u64 inside = bin[0];
#pragma unroll
                for (int i = 0; i < PER - 1; ++i)
                    if (b == i && at + bin[i] < need) {
                        at += bin[i];
                        b = i + 1;
                        inside = bin[i + 1];
                    }
                sh.reached = 1;
                sh.above = at;
                sh.inside = inside;
                sh.need = need;
                sh.low = low + ((uint32_t)(PER * lane + b) << shift);
            }
        }
        __syncthreads();
        if (!sh.reached) return false;
        low = sh.low;
        above = sh.above;
        need = sh.need;
        if (shift == 0) break;
        high = high - low > (1u << shift) - 1 ? low + ((1u << shift) - 1) : high;
    }
    found = Found{low, above, sh.inside, need};
    return true;
}
// The running sum at which a uniform number picks: the first whole number above u times the sum, and no more than the sum (at which the last
// token is reached). A NaN counts as 0.
__device__ __forceinline__ u64 passed_at(float u, u64 total) {
    return min((u64)fmin(fmax((double)u * (double)total, 0.0), (double)total), total - 1) + 1;
}

// The whole choice in a list of at most PICK_FEW tokens: every token is compared with every other one. How many stand before it in the order, and
// what they weigh, says whether it is kept; what the kept ones of smaller indices weigh, whether it is picked. Two rounds of compares (128
// tokens: 0.2 us of them each) and five barriers, where the searches bit by bit take up to a dozen rounds behind one another.
template <int THREADS>
__device__ __forceinline__ void pick_few(PickShared& sh, const PickWeights& weights, int k, double share, bool by_k, bool by_p, u64 need_p, double floor_y,
                                         float u, int32_t* out) {
    const int tid = threadIdx.x, n = sh.n_list;
    const int bits = n <= WAVE ? 6 : 32 - __clz(n - 1);           // entries a row of threads: whole waves, so that a wave compares with one token at a time
    const int i = tid & ((1 << bits) - 1), part = tid >> bits, parts = THREADS >> bits;
    u64 weight = 0;
    int index = 0;
    bool kept = false;
    if (tid < n) {
        const float x = sh.list_x[tid];
        index = sh.list_index[tid];
        weight = weights(x);
        kept = weights.octaves(x) >= floor_y;
        sh.few_ord[tid] = (u64)~key_of(x) << 32 | (uint32_t)index;
        sh.few_weight[tid] = weight;
        sh.few_mass[0][tid] = sh.few_mass[1][tid] = 0;
        sh.few_rank[tid] = 0;
    }
    if (tid < 2) sh.few_sum[tid] = 0;
    __syncthreads();
    u64 mass = 0;
    int rank = 0;
    const u64 ord = sh.few_ord[i];                                // (past the list: not used)
    for (int j = part; j < n; j += parts) {
        const u64 w = sh.few_weight[j];
        const bool before = sh.few_ord[j] < ord;
        rank += before;
        mass += before ? w : 0;
    }
    if (i < n) {
        atomicAdd(&sh.few_mass[0][i], mass);
        atomicAdd(&sh.few_rank[i], rank);
    }
    __syncthreads();
    if (tid < n) {
        mass = sh.few_mass[0][tid];
        rank = sh.few_rank[tid];
        kept = kept && (!by_k || rank < k);
        if (by_k && by_p && rank == min(k, n) - 1) sh.few_sum[0] = mass + weight;
    }
    if (by_k && by_p) {
        __syncthreads();
        need_p = max((u64)1, (u64)ceil(share * (double)sh.few_sum[0]));
    }
    if (by_p) kept = kept && mass < need_p;
    weight = kept ? weight : 0;
    if (tid < PICK_FEW) {                                         // (whole waves)
        if (tid < n) sh.few_weight[tid] = weight;
        const u64 sum = wave_sum_u64(tid < n ? weight : 0);
        if ((tid & (WAVE - 1)) == 0) atomicAdd(&sh.few_sum[1], sum);
    }
    __syncthreads();
    mass = 0;
    for (int j = part; j < n; j += parts) mass += (uint32_t)sh.few_ord[j] < (uint32_t)ord ? sh.few_weight[j] : 0;
    if (i < n) atomicAdd(&sh.few_mass[1][i], mass);
    __syncthreads();
    if (tid < n && weight) {
        const u64 before = sh.few_mass[1][tid], target = passed_at(u, sh.few_sum[1]) - 1;
        if (before <= target && target < before + weight) *out = index;
    }
}

// The same comparison for the border alone: of a list of at most PICK_FEW tokens, the last one in the order that is needed for `need` of their weights.
// False where all of them are fewer.
__device__ __forceinline__ bool pick_border(PickShared& sh, const PickWeights& weights, u64 need, PickSet& set) {
    const int tid = threadIdx.x, n = sh.n_list;
    const int bits = n <= WAVE ? 6 : 32 - __clz(n - 1);
    const int i = tid & ((1 << bits) - 1), part = tid >> bits, parts = PICK_THREADS >> bits;
    if (tid < n) {
        sh.few_ord[tid] = (u64)~key_of(sh.list_x[tid]) << 32 | (uint32_t)sh.list_index[tid];
        sh.few_weight[tid] = weights(sh.list_x[tid]);
        sh.few_mass[0][tid] = 0;
    }
    if (tid == 0) sh.cut = -1;
    __syncthreads();
    u64 mass = 0;
    const u64 ord = sh.few_ord[i];                                // (past the list: not used)
    for (int j = part; j < n; j += parts) mass += sh.few_ord[j] < ord ? sh.few_weight[j] : 0;
    if (i < n) atomicAdd(&sh.few_mass[0][i], mass);
    __syncthreads();
    if (tid < n) {
        const u64 before = sh.few_mass[0][tid];
        if (before < need && need <= before + sh.few_weight[tid]) {
            sh.key_low = ~(uint32_t)(sh.few_ord[tid] >> 32);
            sh.cut = (int)(uint32_t)sh.few_ord[tid];
        }
    }
    __syncthreads();
    if (sh.cut < 0) return false;
    set = PickSet{sh.key_low, sh.cut};
    return true;
}

// What is left to do in the list, in this order; the searches for ties only where not all of them stay
enum { PICK_K, PICK_K_TIES, PICK_P, PICK_P_TIES, PICK_DRAW };

// ---- in the row: the same, a pass over the row for each step
template <bool COUNT>
__device__ __forceinline__ void pick_narrow(PickShared& sh, const PickRow& row, PickSet& set, float top, float bin_scale,
                                            const PickWeights& weights, u64 need, double share) {
    const int tid = threadIdx.x, threads = blockDim.x;
    auto weight = [&](float x) { return COUNT ? (u64)1 : weights(x); };
    auto place = [&](float x) { return (top - x) * bin_scale; };
    __syncthreads();
    for (int b = tid; b < PICK_BINS; b += threads) sh.hist[b] = 0;
    if (tid == 0) {
        sh.key_low = 0xFFFFFFFFu;
        sh.key_high = 0;
    }
    __syncthreads();
    row.each([&](const float (&x)[4], int index) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (place(x[j]) < (float)PICK_BINS && set.has(key_of(x[j]), index + j)) atomicAdd(&sh.hist[(int)place(x[j])], weight(x[j]));
    });
    __syncthreads();
    pick_bin(sh, need, share);
    if (sh.bin < 0) return;                                       // fewer than are asked for: all stay
    u64 above = sh.above, inside = sh.inside;
    need = sh.need;
    const int bin = sh.bin;
    row.each([&](const float (&x)[4], int index) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!(place(x[j]) < (float)PICK_BINS) || (int)place(x[j]) != bin || !set.has(key_of(x[j]), index + j)) continue;
            atomicMin(&sh.key_low, key_of(x[j]));
            atomicMax(&sh.key_high, key_of(x[j]));
        }
    });
    __syncthreads();
    uint32_t low = sh.key_low, high = sh.key_high;
    while (low != high) {                                         // (at most three times: 11 bits of at most 32 each)
        const int bits = 32 - __clz((int)(high - low)), shift = max(0, bits - 11);
        __syncthreads();
        for (int b = tid; b < PICK_BINS; b += threads) sh.hist[b] = 0;
        __syncthreads();
        row.each([&](const float (&x)[4], int index) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t k = key_of(x[j]);
                if (x[j] == x[j] && k >= low && k <= high && set.has(k, index + j)) atomicAdd(&sh.hist[(high - k) >> shift], weight(x[j]));
            }
        });
        __syncthreads();
        pick_bin(sh, need - above, -1.0);
        above += sh.above;
        inside = sh.inside;
        high -= (uint32_t)sh.bin << shift;
        low = high - low > (1u << shift) - 1 ? high - ((1u << shift) - 1) : low;
    }
    // one key is left: so many of its tokens, in the order of their indices, reach what is asked for
    const u64 each = weight(float_of(high)), ties = (need - above + each - 1) / each;
    set.cut = high == set.key ? set.cut : INT_MAX;
    set.key = high;
    if (ties * each >= inside) return;                            // all of them
    const int lane = tid & (WAVE - 1), wave = tid / WAVE;
    const float tie = float_of(high);
    u64 mine = 0;
    row.each([&](const float (&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) mine += __popcll(__ballot(x[j] == tie));
    });
    __syncthreads();
    if (lane == 0) sh.waves[wave] = mine;
    __syncthreads();
    u64 before = 0;
    for (int w = 0; w < wave; ++w) before += sh.waves[w];
    if (before < ties && ties <= before + mine) {
        row.each([&](const float (&x)[4], int index) {
            u64 ahead = before;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const u64 who = __ballot(x[j] == tie);
                ahead += __popcll(who & ((1ull << lane) - 1));
                before += __popcll(who);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (x[j] == tie && ++ahead == ties) sh.cut = index + j;
        });
    }
    __syncthreads();
    set.cut = sh.cut;
}

// The pick out of the row, for what `kept` says of a logit and its index, where the sums over the waves' runs stand in sh.waves: all waves take the turns of
// the run where u falls, then a wave the turn.
template <typename K>
__device__ __forceinline__ void pick_in_runs(PickShared& sh, PickRow row, float u, const PickWeights& weights, int32_t* out, K kept) {
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE, waves = blockDim.x / WAVE;
    u64 total = 0;
    for (int w = 0; w < waves; ++w) total += sh.waves[w];
    const u64 target = passed_at(u, total) - 1;
    u64 before = 0;
    int run = 0;
    while (run < waves - 1 && before + sh.waves[run] <= target) before += sh.waves[run++];
    row.of_wave(run);
    auto four_of = [&](int c, u64 (&w)[4]) {
        float x[4];
        row.values(x, row.load(c), c);
        u64 sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = kept(x[j], row.first + c * 4 * WAVE + j) ? weights(x[j]) : 0;
            sum += w[j];
        }
        return sum;
    };
    for (int c = wave; c < row.turns; c += waves) {
        u64 w[4];
        const u64 sum = wave_sum_u64(four_of(c, w));
        if (lane == 0) sh.turns[c] = sum;
    }
    __syncthreads();
    if (wave != 0) return;
    int c = 0;
    while (c < row.turns - 1 && before + sh.turns[c] <= target) before += sh.turns[c++];
    u64 w[4];
    const u64 four = four_of(c, w), upto = wave_scan(four), past = __ballot(before + upto > target);
    if (lane == __ffsll((long long)past) - 1) {
        u64 at = before + upto - four;
        int j = 0;
        while (j < 3 && at + w[j] <= target) at += w[j++];
        *out = row.first + c * 4 * WAVE + j;
    }
}
// The same, the sums first
template <typename K>
__device__ __forceinline__ void pick_from_row(PickShared& sh, const PickRow& row, float u, const PickWeights& weights, int32_t* out, K kept) {
    u64 mine = 0;
    row.each([&](const float (&x)[4], int index) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (kept(x[j], index + j)) mine += weights(x[j]);
    });
    mine = wave_sum_u64(mine);
    __syncthreads();
    if ((threadIdx.x & (WAVE - 1)) == 0) sh.waves[threadIdx.x / WAVE] = mine;
    __syncthreads();
    pick_in_runs(sh, row, u, weights, out, kept);
}

__global__ __launch_bounds__(PICK_THREADS) void k_pick_rows(
    const float* __restrict__ logits, const float* __restrict__ temperature, const float* __restrict__ uniform,
    const int32_t* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p,
    int32_t* __restrict__ out, int vocab) {
    __shared__ PickShared sh;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    constexpr int THREADS = PICK_THREADS, WAVES = THREADS / WAVE, ROOM = PICK_EACH * THREADS;
    const float* row_at = logits + (size_t)r * vocab;
    const float temp = temperature[r], u = uniform[r];
    const int k = top_k ? top_k[r] : 0;
    const float p = top_p ? top_p[r] : 1.f, mp = min_p ? min_p[r] : 0.f;
    const bool by_k = k > 0 && k < vocab, by_p = p < 1.f, by_m = mp > 0.f;
    if (!(temp > 0.f) || !(by_k || by_p || by_m)) {               // greedy, or the whole distribution
        if (tid < sample_threads(vocab)) sample_row(row_at, temp, u, out + r, vocab, sample_threads(vocab));   // (in whole waves; the others are done)
        return;
    }
    PickRow row;
    row.open(row_at, vocab);
    float own_top = -INFINITY;                                    // the largest of this thread's
    auto largest = [&](const float (&x)[4]) { return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])); };
    for (int i = tid; i < PICK_STEPS; i += THREADS) sh.table[i] = pick_table.v[i];
    for (int b = tid; b < PICK_RUNS * PICK_COARSE; b += THREADS) sh.hist[b] = 0;
    for (int b = tid; b < 2 << PICK_BITS; b += THREADS) (&sh.level[0][0])[b] = 0;
    if (tid == 0) {
        sh.n_list = 0;
        sh.bin = PICK_COARSE - 1;                                 // (found anew under top-p: the largest logit weighs 2^PICK_CUT, in bin 0)
        sh.above = 0;
    }
    row.each<8>([&](const float (&x)[4], int) { own_top = fmaxf(own_top, largest(x)); });
    float top = wave_max(own_top);
    // how far the threads' largest logits lie below the row's, added up: distances, none of them negative however it rounds (a mean of the logits
    // themselves may come out above the largest where all are alike). Infinite or NaN where a thread has none, or the sum is out of range
    const float below_wave = wave_sum(top - own_top);
    if (lane == 0) {
        sh.tops[wave] = top;
        sh.sums[wave] = below_wave;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, sh.tops[w]);
    float below = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) below += sh.sums[w] + WAVE * (top - sh.tops[w]);
    if (!(top < INFINITY) || !(top > -INFINITY)) {                // an infinite logit takes it, or there is none to take
        if (tid < sample_threads(vocab)) sample_row(row_at, 0.f, u, out + r, vocab, sample_threads(vocab));
        return;
    }
    // (the bins are float32: a temperature below 1.4e-36 counts as that, and tells logits apart that differ by 4e-35)
    const double c1 = fmin(1.44269504088896340736 / (double)temp, 1.0e36);
    const PickWeights weights{(double)top, c1 * PICK_STEPS, sh.table};
    const double floor_y = by_m ? fmax(-(double)PICK_CUT, log2((double)fminf(mp, 1.f))) : -(double)PICK_CUT;
    // bins an octave, and a unit of the logit: a logit d below the top is in bin d bin_scale
    constexpr float BINS_AN_OCTAVE = (float)PICK_BINS / PICK_CUT;
    const float whole_scale = BINS_AN_OCTAVE * (float)c1;
    float bin_scale = whole_scale, finer = 1.f;                   // (bin_scale / whole_scale)
    if (by_p && !by_k) {
        // Under top-p alone the bins are as fine as leaves the last one few: where a row is nearly flat, lanes that add to one bin wait for one another,
        // and its border's bin is long: 130,001 logits with a deviation of 0.2, T = 1 and p = 0.5 take 225 us with bins over all octaves, 63 so. Six times the way
        // from the largest logit to the mean of the threads' largest ones ends, in a row like noise, four deviations below the middle (four times: two, where 256
        // such rows had one or another whose border was in the last bin, 120 us more). What lies behind the last bin counts as in it; of no bearing on the result
        const float range = 6.f / THREADS * below;                // (neither infinite nor NaN is less than what it is compared with)
        if (range * whole_scale < (float)PICK_BINS) {
            finer = fminf(fminf((float)PICK_BINS / (range * whole_scale), 1024.f), 1.0e38f / whole_scale);    // (a whole_scale of 0, T infinite: 1024)
            bin_scale = whole_scale * finer;
        }
    }
    const float far = (float)PICK_BINS * finer;                   // so many bins are PICK_CUT octaves
    constexpr int LAST = PICK_COARSE - 1;
    auto place = [&](float x) { return (top - x) * bin_scale; };

    // ---- how far down the list has to reach: `limit`, a number of bins
    float limit = (float)PICK_BINS;
    const double share = (double)fmaxf(p, 0.f);
    u64 need_p = 0;
    bool window = false;                                          // the list has the tokens of the border's bin only: not all that is kept is in it
    if (by_k) {
        if (k <= THREADS / 2) {
            // the k-th largest of the threads' maxima: so many logits at least are no smaller, and not many more
            if (place(own_top) < (float)PICK_BINS) atomicAdd(&sh.hist[(int)place(own_top)], (u64)1);
            __syncthreads();
            pick_bin(sh, (u64)k, -1.0);
            if (sh.bin >= 0) limit = (float)(sh.bin + 1);
        } else {
            row.each([&](const float (&x)[4], int) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (place(x[j]) < (float)PICK_BINS) atomicAdd(&sh.hist[(int)place(x[j])], (u64)1);
            });
            __syncthreads();
            pick_bin(sh, (u64)k, -1.0);
            if (sh.bin >= 0) limit = (float)(sh.bin + 1);
        }
    } else if (by_p) {
        u64* run = sh.hist + wave * PICK_COARSE;
        row.each([&](const float (&x)[4], int) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float at = place(x[j]);
                if (at < far) atomicAdd(&run[min((int)at >> 2, LAST)], weights(x[j]));
            }
        });
        __syncthreads();
        u64 mine = 0;                                             // a thread's bin, over all runs
        if (tid < PICK_COARSE)
#pragma unroll
            for (int w = 0; w < WAVES; ++w) mine += sh.hist[w * PICK_COARSE + tid];
        const u64 upto = wave_scan(mine);
        if (lane == WAVE - 1) sh.waves[wave] = upto;
        __syncthreads();
        u64 at = upto - mine, all = 0;
        for (int w = 0; w < WAVES; ++w) {
            at += w < wave ? sh.waves[w] : 0;
            all += sh.waves[w];
        }
        need_p = max((u64)1, (u64)ceil(share * (double)all));
        if (at < need_p && need_p <= at + mine) {
            sh.bin = tid;
            sh.above = at;
        }
        // about how many tokens that is, from what the bins hold and a token of a bin weighs
        float about = at < need_p ? (float)mine * __builtin_amdgcn_exp2f(((float)tid + 0.5f) * 4.f / (BINS_AN_OCTAVE * finer) - (float)PICK_CUT) : 0.f;
        about = wave_sum(about);
        if (lane == 0) sh.tops[wave] = about;
        __syncthreads();
        about = 0.f;
        for (int w = 0; w < WAVES; ++w) about += sh.tops[w];
        window = about > 0.8f * (float)PICK_FEW;                  // (of no bearing on the result)
        limit = sh.bin < LAST ? 4.f * (float)(sh.bin + 1) : far;
    }
    // min-p's own border, as a number of bins: above its bin nothing is taken out, below it nothing kept (a hundredth aside, for roundings)
    const float floor_place = (float)(-floor_y * (double)BINS_AN_OCTAVE) * finer;
    // (a token that min-p takes out need not be listed, unless top-p asks for the sum of the k largest)
    if (by_m && !(by_k && by_p)) limit = fminf(limit, floor_place * 1.0001f + 0.01f);

    // ---- the list
    auto enlist = [&](float x, int index) {
        const int at = atomicAdd(&sh.n_list, 1);
        if (at < ROOM) {
            sh.list_x[at] = x;
            sh.list_index[at] = index;
        }
    };
    if (!window) {
        row.each([&](const float (&x)[4], int index) {
            if (place(largest(x)) < limit) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (place(x[j]) < limit) enlist(x[j], index + j);
            }
        });
        __syncthreads();
        if (by_p && !by_k && sh.n_list > PICK_FEW) {
            window = true;
            __syncthreads();
            if (tid == 0) sh.n_list = 0;
            __syncthreads();
        }
    }
    // under top-p alone the list then has the tokens of one bin, top-p's or min-p's, whichever is the higher one: all above are kept
    float border = 0.f;
    // (no listed token lies outside these)
    auto highest_listed = [&]() { return fminf(top, top - border / bin_scale * 0.9999f + fabsf(top) * 1.0e-5f); };
    auto lowest_listed = [&]() { return top - limit / bin_scale * 1.0001f - fabsf(top) * 1.0e-5f; };
    bool by_border = false;                                       // (top-p's border is in that bin)
    if (window) {
        const int floor_bin = min((int)fmaxf(floor_place * 0.9999f - 0.01f, 0.f) >> 2, LAST), bin = by_m ? min(sh.bin, floor_bin) : sh.bin;
        by_border = bin == sh.bin;
        border = 4.f * (float)bin;
        limit = bin < LAST ? border + 4.f : far;
        if (by_m && bin == floor_bin) limit = fmaxf(limit, floor_place * 1.0001f + 0.01f);
        // (a few of many: four at a time by their distance from the middle of what may be listed)
        const float low = 0.5f * lowest_listed(), high = 0.5f * highest_listed(), middle = low + high, reach = high - low + (fabsf(low) + fabsf(high)) * 1.0e-5f;
        row.each([&](const float (&x)[4], int index) {
            if (fminf(fminf(fabsf(x[0] - middle), fabsf(x[1] - middle)), fminf(fabsf(x[2] - middle), fabsf(x[3] - middle))) <= reach) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (place(x[j]) < limit && place(x[j]) >= border) enlist(x[j], index + j);
            }
        });
        u64 sure = 0;                                             // what this wave's tokens above that bin weigh
        for (int i = lane; i < bin; i += WAVE) sure += sh.hist[wave * PICK_COARSE + i];
        sure = wave_sum_u64(sure);
        if (lane == 0) sh.turns[wave] = sure;
        __syncthreads();
        if (by_border) need_p -= sh.above;
    }
    PickSet set{0u, INT_MAX};
    const uint32_t key_high = key_of(highest_listed()), key_low = key_of(lowest_listed());
    if (!window && sh.n_list <= PICK_FEW) {
        pick_few<THREADS>(sh, weights, k, share, by_k, by_p, need_p, floor_y, u, out + r);
        return;
    }
    PickList list;
    list.turn = 0;
    int stage = by_k ? PICK_K : by_p ? PICK_P : PICK_DRAW;
    bool from_row = window || sh.n_list > ROOM;                   // the pick is made out of the row
    bool listed = sh.n_list <= ROOM;
    if (window && listed && sh.n_list <= PICK_FEW) {
        if (by_border) pick_border(sh, weights, need_p, set);     // (else, and where fewer are there, all of the bin stay)
        list.take(sh, weights, THREADS);
    } else if (!listed) {                                         // too many for the list as well: over the row itself
        if (by_k) pick_narrow<true>(sh, row, set, top, whole_scale, weights, (u64)k, -1.0);
        if (by_p) pick_narrow<false>(sh, row, set, top, whole_scale, weights, 0, share);
        stage = PICK_DRAW;
    } else if (window && !by_border) {
        list.take(sh, weights, THREADS);
    } else {
        list.take(sh, weights, THREADS);
        Found at;
        int ties_of = 0;                                          // (the search behind the ties)
        u64 ties = 0;
        uint32_t tie_key = 0;
        for (;;) {
            const bool by_index = stage == PICK_K_TIES || stage == PICK_P_TIES || stage == PICK_DRAW, one_each = stage == PICK_K || stage == PICK_K_TIES;
#pragma unroll
            for (int e = 0; e < PICK_EACH; ++e)
                if (e < list.n) {
                    const uint32_t key = key_of(list.x[e]);
                    bool in = set.has(key, list.index[e]);
                    if (stage == PICK_K_TIES || stage == PICK_P_TIES) in = in && key == tie_key;
                    if (stage == PICK_DRAW) in = in && weights.octaves(list.x[e]) >= floor_y;
                    list.counts[e] = !in ? 0 : one_each ? 1 : list.weight[e];
                    list.ord[e] = by_index ? (uint32_t)list.index[e] : ~key;
                }
            const bool reached = list_find(sh, list, by_index ? 0u : ~key_high, by_index ? (uint32_t)vocab - 1 : ~key_low, at, [&](u64 sum) {
                if (stage == PICK_K) return (u64)k;
                if (stage == PICK_P) return by_k ? max((u64)1, (u64)ceil(share * (double)sum)) : need_p;
                if (stage == PICK_DRAW) return passed_at(u, sum);
                return ties;
            });
            if (stage == PICK_DRAW) {
                if (tid == 0) out[r] = (int)at.ord;
                return;
            }
            if (stage == PICK_K || stage == PICK_P) {
                ties_of = 0;
                if (reached) {                                    // (else there are fewer: all stay)
                    const uint32_t key = ~at.ord;
                    set.cut = key == set.key ? set.cut : INT_MAX;
                    set.key = key;
                    // ties are alike in weight: where not all are needed it is those of the smallest indices that reach what is asked for
                    if (at.need < at.above + at.inside) {
                        ties_of = 1;
                        tie_key = key;
                        ties = at.need - at.above;
                    }
                }
            } else {
                set.cut = (int)at.ord;
                ties_of = 0;
            }
            stage = ties_of ? stage + 1 : stage <= PICK_K_TIES && by_p ? PICK_P : PICK_DRAW;
            if (stage == PICK_DRAW && from_row) break;
        }
    }
    // what is kept, as a logit: all above `edge`, and so many as it. min-p's own border is the smallest logit that passes it
    float edge = set.key ? float_of(set.key) : -INFINITY;
    int cut = set.cut;
    float lowest = fmaxf((float)((double)top + floor_y / c1), -FLT_MAX);      // (-inf where that is out of range, NaN for 0 octaves at an infinite temperature)
    auto next = [](float x, int up) { return float_of(key_of(x) + up); };
    for (int i = 0; i < 8 && weights.octaves(next(lowest, -1)) >= floor_y; ++i) lowest = next(lowest, -1);
    for (int i = 0; i < 16 && weights.octaves(lowest) < floor_y; ++i) lowest = next(lowest, 1);
    if (lowest > edge) {
        edge = lowest;
        cut = INT_MAX;
    }
    auto kept = [&](float x, int index) { return x > edge || (x == edge && index <= cut); };
    if (window && listed) {                                       // the runs' sums: what lies above the list's bin, and what is kept of it
        if (tid < WAVES) sh.waves[tid] = sh.turns[tid];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < PICK_EACH; ++e)
            if (e < list.n && kept(list.x[e], list.index[e]))
                atomicAdd(&sh.waves[(list.index[e] + row.skew) / (row.turns * 4 * WAVE)], list.weight[e]);
        __syncthreads();
        pick_in_runs(sh, row, u, weights, out + r, kept);
    } else {
        pick_from_row(sh, row, u, weights, out + r, kept);
    }
}

extern "C" int imparo_pick_rows(const float* logits, const float* temperature, const float* uniform, const int32_t* top_k,
                                const float* top_p, const float* min_p, int32_t* out, int n_rows, int vocab,
                                imparo_stream stream) {
    if (n_rows < 0 || vocab <= 0 || vocab > 1 << 19) return IMPARO_BAD_ARGUMENT;
    if (n_rows == 0) return IMPARO_OK;
    if (!logits || !temperature || !uniform || !out || ((uintptr_t)logits & 3)) return IMPARO_BAD_ARGUMENT;
    hipStream_t s = (hipStream_t)stream;
    k_pick_rows<<<n_rows, PICK_THREADS, 0, s>>>(logits, temperature, uniform, top_k, top_p, min_p, out, vocab);
    return launch_status();
}

// The hash of the sources this library was built from (given by the build), so that a
// library older than its sources is noticed when it is loaded.
#ifndef IMPARO_SOURCE_HASH
#define IMPARO_SOURCE_HASH "unknown"
#endif
extern "C" const char* imparo_hip_source_hash() { return IMPARO_SOURCE_HASH; }

// Asks the runtime about one kernel of this file, which makes it load the file's code onto the
// current device (it loads a file's kernels when one of them is first used; a stream under capture
// cannot do that).
int imparo_load_code_sampling() {
    hipFuncAttributes attributes;
    return hipFuncGetAttributes(&attributes, reinterpret_cast<const void*>(&k_argmax_rows)) == hipSuccess ? IMPARO_OK
                                                                                              : IMPARO_LAUNCH_FAILED;
}
