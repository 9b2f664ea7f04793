// Picking the next token from float32 logits: argmax (smallest index at the
// maximum, NaN never wins) and temperature sampling by inverse CDF.
#include "common.h"
#include "api.h"
#include <limits.h>

struct Best {
    float v;
    int i;
};

__device__ __forceinline__ Best better(Best a, Best b) {
    return (b.v > a.v || (b.v == a.v && b.i < a.i)) ? b : a;
}

__device__ __forceinline__ Best block_best(Best b, Best* scratch) {
    b = better(b, Best{lane_xor<32>(b.v), lane_xor<32>(b.i)});
    b = better(b, Best{lane_xor<16>(b.v), lane_xor<16>(b.i)});
    b = better(b, Best{lane_xor<8>(b.v), lane_xor<8>(b.i)});
    b = better(b, Best{lane_xor<4>(b.v), lane_xor<4>(b.i)});
    b = better(b, Best{lane_xor<2>(b.v), lane_xor<2>(b.i)});
    b = better(b, Best{lane_xor<1>(b.v), lane_xor<1>(b.i)});
    const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
    const int n_waves = (blockDim.x + WAVE - 1) / WAVE;
    __syncthreads();
    if (lane == 0) scratch[wave] = b;
    __syncthreads();
    Best r = scratch[0];
    for (int w = 1; w < n_waves; ++w) r = better(r, scratch[w]);
    return r;
}

__device__ __forceinline__ Best row_best(const float* __restrict__ row, int vocab, Best* scratch) {
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
        if (n4 <= (int)blockDim.x) {
            // one load a thread: the maximum and its index together, one meeting of the block (a row of 1,000 in two 3.8 us)
            const float4 v = row4[min((int)threadIdx.x, n4 - 1)];
            const float vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if ((int)threadIdx.x < n4 && (vs[j] > b.v || (vs[j] == b.v && 4 * (int)threadIdx.x + j < b.i))) {
                    b.v = vs[j];
                    b.i = 4 * (int)threadIdx.x + j;
                }
            b = block_best(b, scratch);
            if (b.i == INT_MAX) b.i = 0;   // every value was NaN
            return b;
        }
        constexpr int DEEP = 16;
        float m = -INFINITY;
        int met = 0;
        for (int first = threadIdx.x; first < n4; first += DEEP * (int)blockDim.x) {
            float4 v[DEEP];
#pragma unroll
            for (int k = 0; k < DEEP; ++k) v[k] = row4[min(first + k * (int)blockDim.x, n4 - 1)];
            float mm = -INFINITY;
#pragma unroll
            for (int k = 0; k < DEEP; ++k) mm = fmaxf(mm, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
            if (mm > m) {
                m = mm;
                met = first;
            }
        }
        float top = wave_max(m);
        const int n_waves = (blockDim.x + WAVE - 1) / WAVE;
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
                for (int k = 0; k < DEEP; ++k) v[k] = row4[min(met + k * (int)blockDim.x, n4 - 1)];
#pragma unroll
                for (int k = DEEP - 1; k >= 0; --k) {
                    const int i = min(met + k * (int)blockDim.x, n4 - 1);
                    const float vs[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
                    for (int j = 3; j >= 0; --j)
                        if (vs[j] == top) b.i = 4 * i + j;
                }
                b.v = top;
            }
            return block_best(b, scratch);
        }
    }
    for (int i = threadIdx.x; i < vocab; i += blockDim.x) {
        const float v = row[i];
        if (v > b.v || (v == b.v && i < b.i)) {
            b.v = v;
            b.i = i;
        }
    }
    b = block_best(b, scratch);
    if (b.i == INT_MAX) b.i = 0;   // every value was NaN
    return b;
}

__global__ void k_argmax_rows(const float* __restrict__ logits, int32_t* __restrict__ out, int vocab) {
    __shared__ Best scratch[16];
    const Best b = row_best(logits + (size_t)blockIdx.x * vocab, vocab, scratch);
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
                                           int vocab) {
    __shared__ Best scratch[16];
    __shared__ __attribute__((aligned(16))) float sums[SAMPLE_THREADS], before[SAMPLE_THREADS];
    __shared__ int first_past, last_positive, found;
    __shared__ float cum_shared, target_shared;
    const Best top = row_best(row, vocab, scratch);
    if (!(temp > 0.f)) {
        if (threadIdx.x == 0) *out = top.i;
        return;
    }
    const float inv_t = 1.0f / temp;
    const int tid = threadIdx.x, threads = blockDim.x;         // (a multiple of 16)
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
    sample_row(logits + (size_t)blockIdx.x * vocab, temperature[blockIdx.x], uniform[blockIdx.x], out + blockIdx.x, vocab);
}

extern "C" int imparo_sample_rows(const float* logits, const float* temperature, const float* uniform, int32_t* out,
                                  int n_rows, int vocab, imparo_stream stream) {
    if (!logits || !temperature || !uniform || !out || n_rows < 0 || vocab <= 0) return IMPARO_BAD_ARGUMENT;
    if (n_rows == 0) return IMPARO_OK;
    const int threads = vocab >= 16384 ? SAMPLE_THREADS : 256;
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
// The border is found without sorting: a histogram in LDS, linear in the logit over the range that weighs anything, a scan for the bin
// where the count (or the weight) is reached, and the same again inside that bin over its keys' bits until one key is left.
// One block a row, which reads it again for each pass (out of L2).
#define PICK_BINS 2048
#define PICK_LIST 2048
#define PICK_CUT 44

typedef unsigned long long u64;

// the float's place in the order of floats
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// 2^y 2^44 to the nearest integer, y <= 0 (0 below 2^-44.5): 2^f = e^(f ln 2) of the fraction |f| <= 1/2 as its power series, cut where the next
// term is below 2^-47, then scaled by the exponent and rounded by an addition of 2^52
__device__ __forceinline__ u64 weight_of(double y) {
    const double k = rint(y), f = (y - k) * 0.69314718055994530942;
    double p = fma(f, 1.0 / 39916800.0, 1.0 / 3628800.0);
    p = fma(f, p, 1.0 / 362880.0);
    p = fma(f, p, 1.0 / 40320.0);
    p = fma(f, p, 1.0 / 5040.0);
    p = fma(f, p, 1.0 / 720.0);
    p = fma(f, p, 1.0 / 120.0);
    p = fma(f, p, 1.0 / 24.0);
    p = fma(f, p, 1.0 / 6.0);
    p = fma(f, p, 0.5);
    p = fma(f, p, 1.0);
    p = fma(f, p, 1.0);
    const double scaled = __hiloint2double(__double2hiint(p) + (((int)k + PICK_CUT) << 20), __double2loint(p));
    return y < -(PICK_CUT + 0.5) ? 0 : (u64)__double_as_longlong(scaled + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
}

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
__device__ __forceinline__ u64 wave_scan_u64(u64 v) {             // the sum over the lanes up to and with this one
    const int lane = threadIdx.x & (WAVE - 1);
#pragma unroll
    for (int n = 1; n < WAVE; n <<= 1) {
        const u64 below = __shfl_up(v, n, WAVE);
        if (lane >= n) v += below;
    }
    return v;
}

struct PickShared {
    u64 hist[PICK_BINS];
    uint32_t list[PICK_LIST];
    u64 waves[16];
    float tops[16], lows[16];
    u64 above, inside, total, need;   // of the bin where the sum is reached: what lies above it, what it holds; all there is; what is asked for
    int bin, n_list;
    uint32_t key_low, key_high;
    int cut;
};

// The bin of sh.hist where the running sum reaches what is asked for: `need`, or for share >= 0 that share of all. Leaves bin,
// above, inside, total and need in LDS; every thread calls, behind and ahead of a barrier of its own.
__device__ __forceinline__ void pick_bin(PickShared& sh, u64 need, double share) {
    const int threads = blockDim.x, per = PICK_BINS / threads, tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    u64 mine = 0;
    for (int i = 0; i < per; ++i) mine += sh.hist[tid * per + i];
    const u64 upto = wave_scan_u64(mine);
    if (lane == WAVE - 1) sh.waves[wave] = upto;
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
        sh.total = total;
        sh.need = need;
    }
    __syncthreads();
}

// A row's logits, lane by lane: wave w has the values of its own run, 256 a turn, four neighbours a lane. What stands in front of
// the row or behind it inside the 16 aligned bytes that hold its first or last value is read with them (the same 16 bytes of
// memory, so it is there) and counts as -inf, as NaN does.
#define PICK_DEEP 8
struct PickRow {
    const float4* base;
    int skew, vocab, turns, first;      // first: index in the row of this lane's first value in turn 0

    __device__ __forceinline__ void open(const float* row, int n) {
        vocab = n;
        skew = (int)(((uintptr_t)row & 15) >> 2);
        base = reinterpret_cast<const float4*>(row - skew);
        const int waves = blockDim.x / WAVE, lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
        turns = (vocab + skew + 4 * WAVE * waves - 1) / (4 * WAVE * waves);
        first = wave * turns * 4 * WAVE + 4 * lane - skew;
    }
    // f(values, index of the first of the four), turn after turn, the loads of PICK_DEEP turns in flight
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int c0 = 0; c0 < turns; c0 += PICK_DEEP) {
            float4 v[PICK_DEEP];
#pragma unroll
            for (int c = 0; c < PICK_DEEP; ++c)
                v[c] = base[min(max(first + skew + (c0 + c) * 4 * WAVE, 0), vocab + skew - 1) >> 2];
#pragma unroll
            for (int c = 0; c < PICK_DEEP; ++c) {
                if (c0 + c >= turns) break;
                const int i = first + (c0 + c) * 4 * WAVE;
                float x[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool on = i + j >= 0 && i + j < vocab && x[j] == x[j];
                    x[j] = on ? x[j] + 0.f : -INFINITY;          // (+ 0: -0 and 0 are one value)
                }
                f(x, i);
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

// Narrows `set` to the beginning of its order where the count (COUNT) reaches `need`, or the weights the share `share` of theirs.
template <bool COUNT>
__device__ __forceinline__ void pick_narrow(PickShared& sh, const PickRow& row, PickSet& set, float top, float bin_scale,
                                            float reach, float c1f, double c1, u64 need, double share) {
    const int tid = threadIdx.x, threads = blockDim.x;
    auto weight = [&](float x) { return COUNT ? (u64)1 : weight_of(((double)x - (double)top) * c1); };
    auto bin_of = [&](float x) { return (int)fminf((top - x) * bin_scale, (float)(PICK_BINS - 1)); };
    for (int b = tid; b < PICK_BINS; b += threads) sh.hist[b] = 0;
    if (tid == 0) {
        sh.n_list = 0;
        sh.key_low = 0xFFFFFFFFu;
        sh.key_high = 0;
        sh.total = 0;
    }
    __syncthreads();
    row.each([&](const float (&x)[4], int index) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (x[j] >= reach && set.has(key_of(x[j]), index + j)) atomicAdd(&sh.hist[bin_of(x[j])], weight(x[j]));
    });
    __syncthreads();
    pick_bin(sh, need, share);
    if (sh.total == 0) return;                                    // fewer than are asked for: all stay
    u64 above = sh.above;
    need = sh.need;
    const int bin = sh.bin;
    row.each([&](const float (&x)[4], int index) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!(x[j] >= reach) || bin_of(x[j]) != bin) continue;
            const uint32_t k = key_of(x[j]);
            if (!set.has(k, index + j)) continue;
            const int at = atomicAdd(&sh.n_list, 1);
            if (at < PICK_LIST) sh.list[at] = k;
            atomicMin(&sh.key_low, k);
            atomicMax(&sh.key_high, k);
        }
    });
    __syncthreads();
    const int n_list = sh.n_list;
    uint32_t low = sh.key_low, high = sh.key_high;
    u64 inside = sh.inside;
    while (low != high) {                                         // (at most three times: 11 bits of at most 32 each)
        const int bits = 32 - __clz((int)(high - low)), shift = max(0, bits - 11);
        __syncthreads();
        for (int b = tid; b < PICK_BINS; b += threads) sh.hist[b] = 0;
        __syncthreads();
        auto float_of = [](uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); };
        if (n_list <= PICK_LIST) {
            for (int i = tid; i < n_list; i += threads) {
                const uint32_t k = sh.list[i];
                if (k >= low && k <= high) atomicAdd(&sh.hist[(high - k) >> shift], weight(float_of(k)));
            }
        } else {
            row.each([&](const float (&x)[4], int index) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t k = key_of(x[j]);
                    if (x[j] >= reach && k >= low && k <= high && set.has(k, index + j)) atomicAdd(&sh.hist[(high - k) >> shift], weight(x[j]));
                }
            });
        }
        __syncthreads();
        pick_bin(sh, need - above, -1.0);
        above += sh.above;
        inside = sh.inside;
        high -= (uint32_t)sh.bin << shift;
        low = high - low > (1u << shift) - 1 ? high - ((1u << shift) - 1) : low;
    }
    // one key is left: so many of its tokens, in the order of their indices, reach what is asked for
    const u64 each = weight(__uint_as_float(high & 0x80000000u ? high ^ 0x80000000u : ~high));
    const u64 ties = (need - above + each - 1) / each;
    const PickSet old = set;
    set.key = high;
    set.cut = INT_MAX;
    if (ties * each >= inside) {                                  // all of them
        if (high == old.key) set.cut = old.cut;
        return;
    }
    const int lane = tid & (WAVE - 1), wave = tid / WAVE;
    u64 mine = 0;
    row.each([&](const float (&x)[4], int index) {
#pragma unroll
        for (int j = 0; j < 4; ++j) mine += __popcll(__ballot(x[j] >= reach && key_of(x[j]) == high));
    });
    if (lane == 0) sh.waves[wave] = mine;
    __syncthreads();
    u64 before = 0;
    for (int w = 0; w < wave; ++w) before += sh.waves[w];
    if (before < ties && ties <= before + mine) {
        row.each([&](const float (&x)[4], int index) {
            u64 ahead = before;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool on = x[j] >= reach && key_of(x[j]) == high;
                const u64 who = __ballot(on);
                ahead += __popcll(who & ((1ull << lane) - 1));
                before += __popcll(who);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (x[j] >= reach && key_of(x[j]) == high && ++ahead == ties) sh.cut = index + j;
        });
    }
    __syncthreads();
    set.cut = sh.cut;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_pick_rows(
    const float* __restrict__ logits, const float* __restrict__ temperature, const float* __restrict__ uniform,
    const int32_t* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p,
    int32_t* __restrict__ out, int vocab) {
    __shared__ PickShared sh;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const float* row_at = logits + (size_t)r * vocab;
    const float temp = temperature[r], u = uniform[r];
    const int k = top_k ? top_k[r] : 0;
    const float p = top_p ? top_p[r] : 1.f, mp = min_p ? min_p[r] : 0.f;
    const bool by_k = k > 0 && k < vocab, by_p = p < 1.f, by_m = mp > 0.f;
    if (!(temp > 0.f) || !(by_k || by_p || by_m)) {               // greedy, or the whole distribution
        sample_row(row_at, temp, u, out + r, vocab);
        return;
    }
    PickRow row;
    row.open(row_at, vocab);
    float top = -INFINITY, low = INFINITY;
    row.each([&](const float (&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            top = fmaxf(top, x[j]);
            low = fminf(low, x[j] > -INFINITY ? x[j] : INFINITY);
        }
    });
    top = wave_max(top);
    low = -wave_max(-low);
    if (lane == 0) {
        sh.tops[wave] = top;
        sh.lows[wave] = low;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / WAVE; ++w) {
        top = fmaxf(top, sh.tops[w]);
        low = fminf(low, sh.lows[w]);
    }
    if (!(top < INFINITY) || !(top > -INFINITY)) {                // an infinite logit takes it, or there is none to take
        sample_row(row_at, 0.f, u, out + r, vocab);
        return;
    }
    const double c1 = 1.44269504088896340736 / (double)temp;
    const float c1f = fminf((float)c1, 3.0e38f);
    // logits below `reach` weigh nothing; a token that min-p takes out is not looked at again either, as every smaller one goes too
    const double floor_y = by_m ? fmax(-(double)PICK_CUT, log2((double)fminf(mp, 1.f))) : -(double)PICK_CUT;
    const float span = fminf(top - low, (float)PICK_CUT / c1f);
    const float reach = fmaxf(low, top - (float)PICK_CUT / c1f);
    const float bin_scale = span > 1e-30f && span < 1e30f ? (float)PICK_BINS * 0.99999f / span : 0.f;
    PickSet set{0u, INT_MAX};
    if (by_k) pick_narrow<true>(sh, row, set, top, bin_scale, reach, c1f, c1, (u64)k, -1.0);
    __syncthreads();
    if (by_p) pick_narrow<false>(sh, row, set, top, bin_scale, reach, c1f, c1, 0, (double)fmaxf(p, 0.f));
    __syncthreads();

    // ---- the pick: sums over the waves' runs, then inside the run where u falls
    auto kept = [&](float x, int index) {
        return x >= reach && set.has(key_of(x), index) && ((double)x - (double)top) * c1 >= floor_y;
    };
    u64 mine = 0;
    int last = -1;
    row.each([&](const float (&x)[4], int index) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (kept(x[j], index + j)) {
                mine += weight_of(((double)x[j] - (double)top) * c1);
                last = index + j;
            }
    });
    mine = wave_sum_u64(mine);
    if (lane == 0) sh.waves[wave] = mine;
    if (tid == 0) sh.cut = -1;
    __syncthreads();
    u64 before = 0, total = 0;
    for (int w = 0; w < THREADS / WAVE; ++w) {
        before += w < wave ? sh.waves[w] : 0;
        total += sh.waves[w];
    }
    const double want = fmax((double)u * (double)total, 0.0);     // (a NaN is 0)
    if (!(want < (double)total)) {                                // u of 1: the last token that is kept
        if (last >= 0) atomicMax(&sh.cut, last);
        __syncthreads();
        if (tid == 0) out[r] = sh.cut;
        return;
    }
    const u64 target = min((u64)want, total - 1);
    if (before <= target && target < before + mine) {
        int found = -1;
        row.each([&](const float (&x)[4], int index) {
            if (found >= 0) return;
            u64 w[4], four = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = kept(x[j], index + j) ? weight_of(((double)x[j] - (double)top) * c1) : 0;
                four += w[j];
            }
            if (!__any(four != 0)) return;
            const u64 upto = wave_scan_u64(four);
            const u64 past = __ballot(before + upto > target);
            if (past) {
                u64 at = before + upto - four;
                int pick = -1;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    at += w[j];
                    if (pick < 0 && at > target) pick = index + j;
                }
                found = __shfl(pick, __ffsll((long long)past) - 1, WAVE);
            }
            before += __shfl(upto, WAVE - 1, WAVE);
        });
        if (lane == 0) out[r] = found;
    }
}

extern "C" int imparo_pick_rows(const float* logits, const float* temperature, const float* uniform, const int32_t* top_k,
                                const float* top_p, const float* min_p, int32_t* out, int n_rows, int vocab,
                                imparo_stream stream) {
    if (n_rows < 0 || vocab <= 0 || vocab > 1 << 19) return IMPARO_BAD_ARGUMENT;
    if (n_rows == 0) return IMPARO_OK;
    if (!logits || !temperature || !uniform || !out || ((uintptr_t)logits & 3)) return IMPARO_BAD_ARGUMENT;
    hipStream_t s = (hipStream_t)stream;
    // (a row without a filter goes through sample_row, whose sums depend on the threads: as many as imparo_sample_rows has)
    if (vocab >= 16384) k_pick_rows<1024><<<n_rows, 1024, 0, s>>>(logits, temperature, uniform, top_k, top_p, min_p, out, vocab);
    else k_pick_rows<256><<<n_rows, 256, 0, s>>>(logits, temperature, uniform, top_k, top_p, min_p, out, vocab);
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
