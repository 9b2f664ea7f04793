// The index arrays of a step, made on the GPU from the requests' lengths: block tables, positions, slots and the list of rows, for
// a loop that keeps its lengths on the device (the engine's own steps are packed on the host).
#include "common.h"
#include "api.h"

#define TABLES_ROWS 4096          // rows a step may have: their running sums stand in LDS
#define TABLES_THREADS 256

struct TableRows {
    const int32_t* lengths;
    const int32_t* new_tokens;
    const int32_t* leader;        // or null: no row takes pages over
    const int32_t* shared;
    int page_shift, n_rows;
    // (a row's last position and its pages, where they are pages of one token, may pass 2^31: unsigned)
    __device__ __forceinline__ uint32_t length(int r) const { return (uint32_t)max(lengths[r], 0); }
    __device__ __forceinline__ int brings(int r) const { return max(new_tokens[r], 0); }
    __device__ __forceinline__ uint32_t need(int r) const {
        const uint32_t tokens = length(r) + (uint32_t)brings(r);
        return (tokens >> page_shift) + ((tokens & ((1u << page_shift) - 1)) != 0);
    }
    __device__ __forceinline__ uint32_t taken(int r) const { return leader ? min((uint32_t)max(shared[r], 0), need(r)) : 0; }
};

// Every block adds up all rows (a row's first page and first token are sums over the rows before it; a few reads a thread, and no
// second launch), then fills one row's table and tokens, a share of them where rows are long (grid y). An entry that a row
// takes over is looked up in its leader's own pages, through the leader's leader where that one took it over too. Bound by its launch and the
// trips to memory behind one another (lengths, sums through LDS, pages): 8 rows 4.8 us, 64 rows of 2,080 pages with portions of up to 512 tokens
// 8.2, 256 rows of 4,097 pages (4 MB of tables) 9.0.
__global__ __launch_bounds__(TABLES_THREADS) void k_step_tables(
    TableRows rows, const int32_t* __restrict__ pages, int n_pages, int32_t* __restrict__ table, int width,
    int32_t* __restrict__ seg_start, int32_t* __restrict__ positions, int32_t* __restrict__ row_of_token,
    int64_t* __restrict__ slots, int n_tokens, int32_t* __restrict__ lists, int32_t* __restrict__ counts) {
    __shared__ long long first_page[TABLES_ROWS];
    __shared__ long long wave_pages[TABLES_THREADS / WAVE], wave_tokens[TABLES_THREADS / WAVE];
    __shared__ int wave_singles[TABLES_THREADS / WAVE], wave_others[TABLES_THREADS / WAVE];
    __shared__ long long start_shared;
    __shared__ int singles_before, others_before;
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE, r = blockIdx.x, n = rows.n_rows;
    const int per = (n + TABLES_THREADS - 1) / TABLES_THREADS, begin = min(n, tid * per), end = min(n, begin + per);
    long long own = 0, tokens = 0;
    int singles = 0, others = 0;
    for (int i = begin; i < end; ++i) {
        const int b = rows.brings(i);
        own += rows.need(i) - rows.taken(i);
        tokens += b;
        singles += b == 1;
        others += b > 1;
    }
    long long own_upto = own, tokens_upto = tokens;
    int singles_upto = singles, others_upto = others;
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) {
        const long long p = __shfl_up(own_upto, d, WAVE), t = __shfl_up(tokens_upto, d, WAVE);
        const int s = __shfl_up(singles_upto, d, WAVE), o = __shfl_up(others_upto, d, WAVE);
        if (lane >= d) own_upto += p, tokens_upto += t, singles_upto += s, others_upto += o;
    }
    if (lane == WAVE - 1) {
        wave_pages[wave] = own_upto;
        wave_tokens[wave] = tokens_upto;
        wave_singles[wave] = singles_upto;
        wave_others[wave] = others_upto;
    }
    __syncthreads();
    long long page = own_upto - own, token = tokens_upto - tokens, all_pages = 0, all_tokens = 0;
    int single = singles_upto - singles, other = others_upto - others, all_singles = 0, all_others = 0;
#pragma unroll
    for (int w = 0; w < TABLES_THREADS / WAVE; ++w) {
        if (w < wave) page += wave_pages[w], token += wave_tokens[w], single += wave_singles[w], other += wave_others[w];
        all_pages += wave_pages[w], all_tokens += wave_tokens[w], all_singles += wave_singles[w], all_others += wave_others[w];
    }
    for (int i = begin; i < end; ++i) {
        const int b = rows.brings(i);
        first_page[i] = page;
        if (i == r) {
            start_shared = token;
            singles_before = single;
            others_before = other;
        }
        page += rows.need(i) - rows.taken(i);
        token += b;
        single += b == 1;
        other += b > 1;
    }
    __syncthreads();

    const int ps = rows.page_shift;
    auto entry = [&](int row, uint32_t j) -> int {                // what stands at place j of a row's table
        if (j >= rows.need(row)) return -1;
        for (int hops = 0; hops < n; ++hops) {
            const uint32_t taken = rows.taken(row);
            if (j >= taken) {
                if (j >= rows.need(row)) return -1;               // (its leader is shorter than what was to be taken over)
                const long long at = first_page[row] + (j - taken);
                return at < n_pages ? pages[at] : -1;
            }
            row = rows.leader[row];
            if (row < 0 || row >= n) return -1;
        }
        return -1;                                                // (leaders in a circle)
    };
    const int step = gridDim.y * TABLES_THREADS, at = blockIdx.y * TABLES_THREADS + tid;
    for (int j = at; j < width; j += step) table[(size_t)r * width + j] = entry(r, j);
    const long long start = start_shared;
    const uint32_t length = rows.length(r);
    const int b = rows.brings(r);
    for (int i = at; i < b && start + i < n_tokens; i += step) {
        const uint32_t pos = length + (uint32_t)i;
        positions[start + i] = (int32_t)min(pos, (uint32_t)INT32_MAX);
        row_of_token[start + i] = r;
        if (slots) {
            const int p = entry(r, pos >> ps);
            slots[start + i] = p < 0 ? -1 : ((int64_t)p << ps) + (pos & ((1 << ps) - 1));
        }
    }
    if (blockIdx.y == 0 && tid == 0) {
        seg_start[r] = (int32_t)min(start, (long long)INT32_MAX);
        if (b == 1) lists[singles_before] = r;
        if (b > 1) lists[all_singles + others_before] = r;
        if (r == 0) {
            counts[0] = (int32_t)min(all_tokens, (long long)INT32_MAX);
            counts[1] = (int32_t)min(all_pages, (long long)INT32_MAX);
            counts[2] = all_singles;
            counts[3] = all_others;
        }
    }
}

extern "C" int imparo_step_tables_max_rows() { return TABLES_ROWS; }

extern "C" int imparo_step_tables(const int32_t* lengths, const int32_t* new_tokens, const int32_t* leader, const int32_t* shared,
                                  const int32_t* pages, int n_pages, int page_size, int n_rows, int32_t* table, int width,
                                  int32_t* seg_start, int32_t* positions, int32_t* row_of_token, int64_t* slots, int n_tokens,
                                  int32_t* lists, int32_t* counts, imparo_stream stream) {
    if (!lengths || !new_tokens || (leader == nullptr) != (shared == nullptr) || n_pages < 0 || (n_pages && !pages) || n_rows < 0 ||
        n_rows > TABLES_ROWS || width < 1 || n_tokens < 0 || (n_tokens && (!positions || !row_of_token)) || !table || !seg_start ||
        !lists || !counts || page_size < 1 || (page_size & (page_size - 1)))
        return IMPARO_BAD_ARGUMENT;
    if (n_rows == 0) return IMPARO_OK;
    const TableRows rows{lengths, new_tokens, leader, shared, __builtin_ctz((unsigned)page_size), n_rows};
    // (a block a row, more where a row's table or tokens may be long: 2,048 of them a block)
    const int longest = width > n_tokens ? width : n_tokens;
    const dim3 grid(n_rows, longest < 2048 * 32 ? (longest + 2047) / 2048 : 32);
    k_step_tables<<<grid, TABLES_THREADS, 0, (hipStream_t)stream>>>(rows, pages, n_pages, table, width, seg_start, positions,
                                                                    row_of_token, slots, n_tokens, lists, counts);
    return launch_status();
}

int imparo_load_code_step_tables() {
    hipFuncAttributes attributes;
    return hipFuncGetAttributes(&attributes, reinterpret_cast<const void*>(&k_step_tables)) == hipSuccess ? IMPARO_OK
                                                                                              : IMPARO_LAUNCH_FAILED;
}
