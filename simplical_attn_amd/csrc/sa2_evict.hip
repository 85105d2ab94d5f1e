// Eviction from a cache: of each sequence's rows the first ones, the latest ones and those that gathered most weight stay, in their order.
//
// Which ones: a workgroup per sequence and head finds the smallest weight that stays digit by digit (11, 11 and 10 bits of the weights
// as ordered integers, counted in LDS), then numbers the rows that stay, of equal ones the first.  Moving them: see move_kernel.
#include "sa2_layer_common.h"

namespace sa2 {
namespace {

constexpr int THREADS = 1024, BINS = 2048;

// Weights as integers of the same order; NaN is below all, zeros are equal
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ int evict_held(const Evict& p, int b) {
    const int64_t room = p.cache.table ? (int64_t)p.cache.width * p.cache.page_size : p.cache.page_size;
    const int n = p.cache.lengths[b];
    return n < 0 ? 0 : n > room ? (int)room : n;
}
// Sum over the threads before this one; `total`: over all.  `lds`: THREADS / 64 integers, free again at the next barrier but one
__device__ __forceinline__ int before_me(int x, int* lds, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(sum, o);
        if (lane >= o) sum += up;
    }
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    int base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        const int y = lds[w];
        base += w < wave ? y : 0;
        total += y;
    }
    return base + sum - x;
}

__global__ __launch_bounds__(THREADS) void choose_kernel(Evict p) {
    __shared__ int bins[BINS];
    __shared__ int sums[2][THREADS / 64];
    __shared__ int found[2];
    const int b = blockIdx.x / p.heads, h = blockIdx.x % p.heads, n = evict_held(p, b);
    const float* const w = p.weights + b * p.sb + h * p.sh;
    float* const left = p.left + (int64_t)blockIdx.x * p.places;
    int32_t* const kept = p.kept + (int64_t)blockIdx.x * p.keep;
    const int stay = n < p.keep ? n : p.keep;
    for (int64_t i = stay + threadIdx.x; i < p.places; i += THREADS) left[i] = 0.f;
    for (int i = stay + threadIdx.x; i < p.keep; i += THREADS) kept[i] = -1;
    if (n <= p.keep) {
        for (int i = threadIdx.x; i < n; i += THREADS) {
            left[i] = w[i];
            kept[i] = i;
        }
        return;
    }
    // the smallest weight of the rows from .. to - 1 that stays, and how many of that weight do
    const int from = p.first, to = n - p.recent;
    int need = p.keep - p.first - p.recent;
    uint32_t prefix = 0;
    if (need > 0) {
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass < 2 ? 11 : 10;
            for (int i = threadIdx.x; i < BINS; i += THREADS) bins[i] = 0;
            __syncthreads();
            for (int i = from + threadIdx.x; i < to; i += THREADS) {
                const uint32_t u = ordered(w[i]);
                if (pass == 0 || u >> (shift + width) == prefix) atomicAdd(&bins[u >> shift & ((1u << width) - 1)], 1);
            }
            __syncthreads();
            // from the highest bin down: the one in which the number that is needed is reached
            const int size = 1 << width, mine = size / THREADS;          // 2 or 1
            int count[2], total;
            count[0] = bins[size - 1 - mine * threadIdx.x];
            count[1] = mine == 2 ? bins[size - 2 - 2 * threadIdx.x] : 0;
            int above = before_me(count[0] + count[1], sums[0], total);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (j < mine && above < need && above + count[j] >= need) {
                    found[0] = size - 1 - mine * threadIdx.x - j;
                    found[1] = need - above;
                }
                above += count[j];
            }
            __syncthreads();
            prefix = prefix << width | (uint32_t)found[0];
            need = found[1];
        }
    }
    const bool any = p.keep > p.first + p.recent;
    // in their order: each thread four rows in a row
    constexpr int EACH = 4;
    int placed = 0, equal = 0;
    for (int base = 0; base < n; base += THREADS * EACH) {
        const int i0 = base + threadIdx.x * EACH;
        float x[EACH];
        bool sure[EACH], same[EACH];
        int ties = 0;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int i = i0 + j;
            x[j] = i < n ? w[i] : 0.f;
            const uint32_t u = ordered(x[j]);
            const bool free = i >= from && i < to;
            sure[j] = i < n && (!free || (any && u > prefix));
            same[j] = free && any && u == prefix;
            ties += same[j];
        }
        int total;
        int rank = equal + before_me(ties, sums[0], total);
        equal += total;
        int count = 0;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            if (same[j] && rank++ < need) sure[j] = true;
            count += sure[j];
        }
        int to_place = placed + before_me(count, sums[1], total);
        placed += total;
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            if (sure[j]) {
                left[to_place] = x[j];
                kept[to_place++] = i0 + j;
            }
    }
}

// Rows to their new places.  A workgroup has `SLICE` pieces of every row of one tensor of a sequence's head and takes the rows in steps:
// reads of a step end before its writes begin, and what later steps read lies behind what this one writes (kept[i] >= i).
constexpr int MOVERS = 256, SLICE = 4, STEP = 8 * MOVERS / SLICE;
template <class UNIT>
__global__ __launch_bounds__(MOVERS) void move_kernel(Evict p, int size, int pieces, int slices) {
    const int slice = blockIdx.x % slices, which = blockIdx.x / slices % 2, stream = blockIdx.x / slices / 2, b = stream / p.HK, hk = stream % p.HK;
    const int n = evict_held(p, b), piece = slice * SLICE + threadIdx.x % SLICE, mine = threadIdx.x / SLICE;
    if (n <= p.keep) return;
    const int32_t* const kept = p.kept + ((int64_t)b * p.heads + (p.heads > 1 ? hk : 0)) * p.keep;
    const Tensor& t = which ? p.cache.v : p.cache.k;
    auto row = [&](int r) -> UNIT* {
        int64_t page = b;
        int at = r;
        if (p.cache.table) {
            const int i = (int)((unsigned)r / (unsigned)p.cache.page_size);
            page = p.cache.table[(int64_t)b * p.cache.width + i];
            at = r - i * p.cache.page_size;
            if (page < 0 || page >= p.cache.pages) return nullptr;
        }
        return (UNIT*)((char*)t.p + t.off(page, at, hk) * size) + piece;
    };
    for (int i0 = 0; i0 < p.keep; i0 += STEP) {
        UNIT x[8];
        UNIT* to[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = i0 + u * (MOVERS / SLICE) + mine, from = i < p.keep ? kept[i] : -1;
            to[u] = nullptr;
            if (from > i && piece < pieces) {
                const UNIT* const src = row(from);
                if (src) {
                    to[u] = row(i);
                    x[u] = *src;
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (to[u]) *to[u] = x[u];
    }
}

}  // namespace

int launch_evict(const Evict& p, int dtype, hipStream_t st) {
    const int size = dtype == SA2_F32 ? 4 : 2;
    const bool wide = (p.D * size) % 16 == 0 && aligned16(p.cache.k, size, true) && aligned16(p.cache.v, size, true);
    const int pieces = wide ? p.D * size / 16 : p.D, slices = (pieces + SLICE - 1) / SLICE;
    const int64_t grid = (int64_t)p.B * p.HK * 2 * slices;
    if ((int64_t)p.B * p.heads > 0x7fffffff || grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    choose_kernel<<<dim3((unsigned)(p.B * p.heads)), dim3(THREADS), 0, st>>>(p);
    if (hipGetLastError() != hipSuccess) return SA2_ERR_LAUNCH_FAILED;
    const dim3 blocks((unsigned)grid), block(MOVERS);
    if (wide) move_kernel<uint4><<<blocks, block, 0, st>>>(p, size, pieces, slices);
    else if (size == 4) move_kernel<uint32_t><<<blocks, block, 0, st>>>(p, size, pieces, slices);
    else move_kernel<uint16_t><<<blocks, block, 0, st>>>(p, size, pieces, slices);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

}  // namespace sa2
