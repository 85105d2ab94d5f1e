// Eviction from a cache: of each sequence's rows the first ones, the latest ones and those that gathered most weight stay, in their order.
//
// Which ones: up to four workgroups per sequence and head find the smallest weight that stays digit by digit (11, 11 and 10 bits of the weights
// as ordered integers, counted in LDS), each for itself, then number a part of the rows that stay, of equal ones the first.  Bound by a CU's vector
// ALU, which has all weights three times and its part once more: 65536 of them take 50 us with four workgroups (56 where they come from memory) and 64
// with one, 2000 10 with one (the unrolled form that keeps them in registers is fetched cold: 31).  Moving them: see move_kernel.
#include "sa2_layer_common.h"

namespace sa2 {
namespace {

constexpr int THREADS = 1024, BINS = 2048, COPIES = 8;      // (lanes count in one of 8 copies: weights of few magnitudes fall into few bins)
constexpr int CREW = THREADS / 64;

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

__global__ __launch_bounds__(THREADS) void choose_kernel(Evict p, int parts) {
    __shared__ __attribute__((aligned(16))) int bins[BINS * COPIES];
    __shared__ int sums[2 * CREW];
    __shared__ int found[2];
    const int stream = blockIdx.x / parts, part = blockIdx.x % parts, b = stream / p.heads, h = stream % p.heads, n = evict_held(p, b), me = part * THREADS + threadIdx.x, all_of_us = parts * THREADS;
    const float* const w = p.weights + b * p.sb + h * p.sh;
    float* const left = p.left + (int64_t)stream * p.places;
    int32_t* const kept = p.kept + (int64_t)stream * p.keep;
    const int stay = n < p.keep ? n : p.keep;
    for (int64_t i = (int64_t)stay + me; i < p.places; i += all_of_us) left[i] = 0.f;
    for (int64_t i = (int64_t)stay + me; i < p.keep; i += all_of_us) kept[i] = -1;
    if (n <= p.keep) {
        for (int64_t i = me; i < n; i += all_of_us) {
            left[i] = w[i];
            kept[i] = (int)i;
        }
        return;
    }
    // the smallest weight of the rows from .. to - 1 that stays, and how many of that weight do
    const int from = p.first, to = n - p.recent, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int need = p.keep - p.first - p.recent;
    const bool any = need > 0;
    uint32_t prefix = 0;
    if (any) {
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass < 2 ? 11 : 10;
            for (int i = threadIdx.x; i < BINS * COPIES / 4; i += THREADS) ((int4*)bins)[i] = make_int4(0, 0, 0, 0);
            __syncthreads();
            const auto tally = [&](float x) {
                const uint32_t u = ordered(x);
                if (pass == 0 || u >> (shift + width) == prefix) atomicAdd(&bins[(u >> shift & ((1u << width) - 1)) * COPIES + threadIdx.x % COPIES], 1);
            };
            int64_t i = (int64_t)from + threadIdx.x;
#pragma unroll 1
            for (; i + 7 * THREADS < to; i += 8 * THREADS) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = w[i + j * THREADS];
#pragma unroll
                for (int j = 0; j < 8; ++j) tally(x[j]);
            }
#pragma unroll 1
            for (; i < to; i += THREADS) tally(w[i]);
            __syncthreads();
            // from the highest bin down: the one in which the number that is needed is reached
            const int size = 1 << width, mine = size / THREADS;          // 2 or 1
            int count[2], total;
            const auto of = [&](int bin) {
                const int4 l = ((const int4*)bins)[2 * bin], h = ((const int4*)bins)[2 * bin + 1];
                return l.x + l.y + l.z + l.w + h.x + h.y + h.z + h.w;
            };
            count[0] = of(size - 1 - mine * threadIdx.x);
            count[1] = mine == 2 ? of(size - 2 - 2 * threadIdx.x) : 0;
            int above = before_me(count[0] + count[1], sums, total);
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
    // In their order, 4096 rows at a time: before a row stand the sure ones before it and, of equal weights, no more than are needed.  Within a
    // wavefront these are bits of ballots, the wavefronts' numbers (sure ones and, 16 bits up, equal ones) go over LDS.
    // Each of the workgroups that share a head numbers its part, and counts what stands before that.
    const auto kind = [&](int64_t i, float weight) {       // 2: stays, 1: of the smallest weight that does
        const uint32_t u = ordered(weight);
        return i >= n ? 0 : i < from || i >= to ? 2 : !any ? 0 : u > prefix ? 2 : u == prefix ? 1 : 0;
    };
    const int steps = (int)(((int64_t)n + 4 * THREADS - 1) / (4 * THREADS));
    const int64_t begin = (int64_t)steps * part / parts * 4 * THREADS, end = (int64_t)steps * (part + 1) / parts * 4 * THREADS;
    int sure_before = 0, same_before = 0;
    if (begin) {
        int sure = 0, same = 0;
#pragma unroll 8
        for (int64_t i = threadIdx.x; i < begin; i += THREADS) {         // (all before n)
            const int what = kind(i, w[i]);
            sure += what == 2;
            same += what == 1;
        }
        before_me(sure, sums, sure_before);
        before_me(same, sums + CREW, same_before);
        __syncthreads();
    }
    const uint64_t lower = ((uint64_t)1 << lane) - 1;
    float x[4], next[4];
    const auto load = [&](int64_t base, float (&to)[4]) {
        const int64_t i = base + 4 * (int)threadIdx.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) to[j] = i + j < n ? w[i + j] : 0.f;
    };
    load(begin, x);
    int turn = 0;
#pragma unroll 1
    for (int64_t base = begin; base < end; base += 4 * THREADS, turn ^= 1) {
        load(base + 4 * THREADS, next);
        const int64_t i = base + 4 * (int)threadIdx.x;
        bool sure[4], same[4];
        int before = 0, all = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int what = kind(i + j, x[j]);
            sure[j] = what == 2;
            same[j] = what == 1;
            const uint64_t of_sure = __ballot(sure[j]), of_same = __ballot(same[j]);
            before += __popcll(of_sure & lower) + (__popcll(of_same & lower) << 16);
            all += __popcll(of_sure) + (__popcll(of_same) << 16);
        }
        if (lane == 0) sums[turn * CREW + wave] = all;
        __syncthreads();
        all = 0;
#pragma unroll
        for (int c = 0; c < CREW; ++c) {
            const int y = sums[turn * CREW + c];
            before += c < wave ? y : 0;
            all += y;
        }
        int place = sure_before + (before & 0xffff), equal = same_before + (before >> 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (sure[j] || (same[j] && equal < need)) {
                const int64_t to = place + (int64_t)(equal < need ? equal : need);
                left[to] = x[j];
                kept[to] = (int)i + j;
            }
            place += sure[j];
            equal += same[j];
            x[j] = next[j];
        }
        sure_before += all & 0xffff;
        same_before += all >> 16;
    }
}

// Rows to their new places.  A workgroup has `SLICE` pieces of every row of one tensor of a sequence's head and takes the rows in steps.  What
// the rows of a step lie behind is not written before them (kept[i] >= i), so that reads may run ahead of writes, never behind: each step's
// rows are asked for a step early, their pages two and their numbers three, and a step's writes begin when all of its reads have ended.
// 16384 rows of 256 bytes of 16 heads: 104 us (2.6 TB/s read and written) by 256 workgroups with two pieces, and where the call before left these
// rows in the card's last cache 88, by 128 workgroups with four pieces 98; 1024 rows of 32 heads: 10 us with four pieces, 15 with two.  One step at a
// time, without the reads ahead, 380 and 26.
typedef uint32_t Quad __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint32_t word(Quad x) { return x.x; }
__device__ __forceinline__ uint32_t word(uint32_t x) { return x; }
constexpr int MOVERS = 512, EACH = 8;
// r / d = r * factor >> shift for r < 2^31: with 2^l >= d, factor d = 2^(31 + l) + e, 0 < e <= 2^l, the product's error is below 1 / d
struct Quotient {
    uint32_t factor;
    int shift;
};
Quotient quotient(uint32_t d) {
    int l = 0;
    while ((uint64_t)1 << l < d) ++l;
    return Quotient{(uint32_t)(((uint64_t)1 << (31 + l)) / d + 1), 31 + l};
}
__device__ const Quad nothing = {0, 0, 0, 0};
template <class UNIT, int SLICE>
__global__ __launch_bounds__(MOVERS) void move_kernel(Evict p, Quotient pages_in, int size, int pieces, int slices) {
    constexpr int STEP = EACH * MOVERS / SLICE;
    int slice, stream;                                      // slices of the same rows on the same XCD, whose cache lines they share
    const int streams = p.B * p.HK * 2, pid = blockIdx.x;
    if (streams % 8 == 0) {
        slice = (pid >> 3) % slices;
        stream = (pid >> 3) / slices * 8 + (pid & 7);
    } else {
        slice = pid / streams;
        stream = pid % streams;
    }
    const int which = stream & 1, b = (stream >> 1) / p.HK, hk = (stream >> 1) % p.HK;
    const int n = evict_held(p, b), piece = slice * SLICE + threadIdx.x % SLICE, mine = threadIdx.x / SLICE;
    if (n <= p.keep) return;
    const int32_t* const kept = p.kept + ((int64_t)b * p.heads + (p.heads > 1 ? hk : 0)) * p.keep;
    const int32_t* const table = p.cache.table ? p.cache.table + (int64_t)b * p.cache.width : nullptr;
    const Tensor& t = which ? p.cache.v : p.cache.k;
    char* const origin = (char*)t.p + (hk * t.sh + (int64_t)piece * (sizeof(UNIT) / size)) * size;
    const bool has = piece < pieces;
    const unsigned keep = p.keep;
    const auto place = [&](int step, int u) { return (unsigned)step * STEP + u * (MOVERS / SLICE) + mine; };        // (may pass 31 bits behind the last row)
    const auto page_of = [&](unsigned r) { return table ? (int)((uint64_t)r * pages_in.factor >> pages_in.shift) : 0; };
    const auto numbers = [&](int step, int (&from)[EACH]) {
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const unsigned i = place(step, u);
            from[u] = kept[i < keep ? i : keep - 1];
        }
    };
    const auto pages = [&](int step, const int (&from)[EACH], int (&src)[EACH], int (&dst)[EACH]) {
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const unsigned i = place(step, u);
            src[u] = table ? table[page_of(from[u])] : b;
            dst[u] = table ? table[page_of(i < keep ? i : keep - 1)] : b;
        }
    };
    const auto at = [&](int page, unsigned r) { return origin + ((int64_t)page * t.sb + (int64_t)(int)(r - page_of(r) * p.cache.page_size) * t.sn) * size; };
    const auto moves = [&](int step, int u, int from, int src, int dst) {
        const unsigned i = place(step, u);
        return has && i < keep && (unsigned)from > i && (unsigned)src < (unsigned)p.cache.pages && (unsigned)dst < (unsigned)p.cache.pages;
    };
    const auto reads = [&](int step, const int (&from)[EACH], const int (&src)[EACH], const int (&dst)[EACH], UNIT (&x)[EACH], UNIT* (&to)[EACH]) {
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const bool go = moves(step, u, from[u], src[u], dst[u]);
            x[u] = *(go ? (const UNIT*)at(src[u], from[u]) : (const UNIT*)&nothing);
            to[u] = go ? (UNIT*)at(dst[u], place(step, u)) : nullptr;
        }
    };
    const int steps = (int)(((int64_t)p.keep + STEP - 1) / STEP);
    int from0[EACH], from1[EACH], from2[EACH], src1[EACH], dst1[EACH];
    UNIT x[EACH];
    UNIT* to[EACH];
    numbers(0, from0);
    numbers(1, from1);
    numbers(2, from2);
    {
        int src0[EACH], dst0[EACH];
        pages(0, from0, src0, dst0);
        pages(1, from1, src1, dst1);
        reads(0, from0, src0, dst0, x, to);
    }
    for (int step = 0; step < steps; ++step) {
        int from3[EACH], src2[EACH], dst2[EACH];
        UNIT next[EACH];
        UNIT* next_to[EACH];
        numbers(step + 3, from3);
        pages(step + 2, from2, src2, dst2);
        reads(step + 1, from1, src1, dst1, next, next_to);
#pragma unroll
        for (int u = 0; u < EACH; ++u) asm volatile("" ::"v"(word(x[u])) : "memory");       // (has come)
        __syncthreads();
#pragma unroll
        for (int u = 0; u < EACH; ++u)
            if (to[u]) *to[u] = x[u];
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            x[u] = next[u];
            to[u] = next_to[u];
            from1[u] = from2[u];
            from2[u] = from3[u];
            src1[u] = src2[u];
            dst1[u] = dst2[u];
        }
    }
}

}  // namespace

int launch_evict(const Evict& p, int dtype, hipStream_t st) {
    const int size = dtype == SA2_F32 ? 4 : 2;
    const bool wide = (p.D * size) % 16 == 0 && aligned16(p.cache.k, size, true) && aligned16(p.cache.v, size, true);
    const int pieces = wide ? p.D * size / 16 : p.D;
    const auto slices_of = [&](int slice) { return (int64_t)p.B * p.HK * 2 * ((pieces + slice - 1) / slice); };
    const bool narrow = slices_of(4) < CUS;                 // half as wide where that leaves CUs without any
    const int64_t grid = slices_of(narrow ? 2 : 4);
    // workgroups that number a head's rows (each finds the smallest weight for itself): four of 65536 rows
    // 50 us, one 64; of 2000 rows one takes 10
    const int64_t room = (int64_t)p.cache.page_size * (p.cache.table ? p.cache.width : 1), streams = (int64_t)p.B * p.heads;
    const int parts = room < 32768 || streams * 2 > CUS ? 1 : streams * 4 > CUS ? 2 : 4;
    if (streams * parts > 0x7fffffff || grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    choose_kernel<<<dim3((unsigned)(p.B * p.heads * parts)), dim3(THREADS), 0, st>>>(p, parts);
    if (hipGetLastError() != hipSuccess) return SA2_ERR_LAUNCH_FAILED;
    const dim3 blocks((unsigned)grid), block(MOVERS);
    const Quotient pages_in = quotient(p.cache.page_size);
    const auto move = [&](auto slice) {
        constexpr int SLICE = decltype(slice)::value;
        const int slices = (pieces + SLICE - 1) / SLICE;
        if (wide) move_kernel<Quad, SLICE><<<blocks, block, 0, st>>>(p, pages_in, size, pieces, slices);
        else if (size == 4) move_kernel<uint32_t, SLICE><<<blocks, block, 0, st>>>(p, pages_in, size, pieces, slices);
        else move_kernel<uint16_t, SLICE><<<blocks, block, 0, st>>>(p, pages_in, size, pieces, slices);
    };
    if (narrow) move(std::integral_constant<int, 2>{});
    else move(std::integral_constant<int, 4>{});
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

}  // namespace sa2
