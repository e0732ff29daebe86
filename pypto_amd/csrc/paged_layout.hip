// A serving step's bookkeeping, gfx950: pages of the cache taken and given back as sequences grow and shrink, and of each new token
// its position, its cache row and, in a tree of drafted tokens, the nodes it sees.
//
// All of it is whole numbers from lengths: sums over the sequences before one, then a look-up per page or token.  Bound by the chain
// of latencies (lengths, sums, table), not by bytes; the sums are made again by every workgroup rather than by a launch of their own.
#include <type_traits>

#include "common.h"
#include "serving_ops.h"

namespace pto {
namespace {

constexpr uint32_t MOST = 0x7fffffffu;

__device__ __forceinline__ uint32_t add_up_to_most(const uint32_t a, const uint32_t b)
{
    const uint32_t s = a + b;                              // (of two numbers up to MOST: no carry)
    return s < MOST ? s : MOST;
}

// Sums of x over this thread and all threads before it, NT of them, none above MOST, and over all threads.  `of_waves` is NT / 64 + 1 words that nobody reads any
// more once every thread has come here.
template <int NT>
__device__ __forceinline__ uint32_t block_sums(uint32_t x, uint32_t *of_waves, uint32_t &total)
{
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_up(x, d);
        if (l >= d) x = add_up_to_most(x, y);
    }
    if (l == 63) of_waves[w] = x;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        const uint32_t y = of_waves[i];
        if (i < w) before = add_up_to_most(before, y);
        all = add_up_to_most(all, y);
    }
    __syncthreads();
    total = all;
    return add_up_to_most(before, x);
}

// The last of n entries, ascending from 0 on, that is at most e.
template <int N>
__device__ __forceinline__ int last_up_to(const uint32_t *at, const int n, const uint32_t e)
{
    int lo = 0;
#pragma unroll
    for (int step = N / 2; step > 0; step /= 2)
        if (lo + step < n && at[lo + step] <= e) lo += step;
    return lo;
}

// One workgroup: what is given back decides what can be taken, and the count of free pages is read and written in one place.  Per 1024 sequences the
// pages are counted out and dealt to the threads, neighbouring ones to neighbouring threads, whichever sequence they are of: which one that is is
// looked up where there are no more pages than threads, else marked where a sequence's pages begin and carried on by a running maximum, for 8192
// pages at a time, whose loads are then on their way together.  A chain of latencies (lengths, sums, table, sums, stack): 32 sequences of which some pass a
// page's end 5.6 us; 1000 of which 50 end and 50 begin, 11 000 pages in all, 19 (one page to a thread at a time, each looked up, 27; counts of the waves
// added one by one instead of by a scan over lanes, 27).
constexpr int PG_THREADS = 1024, PG_EACH = 8, PG_WINDOW = PG_THREADS * PG_EACH;

// sums of x and of y over this lane and all lanes before it
__device__ __forceinline__ void wave_sums(int &x, int &y)
{
    auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
        y += __builtin_amdgcn_update_dpp(0, y, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    };
    const std::integral_constant<int, 0xf> all;
    add(std::integral_constant<int, 0x111>{}, all);        // row_shr:1, 2, 4, 8: within rows of sixteen lanes
    add(std::integral_constant<int, 0x112>{}, all);
    add(std::integral_constant<int, 0x114>{}, all);
    add(std::integral_constant<int, 0x118>{}, all);
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});     // row_bcast:15: rows 0 and 2 into 1 and 3
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});     // row_bcast:31: the lower half into the upper
}

__global__ __launch_bounds__(PG_THREADS) void cache_pages_kernel(const CachePagesParams p)
{
    constexpr int WAVES = PG_THREADS / 64;
    __shared__ int of_waves[2][WAVES], counts[PG_EACH * WAVES];
    __shared__ uint32_t begin[2][PG_THREADS];
    __shared__ int from[2][PG_THREADS];
    __shared__ uint16_t of[PG_WINDOW];
    const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto pages = [&](const int n) {
        const long long k = n > 0 ? ((long long)n + p.bs - 1) / p.bs : 0;
        return (int)(k < p.maxblk ? k : p.maxblk);
    };
    const int given = *p.count;
    int top = given < 0 ? 0 : (given < p.room ? given : (int)p.room);
    uint32_t taken = 0, totals[2] = {0, 0};
    for (int way = 0; way < 2; ++way) {                    // pages given back, then pages taken
        for (int base = 0; base < p.B; base += PG_THREADS) {
            const int here = p.B - base < PG_THREADS ? p.B - base : PG_THREADS;
            if (way == 0 || p.B > PG_THREADS) {            // (all pages of a table are fewer than 2^31)
                int had = 0, has = 0;
                if (tid < here) had = pages(p.before[base + tid]), has = pages(p.after[base + tid]);
                const int back = had > has ? had - has : 0, more = has > had ? has - had : 0;
                int x = back, y = more;
                wave_sums(x, y);
                if (l == 63) of_waves[0][w] = x, of_waves[1][w] = y;
                __syncthreads();
                totals[0] = totals[1] = 0;
#pragma unroll
                for (int i = 0; i < WAVES; ++i) {
                    if (i == w) x += totals[0], y += totals[1];
                    totals[0] += of_waves[0][i], totals[1] += of_waves[1][i];
                }
                begin[0][tid] = x - back, begin[1][tid] = y - more;
                from[0][tid] = has, from[1][tid] = had;
                __syncthreads();
            }
            const uint32_t total = totals[way];            // (the same for all threads)
            for (uint32_t e0 = 0; e0 < total; e0 += PG_WINDOW) {
                const bool few = total <= PG_THREADS;
                if (!few) {                                // of[i]: the sequence that page e0 + i is of
#pragma unroll
                    for (int j = 0; j < PG_EACH; ++j) of[j * PG_THREADS + tid] = 0;
                    __syncthreads();
                    const int mine = tid < here ? (int)((tid + 1 < here ? begin[way][tid + 1] : total) - begin[way][tid]) : 0;
                    const long long at = (long long)begin[way][tid] - e0;
                    if (mine > 0 && at < PG_WINDOW && at + mine > 0) of[at > 0 ? at : 0] = (uint16_t)tid;
                    __syncthreads();
                    // (a thread's eight are neighbours here)
                    int most = 0, run[PG_EACH];
#pragma unroll
                    for (int j = 0; j < PG_EACH; ++j) {
                        const int x = of[PG_EACH * tid + j];
                        most = most > x ? most : x;
                        run[j] = most;
                    }
                    int x = most;
#pragma unroll
                    for (int d = 1; d < 64; d *= 2) {
                        const int y = __shfl_up(x, d);
                        if (l >= d) x = x > y ? x : y;
                    }
                    if (l == 63) of_waves[0][w] = x;
                    int before = __shfl_up(x, 1);
                    if (l == 0) before = 0;
                    __syncthreads();
                    for (int i = 0; i < w; ++i) before = before > of_waves[0][i] ? before : of_waves[0][i];
#pragma unroll
                    for (int j = 0; j < PG_EACH; ++j) of[PG_EACH * tid + j] = (uint16_t)(run[j] > before ? run[j] : before);
                    __syncthreads();
                }
                int32_t *entry[PG_EACH];
                int page[PG_EACH];
#pragma unroll
                for (int j = 0; j < PG_EACH; ++j) {
                    const uint32_t e = e0 + j * PG_THREADS + tid;
                    entry[j] = nullptr;
                    if (e < total) {
                        const int s = few ? last_up_to<PG_THREADS>(begin[way], here, e) : of[j * PG_THREADS + tid];
                        entry[j] = p.bt + (long long)(base + s) * p.maxblk + from[way][s] + (int)(e - begin[way][s]);
                    }
                    if (few) break;                        // (uniform)
                }
                const int n = few ? 1 : PG_EACH;
                if (way == 0) {
#pragma unroll
                    for (int j = 0; j < PG_EACH; ++j)
                        if (j < n) page[j] = entry[j] ? *entry[j] : -1;
                    // pages that there are, in order: by the eighth of the window, then by the wave
                    uint64_t there[PG_EACH];
#pragma unroll
                    for (int j = 0; j < PG_EACH; ++j)
                        if (j < n) {
                            there[j] = __ballot(page[j] >= 0);
                            if (l == 0) counts[j * WAVES + w] = __popcll(there[j]);
                        }
                    __syncthreads();
                    static_assert(PG_EACH * WAVES == 128, "two counts to a lane");
                    const int c0 = 2 * l < n * WAVES ? counts[2 * l] : 0, c1 = 2 * l < n * WAVES ? counts[2 * l + 1] : 0;
                    int with = c0 + c1, other = 0;
                    wave_sums(with, other);
#pragma unroll
                    for (int j = 0; j < PG_EACH; ++j) {
                        if (j >= n) break;
                        const int pair = j * (WAVES / 2) + w / 2;
                        const long long to = (long long)top + __builtin_amdgcn_readlane(with, pair) - __builtin_amdgcn_readlane(c1, pair)
                                     - (w & 1 ? 0 : __builtin_amdgcn_readlane(c0, pair));
                        const long long at = to + __popcll(there[j] & ((1ull << l) - 1));
                        if (page[j] >= 0 && at < p.room) p.stack[at] = page[j];
                    }
                    const long long all = (long long)top + __builtin_amdgcn_readlane(with, 63);
                    top = all < p.room ? (int)all : (int)p.room;
                    __syncthreads();
                } else {
#pragma unroll
                    for (int j = 0; j < PG_EACH; ++j)
                        if (j < n) {
                            const long long at = (long long)top - 1 - taken - (e0 + j * PG_THREADS + tid);
                            page[j] = entry[j] && at >= 0 ? p.stack[at] : -1;
                        }
#pragma unroll
                    for (int j = 0; j < PG_EACH; ++j)
                        if (j < n && entry[j]) *entry[j] = page[j];
                    __syncthreads();
                }
            }
            if (way == 1) taken += total;
            if (p.B > PG_THREADS) __syncthreads();
        }
        __syncthreads();                                   // (the pages on the stack are there for all)
    }
    if (tid == 0) *p.left = (long long)top - taken > 0 ? top - (int)taken : 0;
}

// A workgroup takes the tokens t0 .. t1 - 1, a thread one at a time; the beginnings of up to 1024 sequences are in LDS.  512 single tokens 4.1 us, nine prompts of
// 200 000 tokens in all 4.1, 48 trees of 17 to 63 nodes 5.5 (a node's ancestors are walked up by its own thread, a tree's parents in LDS): a launch, lengths, sums and
// a table entry, one behind the other.  A chain of 1000 nodes 94 with one mask word and with 16 (a walk for each word: 1450), since the last node's steps are behind one another.
constexpr int SL_THREADS = 256, SL_SEQS = 1024, SL_NODES = 64 * SLOTS_MAX_WORDS, SL_PER = SL_SEQS / SL_THREADS;

__global__ __launch_bounds__(SL_THREADS) void cache_slots_kernel(const CacheSlotsParams p, const int each)
{
    __shared__ uint32_t of_waves[SL_THREADS / 64], begin[SL_SEQS];
    __shared__ int first_row[SL_SEQS];
    __shared__ int parent[SL_NODES + SL_THREADS];
    const int tid = threadIdx.x;
    const long long t0 = (long long)blockIdx.x * each, t1 = t0 + each < p.T ? t0 + each : p.T;
    uint32_t before_q = 0, before_k = 0;                   // tokens of the sequences before these 1024
    long long done = t0;                                   // tokens of this workgroup behind these were dealt with
    for (int base = 0; base < p.B; base += SL_SEQS) {
        // (a thread's sequences lie together, so that its own sums are the workgroup's with one more addition each)
        uint32_t nq[SL_PER], nk[SL_PER], sum_q = 0, sum_k = 0;
#pragma unroll
        for (int j = 0; j < SL_PER; ++j) {
            const int b = base + SL_PER * tid + j;
            int q = 0, k = 0;
            if (b < p.B) q = p.new_lens[b], k = p.all_lens[b];
            nq[j] = q > 0 ? q : 0, nk[j] = k > 0 ? k : 0;
            sum_q = add_up_to_most(sum_q, nq[j]), sum_k = add_up_to_most(sum_k, nk[j]);
        }
        uint32_t total_q, total_k = 0;
        uint32_t upto = block_sums<SL_THREADS>(sum_q, of_waves, total_q);
        const int here = p.B - base < SL_SEQS ? p.B - base : SL_SEQS;
        // the sums before a thread's first sequence: those of the thread before it
        uint32_t at = __shfl_up(upto, 1);
        if ((tid & 63) == 63) of_waves[tid >> 6] = upto;
        __syncthreads();
        if ((tid & 63) == 0) at = tid > 0 ? of_waves[(tid >> 6) - 1] : 0;
        uint32_t q_at = at;
#pragma unroll
        for (int j = 0; j < SL_PER; ++j) {
            begin[SL_PER * tid + j] = q_at;
            first_row[SL_PER * tid + j] = (int)nk[j] - (int)nq[j];
            if (blockIdx.x == 0 && base + SL_PER * tid + j < p.B) p.cu_q[base + SL_PER * tid + j] = (int32_t)add_up_to_most(before_q, q_at);
            q_at = add_up_to_most(q_at, nq[j]);
        }
        __syncthreads();
        if (blockIdx.x == 0 && p.cu_k) {
            upto = block_sums<SL_THREADS>(sum_k, of_waves, total_k);
            uint32_t k_at = __shfl_up(upto, 1);
            if ((tid & 63) == 63) of_waves[tid >> 6] = upto;
            __syncthreads();
            if ((tid & 63) == 0) k_at = tid > 0 ? of_waves[(tid >> 6) - 1] : 0;
#pragma unroll
            for (int j = 0; j < SL_PER; ++j) {
                if (base + SL_PER * tid + j < p.B) p.cu_k[base + SL_PER * tid + j] = (int32_t)add_up_to_most(before_k, k_at);
                k_at = add_up_to_most(k_at, nk[j]);
            }
            __syncthreads();
        }
        const long long end = (long long)before_q + total_q < t1 ? (long long)before_q + total_q : t1;
        for (long long i0 = done; i0 < end; i0 += SL_THREADS) {
            const long long t = i0 + tid;
            int s = 0, r = 0, first = 0;                   // sequence, token within it, tokens before the sequence
            if (t < end) {
                s = last_up_to<SL_SEQS>(begin, here, (uint32_t)(t - before_q));
                first = (int)(before_q + begin[s]);
                r = (int)t - first;
            }
            int staged = 0;                                // parents of tokens from this one on are in LDS
            if (p.parents) {
                const long long lead = (long long)before_q + begin[last_up_to<SL_SEQS>(begin, here, (uint32_t)(i0 - before_q))];
                staged = (int)(i0 - lead < SL_NODES ? lead : i0 - SL_NODES);
                const int n = (int)((i0 + SL_THREADS < end ? i0 + SL_THREADS : end) - staged);
                for (int i = tid; i < n; i += SL_THREADS) parent[i] = p.parents[staged + i];
                __syncthreads();
            }
            if (t < end) {
                const long long row = (long long)first_row[s] + r;
                long long slot = -1;
                if (row >= 0 && row < (long long)p.maxblk * p.bs) {
                    const int block = (int)((uint64_t)row / (uint32_t)p.bs);
                    const int page = p.bt[(long long)(base + s) * p.maxblk + block];
                    if (page >= 0) slot = (long long)page * p.bs + (row - (long long)block * p.bs);
                }
                p.slots[t] = slot;
                int depth = r;
                if (p.parents) {
                    // One walk for all words: a parent comes before its child, so the walk ends, and a word that it has left is whole.
                    int word = p.words;                    // words from this one on are written
                    auto zeros_down_to = [&](const int w) {
                        while (word > w) p.mask[t * p.words + --word] = 0;
                    };
                    depth = -1;
                    for (int node = r; node >= 0;) {
                        const int low = node & ~63, at = low >> 6;
                        unsigned long long bits = 0;
                        do {                               // the nodes of a word
                            bits |= 1ull << (node & 63);
                            ++depth;
                            const int of = first + node, up = of >= staged ? parent[of - staged] : p.parents[of];
                            node = up < node ? up : -1;
                        } while (node >= low);
                        zeros_down_to(at + 1);
                        if (at < p.words) p.mask[t * p.words + at] = bits, word = at;
                    }
                    zeros_down_to(0);
                }
                p.positions[t] = (long long)first_row[s] + depth;
            }
            if (p.parents) __syncthreads();
        }
        done = done > end ? done : end;
        before_q = add_up_to_most(before_q, total_q), before_k = add_up_to_most(before_k, total_k);
        __syncthreads();
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.cu_q[p.B] = (int32_t)before_q;
        if (p.cu_k) p.cu_k[p.B] = (int32_t)before_k;
    }
    for (long long t = done + tid; t < t1; t += SL_THREADS) {        // tokens of no sequence
        p.positions[t] = 0;
        p.slots[t] = -1;
        if (p.parents)
            for (int w = 0; w < p.words; ++w) p.mask[t * p.words + w] = 0;
    }
}

}  // namespace

hipError_t cache_pages_launch(const CachePagesParams &p, hipStream_t stream)
{
    hipLaunchKernelGGL(cache_pages_kernel, dim3(1), dim3(PG_THREADS), 0, stream, p);
    return hipGetLastError();
}

hipError_t cache_slots_launch(const CacheSlotsParams &p, hipStream_t stream)
{
    const long long most = 4ll * p.cus * SL_THREADS;
    const long long each = (p.T <= most ? SL_THREADS : (p.T + most - 1) / most * SL_THREADS);
    const long long grid = p.T > 0 ? (p.T + each - 1) / each : 1;
    hipLaunchKernelGGL(cache_slots_kernel, dim3((unsigned)grid), dim3(SL_THREADS), 0, stream, p, (int)each);
    return hipGetLastError();
}

}  // namespace pto
