// What a program asks of a row of logits besides the next token: the log probability of a token that
// was given, the entropy of the row, and the `top` most probable tokens with theirs.
//     m = max x,   l = sum e^(x - m)
//     logprob[t] = (x_t - m) - ln l,   entropy = ln l - (sum e^(x - m) (x - m)) / l
// One pass over the row computes all of it, so the kernel is bound by HBM (16-bit logits: also by
// the exponential unit, at two thirds of its rate when the memory runs at its own).
//
// A row is divided among a cluster of blocks (1, 2, 4 or 8, so that few rows fill the GPU too) and
// read in groups of 32 pieces of 16 bytes, one piece a lane.  Every thread keeps (m, l, s) of its
// own pieces: a new maximum rescales l and s, and moves s's origin: with c = e^(m - m'),
// l' = c l, s' = c (s + (m - m') l).  Threads, warps and blocks are joined by the same rule.
//
// The alternatives cost the pass one reduction a group: its largest logit, kept in shared memory.
// The `top` first logits, larger ones first and the lower index first among equals, lie in the `top`
// first groups by (largest logit, index), since each group ahead of an element's own holds an
// element ahead of it.  So the first block, whose memory the others of the cluster store their groups'
// to, finds a threshold that `top` groups reach and not many more (by bisection over the floats' order
// where the first guess has too many), reads those groups once more and ranks what reaches it.
//
// Measured on a B200, rows of 128256: 2048 of bf16 with 5 alternatives 102 us, 5.1 TB/s (92 without:
// 5.7 TB/s), of f32 162 us, 6.5 TB/s; 64 of f32 12.5 us; one of bf16 with 20 alternatives 8.9 us, half of
// it the way from the last logit over the cluster's barrier to the ranked list.  (2048 of bf16 in a run of a second, at
// the clock that the power limit leaves, 1.84 GHz: 107 us.)
//
// Slow is a row of no more groups than alternatives: no group can be left out, and a block bisects over all of its
// elements.  1000 bf16 rows of 1000 logits 27 us with 20 alternatives, 70 with 99 % of them forbidden, 7 without
// alternatives; of 2890, 63, 83 and 8; of 8200 logits 18, 18 and 9.
#include <cooperative_groups.h>

#include "mma.cuh"

namespace b200q {
namespace cg = cooperative_groups;
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kHeld = 4;          // pieces a thread has in flight
constexpr int kMaxTop = 32;
constexpr int kPicked = 64;       // groups that are read again
constexpr int kRanked = kThreads; // elements that are ranked against one another, one a thread
constexpr float kLowest = -3.402823466e38f;
constexpr float kNothing = -200.0f;  // e^-200 is 0 in f32

struct LogprobArgs {
    const void* logits;
    int64_t stride;               // of a row, in elements
    const int64_t* tokens;
    float* logprob;
    float* entropy;
    float* top_logprob;
    int64_t* top_token;
    int vocab, top, groups;
    int* status;
};

__device__ __forceinline__ float exp2_approx(float x) {  // relative error 2^-22; 2^-289 is 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // leaves NaN out
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The order of floats as unsigned numbers, -0 with 0, NaN with -inf (so that no element is ahead of
// the largest of its group, which leaves NaN out).
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t bits = __float_as_uint(x + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ float of_order(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

template <typename T>
struct Logit;  // E elements a 16-byte piece
template <>
struct Logit<float> {
    static constexpr int E = 4;
    __device__ static __forceinline__ void widen(const uint4& p, float (&x)[4]) {
        x[0] = __uint_as_float(p.x), x[1] = __uint_as_float(p.y), x[2] = __uint_as_float(p.z), x[3] = __uint_as_float(p.w);
    }
    __device__ static __forceinline__ float one(const void* base, int64_t i) {
        return ld_mutable(static_cast<const float*>(base) + i);
    }
};
template <typename T>
struct Logit16 {
    static constexpr int E = 8;
    __device__ static __forceinline__ void widen(const uint4& p, float (&x)[8]) {
        const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = Half16<T>::to_float(w[i] & 0xFFFFu);
            x[2 * i + 1] = Half16<T>::to_float(w[i] >> 16);
        }
    }
    __device__ static __forceinline__ float one(const void* base, int64_t i) {
        return Half16<T>::to_float(ld_mutable(static_cast<const uint16_t*>(base) + i));
    }
};
template <>
struct Logit<__nv_bfloat16> : Logit16<__nv_bfloat16> {};
template <>
struct Logit<__half> : Logit16<__half> {};

struct Sums {
    float m, l, s;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    const float da = a.m - r.m, db = b.m - r.m, ca = expf(da), cb = expf(db);
    r.l = ca * a.l + cb * b.l;
    // (a side that has nothing may be infinitely far below: 0 * inf)
    r.s = (ca > 0.0f ? ca * (a.s + da * a.l) : 0.0f) + (cb > 0.0f ? cb * (b.s + db * b.l) : 0.0f);
    return r;
}

// A row seen as pieces that start on 16-byte boundaries: element i is number i + shift of them.
template <typename T>
struct Row {
    static constexpr int E = Logit<T>::E;
    const T* base;
    int shift, vocab, pieces;
    __device__ __forceinline__ Row(const LogprobArgs& a, int row) {
        base = static_cast<const T*>(a.logits) + row * a.stride;
        shift = int(reinterpret_cast<uintptr_t>(base) % 16 / sizeof(T));
        vocab = a.vocab;
        pieces = (shift + vocab + E - 1) / E;
    }
    __device__ __forceinline__ const uint4* pieces_at() const { return reinterpret_cast<const uint4*>(base - shift); }
    // The elements of piece p; those outside the row read -inf.
    __device__ __forceinline__ bool whole(int p) const { return p * E >= shift && p * E - shift + E <= vocab; }
    __device__ __forceinline__ uint4 load(int p) const {
        return ld_mutable(reinterpret_cast<const uint4*>(base - shift + int64_t(p) * E));
    }
    __device__ __forceinline__ void edge(int p, float (&x)[E]) const {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = p * E + e - shift;
            x[e] = i >= 0 && i < vocab ? Logit<T>::one(base, i) : -INFINITY;
        }
    }
};

// Adds E logits to a thread's sums; returns the largest.
template <int E>
__device__ __forceinline__ float largest(const float (&x)[E]) {
    if constexpr (E == 4) return fmaxf(max3(x[0], x[1], x[2]), x[3]);
    else return max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), fmaxf(x[6], x[7]));
}
template <int E>
__device__ __forceinline__ void add(const float (&x)[E], float m, float2& l, float2& s) {
    const float2 minus = make_float2(-m, -m), log2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        float2 d = __fadd2_rn(make_float2(x[e], x[e + 1]), minus);
        d.x = max_nan(d.x, kNothing), d.y = max_nan(d.y, kNothing);
        const float2 t = __fmul2_rn(d, log2e), w = make_float2(exp2_approx(t.x), exp2_approx(t.y));
        l = __fadd2_rn(l, w);
        s = __ffma2_rn(w, d, s);
    }
}

// With alternatives, five blocks a multiprocessor: one's ranking goes by while the others read.  2048 rows with five:
// 102 us so (of 48 registers, with 44 bytes spilled), 106 with four, 120 with three, 142 with six (of 40 registers each);
// f32 162 (of 46, nothing spilled), 173, 184, 175.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, TOP ? 5 : 0)
token_logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    constexpr int E = Logit<T>::E;
    extern __shared__ float group_max[];  // of the row's groups, in the first block
    __shared__ Sums warp_sums[kWarps], block_sums[8];  // the cluster's, in its first block
    __shared__ double row_max, row_log;  // m and ln l: their sum would lose the second where logits are huge
    __shared__ int picked[kPicked];
    __shared__ uint64_t ranked[kRanked];
    __shared__ uint32_t threshold, class_max[32];
    __shared__ int picked_count, ranked_count, reached;
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = int(cluster.num_blocks()), rank = int(cluster.block_rank()), row = int(blockIdx.x) / blocks;
    // (the first block has started when the others store to its memory)
    if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    pdl_launch_dependents();
    pdl_wait();
    if (blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    float* const all_max = blocks > 1 ? cluster.map_shared_rank(group_max, 0) : group_max;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const Row<T> logits(a, row);
    // groups of this row (a row that starts past a boundary may have one more than others), divided evenly
    const int groups = (logits.pieces + 31) / 32;
    const int first = int(int64_t(groups) * rank / blocks), last = int(int64_t(groups) * (rank + 1) / blocks);

    float m = kLowest;
    float2 l = make_float2(0.0f, 0.0f), s = l;
    // kHeld pieces a lane; the first group's number, and of how many groups the largest are kept
    auto take = [&](float (&x)[kHeld][E], int g0, int kept) {
        float peak[kHeld], most = m;
#pragma unroll
        for (int u = 0; u < kHeld; ++u) peak[u] = largest(x[u]), most = fmaxf(most, peak[u]);
        if (most > m) {  // (else all of them are at most m, or NaN, which the sums take in)
            const float d = m - most, c = exp2_approx(d * 1.4426950408889634f), by = fmaxf(d, kNothing);
            s = make_float2(c * (s.x + by * l.x), c * (s.y + by * l.y));
            l = make_float2(c * l.x, c * l.y);
            m = most;
        }
#pragma unroll
        for (int u = 0; u < kHeld; ++u) add(x[u], m, l, s);
        if (TOP) {
#pragma unroll
            for (int u = 0; u < kHeld; ++u) {
                float peak_all;
                asm volatile("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(peak_all) : "f"(peak[u]));
                if (lane == u) peak[0] = peak_all;
            }
            if (lane < kept) all_max[g0 + lane] = peak[0];
        }
    };
    // Groups without an edge of the row, kHeld at a time; what is left of them, and the edges, after that.
    const int inner_first = max(first, logits.shift > 0 ? 1 : 0), inner_last = min(last, (logits.shift + logits.vocab) / (32 * E));
    const int rounds = max(0, inner_last - inner_first) / kHeld;
    {
        const uint4* from = logits.pieces_at() + (inner_first + warp * kHeld) * 32 + lane;
        for (int r = warp; r < rounds; r += kWarps, from += kWarps * kHeld * 32) {
            uint4 held[kHeld];
#pragma unroll
            for (int u = 0; u < kHeld; ++u) held[u] = ld_mutable(from + u * 32);
            float x[kHeld][E];
#pragma unroll
            for (int u = 0; u < kHeld; ++u) Logit<T>::widen(held[u], x[u]);
            take(x, inner_first + r * kHeld, kHeld);
        }
    }
    // The groups left, one a warp: the first one's edge, the last one's, and those of an unfinished round.
    const int tail = inner_first + rounds * kHeld, left = (inner_first - first) + (last - tail);
    for (int i = warp; i < left; i += kWarps) {
        const int g = i < inner_first - first ? first + i : tail + i - (inner_first - first), p = g * 32 + lane;
        float x[kHeld][E];
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) x[u][e] = -INFINITY;
        if (p < logits.pieces) {
            if (logits.whole(p)) Logit<T>::widen(logits.load(p), x[0]);
            else logits.edge(p, x[0]);
        }
        take(x, g, 1);
    }
    Sums mine = {m, l.x + l.y, s.x + s.y};
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
        const Sums theirs = {__shfl_xor_sync(0xFFFFFFFFu, mine.m, d), __shfl_xor_sync(0xFFFFFFFFu, mine.l, d),
                             __shfl_xor_sync(0xFFFFFFFFu, mine.s, d)};
        mine = join(mine, theirs);
    }
    if (lane == 0) warp_sums[warp] = mine;
    if (threadIdx.x == 0) ranked_count = picked_count = 0;
    if (threadIdx.x < 32) class_max[threadIdx.x] = 0;
    __syncthreads();
    auto join_lanes = [&](int count) {  // the sums of the first `count` lanes (a power of two), in lane 0
        for (int d = count / 2; d >= 1; d >>= 1) {
            const Sums theirs = {__shfl_xor_sync(0xFFFFFFFFu, mine.m, d), __shfl_xor_sync(0xFFFFFFFFu, mine.l, d),
                                 __shfl_xor_sync(0xFFFFFFFFu, mine.s, d)};
            mine = join(mine, theirs);
        }
    };
    if (warp == kWarps - 1) {
        mine = warp_sums[lane % kWarps];
        join_lanes(kWarps);
        if (blocks > 1 && lane == 0) cluster.map_shared_rank(block_sums, 0)[rank] = mine;
    }
    if (blocks > 1) cluster.sync();  // every block's sums and groups are in the first one's memory
    else __syncthreads();
    if (rank != 0) return;
    if (blocks > 1 && warp == kWarps - 1) {
        mine = block_sums[lane % blocks];
        join_lanes(blocks);
    }
    if (threadIdx.x == (kWarps - 1) * 32) {
        const double most = double(mine.m), norm = log(double(mine.l));
        row_max = most, row_log = norm;
        const int64_t token = ld_mutable(a.tokens + row);
        float given = 0.0f;  // none given
        if (token >= a.vocab) {
            record_bad_position(a.status, row);
            given = __int_as_float(0x7FC00000);
        } else if (token >= 0) {
            given = float(double(Logit<T>::one(logits.base, token)) - most - norm);
        }
        a.logprob[row] = given;
        a.entropy[row] = float(norm - double(mine.s) / double(mine.l));
    }
    if (!TOP) return;

    // ---- the groups that are read again: those above `low` ----
    const int top = a.top;
    // The largest of every 32nd group, 32 of them: the top-th of those is reached by `top` groups at least, and seldom by
    // many more.
    uint32_t best = 0, low;
    for (int g = threadIdx.x; g < groups; g += kThreads) best = max(best, order_of(group_max[g]));
    atomicMax(&class_max[lane], best);
    __syncthreads();
    best = class_max[lane];
    int others = 0;
#pragma unroll
    for (int other = 0; other < 32; ++other) {
        const uint32_t theirs = __shfl_sync(0xFFFFFFFFu, best, other);
        others += theirs > best || (theirs == best && other < lane);
    }
    const uint32_t reached_by_top = __shfl_sync(0xFFFFFFFFu, best, __ffs(__ballot_sync(0xFFFFFFFFu, others == top - 1)) - 1);
    low = reached_by_top - 1;
    if (groups >= 32)
        for (int g = threadIdx.x; g < groups; g += kThreads)
            if (order_of(group_max[g]) > low) {
                const int i = atomicAdd(&picked_count, 1);
                if (i < kPicked) picked[i] = g;
            }
    __syncthreads();
    const bool in_order = groups < 32 || picked_count > kPicked;  // the picked groups are, by index
    if (in_order) {
        __syncthreads();
        if (warp == 0) {
            // low: at least min(top, groups) groups reach it; high: fewer do
            uint32_t least = 0xFFFFFFFFu, most = 0;
            for (int g = lane; g < groups; g += 32) {
                const uint32_t k = order_of(group_max[g]);
                least = min(least, k), most = max(most, k);
            }
            least = __reduce_min_sync(0xFFFFFFFFu, least), most = __reduce_max_sync(0xFFFFFFFFu, most);
            low = least;
            uint32_t high = most + 1;
            int reach = groups;
            if (groups <= top) low = 0;
            while (groups > top && reach > kPicked && high - low > 1) {
                const uint32_t mid = low + (high - low) / 2;
                int c = 0;
                for (int g = lane; g < groups; g += 32) c += order_of(group_max[g]) >= mid;
                c = __reduce_add_sync(0xFFFFFFFFu, c);
                if (c >= top) low = mid, reach = c;
                else high = mid;
            }
            // All groups above `low`; of those that just reach it as many as there is room for, the first ones.
            int above = 0;
            for (int g = lane; g < groups; g += 32) above += order_of(group_max[g]) > low;
            above = __reduce_add_sync(0xFFFFFFFFu, above);
            int room = kPicked - above, n = 0;
            for (int g0 = 0; g0 < groups; g0 += 32) {
                const int g = g0 + lane;
                const uint32_t k = g < groups ? order_of(group_max[g]) : 0;
                const bool just = g < groups && k == low;
                const uint32_t ties = __ballot_sync(0xFFFFFFFFu, just);
                const bool take = (g < groups && k > low) || (just && __popc(ties & ((1u << lane) - 1)) < room);
                const uint32_t taken = __ballot_sync(0xFFFFFFFFu, take);
                if (take) picked[n + __popc(taken & ((1u << lane) - 1))] = g;
                n += __popc(taken);
                room -= min(room, __popc(ties));
            }
            if (lane == 0) picked_count = n, threshold = low;
        }
        __syncthreads();
        low = threshold;
    }

    // Calls `f(order, element)` for every element of the picked groups; one warp a group.
    const int picks = picked_count;
    auto each = [&](auto f) {
#pragma unroll 1
        for (int i = warp; i < picks; i += kWarps) {
            const int p = picked[i] * 32 + lane;
            float x[E];
            if (p < logits.pieces) {
                if (logits.whole(p)) Logit<T>::widen(logits.load(p), x);
                else logits.edge(p, x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int at = p * E + e - logits.shift;
                    if (at >= 0 && at < a.vocab) f(order_of(x[e]), at);
                }
            }
        }
    };
    auto collect = [&](uint32_t low) {  // what exceeds `low`, as far as there is room
        each([&](uint32_t k, int i) {
            if (k > low) {
                const int at = atomicAdd(&ranked_count, 1);
                if (at < kRanked) ranked[at] = uint64_t(k) << 32 | uint32_t(~i);
            }
        });
        __syncthreads();
    };
    collect(low);
    if (ranked_count > kRanked) {  // many above a threshold made for groups: bisect over the elements
        if (!in_order) {           // (ties at the end of that go by index)
            int mine_at = 0, mine_group = 0;
            if (int(threadIdx.x) < picks) {
                mine_group = picked[threadIdx.x];
                for (int i = 0; i < picks; ++i) mine_at += picked[i] < mine_group;
            }
            __syncthreads();
            if (int(threadIdx.x) < picks) picked[mine_at] = mine_group;
            __syncthreads();
        }
        uint32_t high = 0xFFFFFFFFu;
        while (high - low > 1) {
            if (threadIdx.x == 0) reached = 0;
            __syncthreads();
            const uint32_t mid = low + (high - low) / 2;
            int c = 0;
            each([&](uint32_t k, int) { c += k >= mid; });
            c = __reduce_add_sync(0xFFFFFFFFu, c);
            if (lane == 0) atomicAdd(&reached, c);
            __syncthreads();
            const int now = reached;
            if (now >= top) low = mid;
            else high = mid;
            if (now >= top && now <= kRanked) break;
            __syncthreads();
        }
        if (threadIdx.x == 0) ranked_count = 0;
        __syncthreads();
        collect(low);
    }
    const int above = ranked_count;
    const double most = row_max, norm = row_log;
    auto emit = [&](int at, float x, int i) {
        a.top_logprob[int64_t(row) * top + at] = float(double(x) - most - norm);
        a.top_token[int64_t(row) * top + at] = i;
    };
    if (int(threadIdx.x) < above) {
        const uint64_t own = ranked[threadIdx.x];
        int ahead = 0;
        for (int j = 0; j < above; ++j) ahead += ranked[j] > own;
        if (ahead < top) {
            emit(ahead, of_order(uint32_t(own >> 32)), int(~uint32_t(own)));
        }
    }
    // Those that just reach the threshold fill what is left, the lower index first.
    if (above < top && warp == 0) {
        int n = above;
#pragma unroll 1
        for (int g = 0; g < picks && n < top; ++g) {
            const int p = picked[g] * 32 + lane;
            uint32_t ties = 0;
            float x[E];
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = 0.0f;
            if (p < logits.pieces) {
                if (logits.whole(p)) Logit<T>::widen(logits.load(p), x);
                else logits.edge(p, x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int i = p * E + e - logits.shift;
                    if (i >= 0 && i < a.vocab && order_of(x[e]) == low) ties |= 1u << e;
                }
            }
            int before = __popc(ties);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int other = __shfl_up_sync(0xFFFFFFFFu, before, d);
                if (lane >= d) before += other;
            }
            const int all = __shfl_sync(0xFFFFFFFFu, before, 31);
            int at = n + before - __popc(ties);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (ties >> e & 1) {
                    if (at < top) emit(at, x[e], p * E + e - logits.shift);
                    ++at;
                }
            n += all;
        }
    }
}

template <typename T, bool TOP>
cudaError_t launch(const LogprobArgs& a, int rows, int blocks, cudaStream_t stream) {
    const size_t smem = TOP ? sizeof(float) * size_t(a.groups) : 0;
    auto kernel = token_logprobs_kernel<T, TOP>;
    cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(blocks) * unsigned(rows));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(blocks);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, kernel, a);
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int32_t b200q_token_logprobs(const void* logits, const int64_t* tokens, float* logprob, float* entropy,
                                        float* top_logprob, int64_t* top_token, int64_t rows, int64_t vocab, int64_t stride,
                                        int64_t top, int32_t dtype, void* stream) {
    B200Q_REQUIRE(rows >= 0 && rows < (int64_t(1) << 27) && vocab > 0 && vocab <= (int64_t(1) << 20) && stride >= 0,
                  "token_logprobs: fewer than 2^27 rows of 1 to 2^20 logits, not %lld of %lld", (long long)rows, (long long)vocab);
    B200Q_REQUIRE(top >= 0 && top <= kMaxTop && top <= vocab, "token_logprobs: 0 to %d alternatives of a row, not %lld",
                  int(kMaxTop < vocab ? kMaxTop : vocab), (long long)top);
    B200Q_REQUIRE(dtype == B200Q_F32 || dtype == B200Q_BF16 || dtype == B200Q_F16, "token_logprobs: f32, bf16 or f16");
    if (rows == 0) return B200Q_OK;
    const int size = dtype == B200Q_F32 ? 4 : 2, elements = 16 / size;
    B200Q_REQUIRE(logits && tokens && logprob && entropy && (top == 0 || (top_logprob && top_token)) &&
                      aligned(logits, size_t(size)) && aligned(tokens, 8) && aligned(logprob, 4) && aligned(entropy, 4) &&
                      aligned(top_logprob, 4) && aligned(top_token, 8),
                  "token_logprobs: null or misaligned tensor");
    LogprobArgs a = {};
    a.logits = logits, a.stride = stride, a.tokens = tokens;
    a.logprob = logprob, a.entropy = entropy, a.top_logprob = top_logprob, a.top_token = top_token;
    a.vocab = int(vocab), a.top = int(top);
    a.groups = int((vocab + elements - 1 + 32 * elements - 1) / (32 * elements));  // of a row wherever it starts
    a.status = decoder_error_word();
    // Blocks a row: twice as many while there are fewer than four a multiprocessor and each has a round of its own.
    // With five alternatives, 64 f32 rows of 128256: 12.7 us with eight blocks each, 30.1 with one; 148: 19.8 with four, 25.0
    // with two, 23.0 with eight; 333: 33.2 with two, 41.7 with one.  The rule knows neither the type nor how many blocks are
    // resident (four to six a multiprocessor), and costs some rows a second round of them: 333 16-bit rows of 32003 without
    // alternatives take 10.4 with its two and 10.0 with one, 222 of them 10.3 with its four and 7.6 with two.
    const int64_t each = int64_t(kWarps) * kHeld;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t err = cudaSuccess;
    const int n = int(rows);
    int blocks = 1;
    while (blocks < 8 && rows * blocks < 4 * sm_count() && a.groups > blocks * each) blocks *= 2;
    if (dtype == B200Q_F32) err = top ? launch<float, true>(a, n, blocks, s) : launch<float, false>(a, n, blocks, s);
    else if (dtype == B200Q_BF16)
        err = top ? launch<__nv_bfloat16, true>(a, n, blocks, s) : launch<__nv_bfloat16, false>(a, n, blocks, s);
    else err = top ? launch<__half, true>(a, n, blocks, s) : launch<__half, false>(a, n, blocks, s);
    return launch_status("token_logprobs", err);
}
