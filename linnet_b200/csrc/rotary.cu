// Rotary positions: the first 2 * pairs numbers of every head, taken as pairs, are turned by
// position * frequency:
//     (a, b) -> factor * (a cos - b sin, b cos + a sin),   angle = position * frequencies[pair]
// Pairs are the two halves (i, i + pairs) or neighbours (2i, 2i + 1); numbers past them are copied.
// The frequencies come as f64, so that any scaling for long contexts is the caller's, and the angle
// is formed in f64 turns and reduced to half a turn before it becomes f32: at position 10^6 an f32
// angle is off by up to 0.03 radians, this one by 2^-24 of itself.
//
// The kernel reads q and k once and writes them once, so it is bound by HBM.  A block takes a few
// tokens and computes cosine and sine of a token's pairs once for all of its heads; a thread takes the
// same pairs (a unit: two 16-byte pieces) of several heads, so that it reads their cosines and sines
// from shared memory once, and has five heads in flight before it needs them.  (With a unit of any
// head a thread, reading the cosines took 60 % of the shared memory's time.)  With few tokens the heads
// of one are divided among blocks too.
//
// Measured on a B200: 8192 tokens of 32 + 8 heads of 128, bf16, 33.2 us, 5.05 TB/s; one token 2.5 us, its latency.
#include "mma.cuh"

namespace b200q {
namespace {

constexpr int kThreads = 128;      // 8192 tokens 33.2 us, of neighbours 33.3; with 256 threads 34.4 and 38.2
constexpr int kHeld = 5;           // heads a thread has in flight, of large calls; of small ones 1
constexpr int kMaxTokens = 16;     // of a block
constexpr int kMaxTurns = 4096;    // (cos, sin) pairs of a block: 32 KB

struct RotaryArgs {
    const uint16_t* src[3];        // q, k, v
    uint16_t* dst[3];
    int64_t src_token[3], src_head[3], dst_token[3], dst_head[3];  // strides, in numbers
    const int64_t* positions;
    const double* frequencies;
    const int64_t* offset_at;      // added to the positions: read on the device, or `offset`
    int64_t offset;
    int64_t slots;                 // > 0: k and v go to slot `position` of caches that long
    int tokens, nq, nkv, heads;    // heads: all that are written, v's among them
    int pairs, units, turning;     // units of a head: `turning` of them hold pairs, the others are copied
    int token_threads, step;       // threads of a token; heads they take at a time
    int head_dim, block_tokens, block_heads;
    float factor;
    int* status;
};

// W numbers a piece, two pieces a unit: W = 8, 16-byte accesses; W = 1 takes any size and alignment.
template <int W>
struct Piece;
template <>
struct Piece<8> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const uint16_t* p) {
        const uint4 v = ld_mutable(reinterpret_cast<const uint4*>(p));
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
    __device__ __forceinline__ void store(uint16_t* p) const {
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <>
struct Piece<1> {
    uint32_t w[1];
    __device__ __forceinline__ void load(const uint16_t* p) { w[0] = ld_mutable(p); }
    __device__ __forceinline__ void store(uint16_t* p) const { *p = uint16_t(w[0]); }
};

// (a, b) of one pair, turned.
__device__ __forceinline__ float2 turned(float a, float b, float2 cs) {
    return make_float2(a * cs.x - b * cs.y, b * cs.x + a * cs.y);
}
template <typename T>
__device__ __forceinline__ float low(uint32_t w) { return Half16<T>::to_float(w & 0xFFFFu); }
template <typename T>
__device__ __forceinline__ float high(uint32_t w) { return Half16<T>::to_float(w >> 16); }

template <typename T, bool NEIGHBOURS, int W, int HELD>
__global__ void __launch_bounds__(kThreads)
rotary_kernel(const __grid_constant__ RotaryArgs a) {
    extern __shared__ float2 turns[];          // [token of the block][pair]
    __shared__ int64_t at[kMaxTokens];         // its position; -1: outside the cache, nothing is stored
    pdl_launch_dependents();
    pdl_wait();
    const int token0 = blockIdx.x * a.block_tokens, tokens = min(a.block_tokens, a.tokens - token0);
    const int head0 = blockIdx.y * a.block_heads, heads = min(a.block_heads, a.heads - head0);
    // Numbers of the unit's two pieces within a head of q or k, and of v; none: < 0.
    struct Unit {
        int first, second;
        bool turns;
    };
    auto of_head = [&](int unit) {
        Unit u;
        u.turns = unit < a.turning;
        const int past = 2 * a.pairs + 2 * W * (unit - a.turning);
        u.first = u.turns ? (NEIGHBOURS ? 2 * W * unit : W * unit) : past < a.head_dim ? past : -1;
        u.second = u.turns ? (NEIGHBOURS ? 2 * W * unit + W : a.pairs + W * unit) : past + W < a.head_dim ? past + W : -1;
        return u;
    };
    auto of_value = [&](int unit) {
        const int at = 2 * W * unit;
        return Unit{at < a.head_dim ? at : -1, at + W < a.head_dim ? at + W : -1, false};
    };
    const int mine = threadIdx.x / a.token_threads, within = threadIdx.x - mine * a.token_threads;
    const int lane_head = a.step > 1 ? within / a.units : 0;
    const bool works = mine < tokens && lane_head < a.step;
    Piece<W> one[HELD], two[HELD];
    auto kind_of = [&](int head) { return head < a.nq ? 0 : head < a.nq + a.nkv ? 1 : 2; };
    auto load = [&](int unit, int h0) {
#pragma unroll
        for (int s = 0; s < HELD; ++s) {
            const int h = h0 + s * a.step;
            if (h >= heads) continue;
            const int head = head0 + h, kind = kind_of(head);
            const Unit u = kind < 2 ? of_head(unit) : of_value(unit);
            const uint16_t* p = a.src[kind] + (token0 + mine) * a.src_token[kind] +
                                (head - (kind > 0 ? a.nq : 0) - (kind > 1 ? a.nkv : 0)) * a.src_head[kind];
            if (u.first >= 0) one[s].load(p + u.first);
            if (u.second >= 0) two[s].load(p + u.second);
        }
    };
    const int unit0 = within - lane_head * a.units;
    if (works && unit0 < a.units) load(unit0, lane_head);

    const int64_t offset = a.offset_at != nullptr ? ld_mutable(a.offset_at) : a.offset;
    for (int i = threadIdx.x; i < tokens * a.pairs; i += kThreads) {
        const int token = i / a.pairs, pair = i - token * a.pairs;
        int64_t position = ld_mutable(a.positions + token0 + token);
        if (a.slots > 0 && (position < 0 || position >= a.slots)) position = 0;
        // turns, less the whole ones; exact to 2^-53 of the turns passed
        const double frequency = __longlong_as_double(ld_mutable(reinterpret_cast<const int64_t*>(a.frequencies) + pair));
        const double turn = double(position + offset) * (frequency * 0.15915494309189533577);
        float s, c;
        sincospif(2.0f * float(turn - rint(turn)), &s, &c);
        turns[i] = make_float2(c * a.factor, s * a.factor);
    }
    if (int(threadIdx.x) < tokens) {
        const int64_t position = ld_mutable(a.positions + token0 + threadIdx.x);
        const bool bad = a.slots > 0 && (position < 0 || position >= a.slots);
        if (bad && head0 == 0) record_bad_position(a.status, token0 + threadIdx.x);
        at[threadIdx.x] = bad ? -1 : position;
    }
    __syncthreads();
    if (!works) return;

    for (int unit = unit0; unit < a.units; unit += a.token_threads) {
        constexpr int kTurns = W;        // pairs of a unit
        float2 cs[kTurns];
        const Unit turning = of_head(unit);
        if (turning.turns) {
            const float2* from = turns + mine * a.pairs + unit * kTurns;
#pragma unroll
            for (int j = 0; j < kTurns; ++j) cs[j] = from[j];
        }
        for (int h0 = lane_head; h0 < heads; h0 += HELD * a.step) {
            if (unit != unit0 || h0 != lane_head) load(unit, h0);
#pragma unroll
            for (int s = 0; s < HELD; ++s) {
                const int h = h0 + s * a.step;
                if (h >= heads) continue;
                const int head = head0 + h, kind = kind_of(head);
                const Unit u = kind < 2 ? turning : of_value(unit);
                if (u.turns) {
                    if constexpr (W == 8 && NEIGHBOURS) {  // a word is a pair
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 x = turned(low<T>(one[s].w[j]), high<T>(one[s].w[j]), cs[j]);
                            const float2 y = turned(low<T>(two[s].w[j]), high<T>(two[s].w[j]), cs[4 + j]);
                            one[s].w[j] = Half16<T>::pack(x.x, x.y);
                            two[s].w[j] = Half16<T>::pack(y.x, y.y);
                        }
                    } else if constexpr (W == 8) {         // a word holds the first (or second) numbers of two pairs
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 x = turned(low<T>(one[s].w[j]), low<T>(two[s].w[j]), cs[2 * j]);
                            const float2 y = turned(high<T>(one[s].w[j]), high<T>(two[s].w[j]), cs[2 * j + 1]);
                            one[s].w[j] = Half16<T>::pack(x.x, y.x);
                            two[s].w[j] = Half16<T>::pack(x.y, y.y);
                        }
                    } else {
                        const float2 x = turned(low<T>(one[s].w[0]), low<T>(two[s].w[0]), cs[0]);
                        one[s].w[0] = Half16<T>::from_float(x.x);
                        two[s].w[0] = Half16<T>::from_float(x.y);
                    }
                }
                uint16_t* p = a.dst[kind] + (token0 + mine) * a.dst_token[kind] +
                              (head - (kind > 0 ? a.nq : 0) - (kind > 1 ? a.nkv : 0)) * a.dst_head[kind];
                if (kind > 0 && a.slots > 0) {
                    if (at[mine] < 0) continue;
                    p += at[mine] * a.head_dim;
                }
                if (u.first >= 0) one[s].store(p + u.first);
                if (u.second >= 0) two[s].store(p + u.second);
            }
        }
    }
}

// table[position][pair] = factor * (cos, sin)(position * frequency), as rotary_kernel has them.
__global__ void rotary_table_kernel(float2* __restrict__ table, const double* frequencies, int pairs, int64_t total,
                                    float factor) {
    pdl_wait();
    for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < total; e += int64_t(gridDim.x) * blockDim.x) {
        const int64_t position = e / pairs;
        const double turn = double(position) * (frequencies[e - position * pairs] * 0.15915494309189533577);
        float s, c;
        sincospif(2.0f * float(turn - rint(turn)), &s, &c);
        table[e] = make_float2(c * factor, s * factor);
    }
}

template <typename T, bool NEIGHBOURS>
cudaError_t launch_width(const RotaryArgs& a, bool wide, bool few, dim3 grid, size_t smem, cudaStream_t stream) {
    auto* kernel = wide ? (few ? rotary_kernel<T, NEIGHBOURS, 8, 1> : rotary_kernel<T, NEIGHBOURS, 8, kHeld>)
                        : (few ? rotary_kernel<T, NEIGHBOURS, 1, 1> : rotary_kernel<T, NEIGHBOURS, 1, kHeld>);
    return launch_overlapped(kernel, grid, dim3(kThreads), smem, stream, a);
}

int32_t launch_rotary(const char* who, RotaryArgs a, int32_t layout, int32_t dtype, cudaStream_t stream) {
    bool wide = a.pairs % 8 == 0 && a.head_dim % 8 == 0;
    const int kinds = a.heads > a.nq + a.nkv ? 3 : a.nkv > 0 ? 2 : 1;
    for (int k = 0; k < kinds; ++k)
        wide = wide && aligned(a.src[k], 16) && aligned(a.dst[k], 16) && a.src_token[k] % 8 == 0 && a.src_head[k] % 8 == 0 &&
               a.dst_token[k] % 8 == 0 && a.dst_head[k] % 8 == 0;
    const int w = wide ? 8 : 1;
    a.turning = a.pairs / w;
    const int copied = (a.head_dim - 2 * a.pairs + 2 * w - 1) / (2 * w), whole = (a.head_dim + 2 * w - 1) / (2 * w);
    a.units = a.turning + copied;
    if (kinds == 3 && a.units < whole) a.units = whole;  // a head of v is copied whole
    // Few units (eight blocks of one a thread on every multiprocessor have them all): one head at a time, the shorter
    // kernel.  16 tokens, 32 + 8 heads of 128: 2.5 us so and 2.8 with five heads in flight; 512 tokens 5.4 so and 4.5; 8192
    // tokens 34.1 so and 33.2 (36.7 with four, 36.0 with eight).
    const int sms = sm_count(), per_token = a.heads * a.units;
    const bool few = int64_t(a.tokens) * per_token <= int64_t(8) * sms * kThreads;
    const int held = few ? 1 : kHeld;
    // As many tokens a block as give a thread about as many heads; with few tokens, fewer, so that every
    // multiprocessor has a block.
    int tokens = 1;
    while (tokens < kMaxTokens && 2 * tokens * a.pairs <= kMaxTurns && kThreads / (2 * tokens) >= a.units &&
           2 * tokens * per_token <= held * kThreads && (a.tokens + 2 * tokens - 1) / (2 * tokens) >= 2 * sms)
        tokens *= 2;
    a.block_tokens = tokens;
    a.token_threads = kThreads / tokens;
    a.step = a.token_threads / a.units > 1 ? a.token_threads / a.units : 1;
    const int blocks = (a.tokens + tokens - 1) / tokens;
    int parts = 2 * sms / blocks;                                    // blocks a token's heads are divided among
    const int most = (per_token + kThreads / 2 - 1) / (kThreads / 2);  // at least half the threads have a unit
    parts = parts > most ? most : parts;
    parts = parts > a.heads ? a.heads : parts < 1 ? 1 : parts;
    a.block_heads = (a.heads + parts - 1) / parts;
    const dim3 grid{unsigned(blocks), unsigned((a.heads + a.block_heads - 1) / a.block_heads)};
    const size_t smem = size_t(tokens) * a.pairs * sizeof(float2);
    cudaError_t err;
    if (dtype == B200Q_BF16)
        err = layout ? launch_width<__nv_bfloat16, true>(a, wide, few, grid, smem, stream)
                     : launch_width<__nv_bfloat16, false>(a, wide, few, grid, smem, stream);
    else
        err = layout ? launch_width<__half, true>(a, wide, few, grid, smem, stream)
                     : launch_width<__half, false>(a, wide, few, grid, smem, stream);
    return launch_status(who, err);
}

// What both entries check before they look at pointers.
int32_t check_rotary(const char* who, int64_t tokens, int64_t nq, int64_t nkv, int64_t head_dim, int64_t pairs,
                     int32_t layout, int32_t dtype) {
    B200Q_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 30) && nq > 0 && nkv >= 0 && nq < 16384 && nkv < 16384,
                  "%s: bad shape", who);
    B200Q_REQUIRE(head_dim > 0 && head_dim <= 1024 && pairs > 0 && 2 * pairs <= head_dim,
                  "%s: %lld pairs of a head of %lld numbers (1024 at most)", who, (long long)pairs, (long long)head_dim);
    B200Q_REQUIRE(layout == 0 || layout == 1, "%s: layout is 0 (halves) or 1 (neighbours)", who);
    B200Q_REQUIRE(dtype == B200Q_BF16 || dtype == B200Q_F16, "%s: bf16 or f16", who);
    return B200Q_OK;
}

// Whether heads of an output share memory.  (A sufficient rule for those that do not: the farther apart of its two
// dimensions steps over all that the nearer one spans.)
bool overlaps_itself(int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride, int64_t head_dim) {
    __int128 inner = head_stride, outer = token_stride;
    int64_t inner_count = heads, outer_count = tokens;
    if (inner < 0) inner = -inner;
    if (outer < 0) outer = -outer;
    if (outer_count <= 1 || (inner_count > 1 && outer < inner)) {
        const __int128 stride = inner;
        const int64_t count = inner_count;
        inner = outer, inner_count = outer_count, outer = stride, outer_count = count;
    }
    if (inner_count <= 1) return outer_count > 1 && outer < head_dim;
    return inner < head_dim || (outer_count > 1 && outer < inner * (inner_count - 1) + head_dim);
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int32_t b200q_rotary(const void* q, const void* k, const int64_t* positions, const double* frequencies,
                                void* q_out, void* k_out, int64_t tokens, int64_t nq, int64_t nkv, int64_t head_dim,
                                int64_t pairs, int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head,
                                int64_t q_out_token, int64_t q_out_head, int64_t k_out_token, int64_t k_out_head,
                                float factor, int32_t layout, int32_t dtype, void* stream) {
    const int32_t checked = check_rotary("rotary", tokens, nq, nkv, head_dim, pairs, layout, dtype);
    if (checked != B200Q_OK || tokens == 0) return checked;
    B200Q_REQUIRE(q && q_out && positions && frequencies && (nkv == 0 || (k && k_out)) && aligned(q, 2) && aligned(q_out, 2) &&
                      aligned(k, 2) && aligned(k_out, 2) && aligned(positions, 8) && aligned(frequencies, 8),
                  "rotary: null or misaligned tensor");
    B200Q_REQUIRE(!overlaps_itself(tokens, q_out_token, nq, q_out_head, head_dim) &&
                      (nkv == 0 || !overlaps_itself(tokens, k_out_token, nkv, k_out_head, head_dim)),
                  "rotary: an output overlaps itself");
    RotaryArgs a = {};
    a.src[0] = static_cast<const uint16_t*>(q), a.dst[0] = static_cast<uint16_t*>(q_out);
    a.src[1] = static_cast<const uint16_t*>(k), a.dst[1] = static_cast<uint16_t*>(k_out);
    a.src_token[0] = q_token, a.src_head[0] = q_head, a.dst_token[0] = q_out_token, a.dst_head[0] = q_out_head;
    a.src_token[1] = k_token, a.src_head[1] = k_head, a.dst_token[1] = k_out_token, a.dst_head[1] = k_out_head;
    a.positions = positions, a.frequencies = frequencies, a.factor = factor;
    a.tokens = int(tokens), a.nq = int(nq), a.nkv = int(nkv), a.heads = int(nq + nkv);
    a.pairs = int(pairs), a.head_dim = int(head_dim);
    return launch_rotary("rotary", a, layout, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int32_t b200q_rotary_cache(const void* qkv, const int64_t* positions, const double* frequencies,
                                      const int64_t* offset_at, int64_t offset, void* q_out, void* cache_k, void* cache_v,
                                      int64_t batch, int64_t nq, int64_t nkv, int64_t head_dim, int64_t pairs,
                                      int64_t max_seq, float factor, int32_t layout, int32_t dtype, void* stream) {
    const int32_t checked = check_rotary("rotary_cache", batch, nq, nkv, head_dim, pairs, layout, dtype);
    if (checked != B200Q_OK) return checked;
    B200Q_REQUIRE(nkv > 0 && max_seq > 0, "rotary_cache: bad shape");
    if (batch == 0) return B200Q_OK;
    B200Q_REQUIRE(qkv && positions && frequencies && q_out && cache_k && cache_v && aligned(qkv, 2) && aligned(q_out, 2) &&
                      aligned(cache_k, 2) && aligned(cache_v, 2) && aligned(positions, 8) && aligned(frequencies, 8) &&
                      aligned(offset_at, 8),
                  "rotary_cache: null or misaligned tensor");
    RotaryArgs a = {};
    const uint16_t* from = static_cast<const uint16_t*>(qkv);
    const int64_t row = (nq + 2 * nkv) * head_dim;
    for (int kind = 0; kind < 3; ++kind) {
        a.src[kind] = from + (kind > 0 ? nq : 0) * head_dim + (kind > 1 ? nkv : 0) * head_dim;
        a.src_token[kind] = row, a.src_head[kind] = head_dim;
        a.dst_token[kind] = kind == 0 ? nq * head_dim : nkv * max_seq * head_dim;
        a.dst_head[kind] = kind == 0 ? head_dim : max_seq * head_dim;
    }
    a.dst[0] = static_cast<uint16_t*>(q_out), a.dst[1] = static_cast<uint16_t*>(cache_k);
    a.dst[2] = static_cast<uint16_t*>(cache_v);
    a.positions = positions, a.frequencies = frequencies, a.factor = factor;
    a.offset_at = offset_at, a.offset = offset, a.slots = max_seq, a.status = decoder_error_word();
    a.tokens = int(batch), a.nq = int(nq), a.nkv = int(nkv), a.heads = int(nq + 2 * nkv);
    a.pairs = int(pairs), a.head_dim = int(head_dim);
    return launch_rotary("rotary_cache", a, layout, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int32_t b200q_rotary_table(void* table, const double* frequencies, int64_t max_seq, int64_t pairs, float factor,
                                      void* stream) {
    B200Q_REQUIRE(table && frequencies && aligned(table, 8) && aligned(frequencies, 8) && max_seq > 0 && pairs > 0 &&
                      pairs <= 512 && max_seq < (int64_t(1) << 40),
                  "rotary_table: bad arguments");
    const int64_t total = max_seq * pairs, blocks = (total + 255) / 256;
    return launch_status("rotary_table",
                         launch_overlapped(rotary_table_kernel, dim3(unsigned(blocks > 4096 ? 4096 : blocks)), dim3(256), 0,
                                           static_cast<cudaStream_t>(stream), static_cast<float2*>(table), frequencies,
                                           int(pairs), total, factor));
}
