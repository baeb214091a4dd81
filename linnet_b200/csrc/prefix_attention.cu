// Single-query attention of a batch whose rows share a long prefix (many answers to one prompt):
//     out[b, head] = sum_j softmax_j(scale * q[b, head] . k_j) v_j
// over the prefix's keys (one copy for the batch) and then the row's own, 0 .. positions[b] of its
// cache.  Row by row the prefix would be read once a row; here all rows of a KV head that share it are
// the 128 rows of a tcgen05 product, so its keys and values cross HBM once.
//
// Work is cut into TILES of 128 keys.  An ITEM is the prefix of one KV head for up to 256 query rows
// (rep = heads / kv_heads rows a batch row), or one batch row's own keys of one KV head.  The items'
// tiles stand in one sequence, prefix first, and block c of G takes the c-th G-th of it, so blocks
// have equal work whatever the lengths; where a block's share begins and ends, an item is cut into
// PIECES, each with its own softmax statistics, and a second kernel joins the pieces of a row.  An
// item and a block have at most one piece in common, and (item + block) grows along the sequence:
// that is a piece's place in the scratch memory.
//
// A block: two softmax groups (4 warps, one query row a thread), a TMA producer, an issuer of the
// products, a loader of queries.  Per task (a tile for one group):
//   S [128 rows x 128 keys] = Q . K^T      Q and K in shared memory as TMA's 128-byte swizzle has them
//   P = 2^(scale' S - m), l += sum P       one row a thread: no exchange between threads
//   O [128 rows x D] += P . V              P in tensor memory over S's columns; V's rows are the keys, so
//                                          it is the MN-major operand as it lies in memory
// An item of more than 128 rows gives each group half of the rows and both every tile; one of fewer
// gives both groups the same rows and alternate tiles.  Either way one group's products run while
// the other has its exponentials.
// m is a row's maximum of the first tile; a later tile whose own exceeds it by more than 2^8 moves it
// and rescales O and l in tensor memory (rare: P stays below 2^8, and the sums are f32 anyway).
// P is rounded to the tensors' type, as the product takes it; l sums P before that rounding.
//
// What bounds it: few rows, HBM (64 KB a tile of 128 keys at D = 128); many rows, the two products
// (1024 clocks a task) and the 128 x 128 exponentials (1024 clocks of the special-function unit), which
// overlap between the two groups.
#include "mma.cuh"
#include "umma.cuh"

namespace b200q {
namespace {

using namespace umma;

constexpr int kKeys = 128;                 // of a tile
constexpr int kRows = 128;                 // of a group's products
constexpr int kProducerWarp = 8, kIssuerWarp = 9, kQueryWarp = 10;
constexpr int kThreads = 11 * 32;
constexpr uint32_t kTmemColumns = 512;     // S of both groups, O of both groups
constexpr float kStale = 8.0f;             // how far (log2) a tile's maximum may exceed the row's before it moves

template <int HD>
struct Shape {
    static constexpr int kHalves = HD / 64;                    // 128-byte columns of a tile
    static constexpr uint32_t kHalf = kKeys * 128;             // bytes of one
    static constexpr uint32_t kSlot = kHalves * kHalf;         // a tile of K or V
    static constexpr int kSlots = HD == 128 ? 5 : 10;
    static constexpr uint32_t kQuery = kHalves * kRows * 128;  // a group's queries; two of them
    static constexpr uint32_t kBytes = 2 * kQuery + kSlots * kSlot;
};

struct PrefixArgs {
    const uint16_t* q;
    int64_t q_row, q_head;                 // strides, in numbers
    const int64_t* positions;
    const int64_t* prefix_at;              // its length on the device, or null: `prefix`
    uint16_t* out;
    float* scratch;
    int* cum;                              // [batch + 1]: tiles of a KV head before row b; then the total, then tiles of an item's prefix
    int batch, nq, nkv, rep, prefix, slots;  // slots: of a row's own cache
    int tile_rows;                         // batch rows of a group's products: 128 / rep
    int row_tiles, items;                  // of the prefix: ceil(batch / 2 tile_rows), that times nkv
    int64_t own_at;                        // where the scratch memory of own pieces begins, in floats
    float scale_log2;
    int* status;
    int* error;
};

// ---- the sequence of tiles ---------------------------------------------------------------------

__device__ __forceinline__ int own_tiles(const PrefixArgs& a, int64_t position) {
    const int keys = position < -1 || position >= a.slots ? 0 : int(position) + 1;  // outside the cache: none
    return (keys + kKeys - 1) / kKeys;
}
__device__ __forceinline__ int prefix_length(const PrefixArgs& a) {
    if (a.prefix_at == nullptr) return a.prefix;
    const int64_t given = ld_mutable(a.prefix_at);
    return int(given < 0 ? 0 : given > a.prefix ? a.prefix : given);
}
// The first tile of block c, and the block that takes tile t, of `total` over `blocks`: no more of
// them than tiles, so that none between two has nothing.
__device__ __forceinline__ int first_tile(int c, int total, int blocks) {
    return total <= blocks ? min(c, total) : int(int64_t(total) * c / blocks);
}
__device__ __forceinline__ int block_of(int t, int total, int blocks) {
    return total <= blocks ? t : int(((int64_t(t) + 1) * blocks - 1) / total);
}

struct Share {  // of a block; in shared memory
    int total, first, last;   // tiles
    int prefix_keys, prefix_tiles;
    int row, row_tile;        // the batch row whose own tiles hold the first own tile of the share, and where that row begins
};

struct Piece {
    int place;                // item + block: of the scratch memory
    bool prefix, both;        // both: the groups take different rows (else alternate tiles)
    int head, row, rows;      // KV head, first batch row, batch rows
    int key, keys, tiles;     // first key, keys to the end of the item, tiles
};

// The pieces of a block's share, in order.  Every role walks it for itself.
struct Walk {
    int t, row, at;           // next tile; the batch row that own tiles are looked up in, and its first tile
    int64_t position, next;   // of that row and of the one after (read ahead)
    __device__ __forceinline__ Walk(const PrefixArgs& a, const Share& s) {
        t = s.first, row = s.row, at = s.row_tile;
        position = row < a.batch ? ld_mutable(a.positions + row) : -1;
        next = row + 1 < a.batch ? ld_mutable(a.positions + row + 1) : -1;
    }
    __device__ __forceinline__ bool step(const PrefixArgs& a, const Share& s, Piece& p) {
        if (t >= s.last) return false;
        const int prefix_total = a.items * s.prefix_tiles;
        if (t < prefix_total) {
            const int item = t / s.prefix_tiles, skipped = t - item * s.prefix_tiles;
            p.prefix = true;
            p.head = item / a.row_tiles;
            p.row = (item - p.head * a.row_tiles) * 2 * a.tile_rows;
            p.rows = min(2 * a.tile_rows, a.batch - p.row);
            p.both = p.rows > a.tile_rows;
            p.key = skipped * kKeys, p.keys = s.prefix_keys - p.key;
            p.tiles = min(s.prefix_tiles - skipped, s.last - t);
            p.place = item + int(blockIdx.x);
        } else {
            int each = own_tiles(a, position);
            while (t >= at + each * a.nkv) {  // (t is before the end of the sequence: some row has it)
                at += each * a.nkv;
                position = next, ++row;
                next = row + 1 < a.batch ? ld_mutable(a.positions + row + 1) : -1;
                each = own_tiles(a, position);
            }
            p.prefix = false, p.both = false;
            p.head = (t - at) / each;
            const int skipped = t - at - p.head * each;
            p.row = row, p.rows = 1;
            p.key = skipped * kKeys, p.keys = int(position) + 1 - p.key;
            p.tiles = min(each - skipped, s.last - t);
            p.place = row * a.nkv + p.head + int(blockIdx.x);
        }
        t += p.tiles;
        return true;
    }
};

// Place of a tile's K and V among the loads of a piece: the order in which the products want them
// (K of the task after next comes before V of the next one).
__device__ __forceinline__ int place_of_k(const Piece& p, int tile) { return p.both ? 2 * tile : tile < 2 ? tile : 2 * tile - 1; }
__device__ __forceinline__ int place_of_v(const Piece& p, int tile) {
    return p.both ? 2 * tile + 1 : tile == p.tiles - 1 ? 2 * tile + 1 : 2 * tile + 2;
}

// ---- scratch memory: of a piece, per group, O as [D / 4][rows] float4, then m [rows] and l [rows] ----

// (a whole number of 16-byte steps)
__host__ __device__ constexpr int64_t group_floats(int rows, int hd) { return (int64_t(rows) * (hd + 2) + 3) / 4 * 4; }

// ---- instructions --------------------------------------------------------------------------------

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}
// D[tmem] (+)= A[smem] . B[smem]^T, and with A in tensor memory: 128 x N x 16, 16-bit, f32 accumulate.
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 32 columns of this thread's lane: asked for; there after tmem_arrived() of all that were asked for.
__device__ __forceinline__ void tmem_ask_32(uint32_t* v, uint32_t taddr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_arrived(uint32_t* v) {  // (v passes through: no use of it moves above)
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                   "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                   "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_put_32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {  // relative error 2^-22
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2,%3};\nmov.b64 y, {%4,%5};\nadd.rn.f32x2 z, x, y;\nmov.b64 {%0,%1}, z;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2,%3};\nmov.b64 y, {%4,%5};\nmov.b64 z, {%6,%7};\n"
        "fma.rn.f32x2 w, x, y, z;\nmov.b64 {%0,%1}, w;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
// V, MN-major with the 128-byte swizzle: rows (keys) of 128 bytes, 8-row atoms 1024 bytes apart along
// the keys, columns 64..127 of D a half further.
__device__ __forceinline__ uint64_t value_desc(uint32_t addr, uint32_t half) {
    return uint64_t((addr & 0x3FFFFu) >> 4) | (uint64_t(half >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

struct Barriers {
    uint64_t full[10], empty[10];          // tiles of K and V
    uint64_t query_full[2], query_empty[2];
    uint64_t scores[2], weights[2], result[2];  // of the groups: S is there, P is there, O of a piece is complete
    uint32_t tmem_base;
};

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
prefix_attention_kernel(const __grid_constant__ CUtensorMap prefix_k, const __grid_constant__ CUtensorMap prefix_v,
                        const __grid_constant__ CUtensorMap cache_k, const __grid_constant__ CUtensorMap cache_v,
                        const __grid_constant__ PrefixArgs a) {
    using H = Half16<T>;
    using S = Shape<HD>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* slots = smem + 2 * S::kQuery;
    __shared__ Barriers bars;
    __shared__ Share share;
    __shared__ int warp_tiles[kThreads / 32];
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) / 32, 0), lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kSlots; ++s) mbar_init(&bars.full[s], 1), mbar_init(&bars.empty[s], 1);
        for (int g = 0; g < 2; ++g) {
            mbar_init(&bars.query_full[g], 1), mbar_init(&bars.query_empty[g], 1);
            mbar_init(&bars.scores[g], 1), mbar_init(&bars.weights[g], 4), mbar_init(&bars.result[g], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssuerWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)),
                     "r"(kTmemColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_launch_dependents();
    pdl_wait();

    // ---- this block's share: every thread sums some rows' own tiles ----
    {
        const int per = (a.batch + kThreads - 1) / kThreads, from = min(int(threadIdx.x) * per, a.batch), to = min(from + per, a.batch);
        int mine = 0;
        for (int b = from; b < to; ++b) {
            const int64_t position = ld_mutable(a.positions + b);
            if (blockIdx.x == 0 && (position < -1 || position >= a.slots)) record_bad_position(a.status, b);
            mine += own_tiles(a, position);
        }
        int before = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int other = __shfl_up_sync(0xFFFFFFFFu, before, d);
            if (lane >= d) before += other;
        }
        if (lane == 31) warp_tiles[warp] = before;
        before -= mine;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += warp_tiles[w];
            all += warp_tiles[w];
        }
        const int keys = prefix_length(a), tiles = (keys + kKeys - 1) / kKeys;
        if (a.prefix_at != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
            const int64_t given = ld_mutable(a.prefix_at);
            if (given < 0 || given > a.prefix) record_bad_position(a.status, 0);
        }
        const int own_first = a.items * tiles, total = own_first + all * a.nkv;
        const int first = first_tile(blockIdx.x, total, gridDim.x), last = first_tile(blockIdx.x + 1, total, gridDim.x);
        const int look = max(first, own_first);  // the first own tile this block can have
        if (threadIdx.x == 0) {
            share.total = total, share.first = first, share.last = last;
            share.prefix_keys = keys, share.prefix_tiles = tiles;
            if (look >= total) share.row = a.batch, share.row_tile = total;
        }
        const int begin = own_first + before * a.nkv, end = begin + mine * a.nkv;
        if (look >= begin && look < end) {
            int row = from, at = begin;
            for (;;) {
                const int each = own_tiles(a, ld_mutable(a.positions + row));
                if (look < at + each * a.nkv) break;
                at += each * a.nkv, ++row;
            }
            share.row = row, share.row_tile = at;
        }
        if (blockIdx.x == 0) {  // for the joining kernel
            int c = before;
            for (int b = from; b < to; ++b) {
                a.cum[b] = c;
                c += own_tiles(a, ld_mutable(a.positions + b));
            }
            if (threadIdx.x == 0) a.cum[a.batch] = total, a.cum[a.batch + 1] = tiles;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem_base);

    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {  // of a whole warp; bounded
        return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, a.error, code));
    };
    Walk walk(a, share);
    Piece p;
    bool ok = true;

    if (warp == kProducerWarp) {
        uint32_t n = 0;  // loads so far
        while (ok && walk.step(a, share, p)) {
            for (int i = 0; i < 2 * p.tiles && ok; ++i, ++n) {
                // the i-th load of the piece
                int tile, value;
                if (p.both) tile = i >> 1, value = i & 1;
                else if (i < 2) tile = p.tiles > 1 ? i : 0, value = p.tiles > 1 ? 0 : i;
                else if (i == 2 * p.tiles - 1) tile = p.tiles - 1, value = 1;
                else tile = (i & 1) ? (i + 1) / 2 : (i - 2) / 2, value = (i & 1) ^ 1;
                const uint32_t slot = n % S::kSlots, lap = n / S::kSlots;
                if (lap > 0) ok = wait(&bars.empty[slot], (lap - 1) & 1, 41);
                if (!ok) break;
                if (lane == 0) {
                    mbar_expect_tx(&bars.full[slot], S::kSlot);
                    const int key = p.key + tile * kKeys;
#pragma unroll
                    for (int h = 0; h < S::kHalves; ++h) {
                        const uint32_t dst = smem_u32(slots) + slot * S::kSlot + h * S::kHalf;
                        if (p.prefix) tma_load_3d(dst, value ? &prefix_v : &prefix_k, h * 64, key, p.head, &bars.full[slot]);
                        else tma_load_4d(dst, value ? &cache_v : &cache_k, h * 64, key, p.head, p.row, &bars.full[slot]);
                    }
                }
                __syncwarp();
            }
        }
        if (!ok)  // what is in flight lands before the block leaves
            for (uint32_t i = n > S::kSlots ? n - S::kSlots : 0; i < n; ++i) mbar_wait(&bars.full[i % S::kSlots], (i / S::kSlots) & 1, a.error, 42);
    } else if (warp == kIssuerWarp) {
        constexpr uint32_t kType = H::kDtype == B200Q_BF16 ? 1u : 0u;
        constexpr uint32_t kScores = (1u << 4) | (kType << 7) | (kType << 10) | (uint32_t(kKeys >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
        constexpr uint32_t kValues = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | (uint32_t(HD >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
        const bool leader = elect_one();
        uint32_t n = 0, queries = 0, done[2] = {0, 0};  // loads, query buffers and tasks of the groups before this piece
        while (ok && walk.step(a, share, p)) {
            const int tasks = p.both ? 2 * p.tiles : p.tiles;
            auto scores = [&](int t) {
                const int g = t & 1, tile = p.both ? t >> 1 : t;
                const uint32_t query = queries + (p.both ? uint32_t(g) : 0u), buffer = query & 1;
                if (t < 2) ok = wait(&bars.query_full[buffer], (query >> 1) & 1, 43);
                const uint32_t load = n + uint32_t(place_of_k(p, tile)), slot = load % S::kSlots;
                ok = ok && wait(&bars.full[slot], (load / S::kSlots) & 1, 44);
                if (!ok) return;
                tc_fence_after();
                if (leader) {
                    const uint64_t qd = smem_desc(smem_u32(smem) + buffer * S::kQuery), kd = smem_desc(smem_u32(slots) + slot * S::kSlot);
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint32_t step = uint32_t(k / 4) * (S::kHalf >> 4) + uint32_t(k % 4) * 2;
                        umma_f16_ss(tmem + uint32_t(g) * kKeys, qd + step, kd + step, kScores, k > 0);
                    }
                    umma_commit(&bars.scores[g]);
                    if (!p.both || g == 1) umma_commit(&bars.empty[slot]);
                    if (p.both ? t >= tasks - 2 : t == tasks - 1) umma_commit(&bars.query_empty[buffer]);
                }
                __syncwarp();
            };
            scores(0);
            if (ok && tasks > 1) scores(1);
            for (int t = 0; t < tasks && ok; ++t) {
                const int g = t & 1, tile = p.both ? t >> 1 : t;
                ok = wait(&bars.weights[g], done[g] & 1, 45);
                const uint32_t load = n + uint32_t(place_of_v(p, tile)), slot = load % S::kSlots;
                ok = ok && wait(&bars.full[slot], (load / S::kSlots) & 1, 46);
                if (!ok) break;
                ++done[g];
                tc_fence_after();
                if (leader) {
                    const uint64_t vd = value_desc(smem_u32(slots) + slot * S::kSlot, S::kHalf);
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        umma_f16_ts(tmem + 2 * kKeys + uint32_t(g) * HD, tmem + uint32_t(g) * kKeys + k * 8, vd + uint32_t(k) * (2048 >> 4),
                                    kValues, k > 0 || t >= 2);
                    if (!p.both || g == 1) umma_commit(&bars.empty[slot]);
                    if (t >= tasks - 2) umma_commit(&bars.result[g]);
                }
                __syncwarp();
                if (t + 2 < tasks) scores(t + 2);
            }
            n += 2 * uint32_t(p.tiles);
            queries += p.both ? 2 : 1;
        }
    } else if (warp == kQueryWarp) {
        uint32_t query = 0;
        while (ok && walk.step(a, share, p)) {
            for (int g = 0; g < (p.both ? 2 : 1) && ok; ++g, ++query) {
                const uint32_t buffer = query & 1;
                if (query >= 2) ok = wait(&bars.query_empty[buffer], ((query >> 1) - 1) & 1, 47);
                if (!ok) break;
                const int row0 = p.row + g * a.tile_rows, rows = min(a.tile_rows, p.row + p.rows - row0) * a.rep;
                const uint32_t to = smem_u32(smem) + buffer * S::kQuery;
                constexpr int kPieces = HD / 8;  // of 16 bytes a row
                for (int i = lane; i < rows * kPieces; i += 32) {
                    const int r = i / kPieces, c = i % kPieces, b = r / a.rep;
                    const uint16_t* src = a.q + (row0 + b) * a.q_row + (p.head * a.rep + r - b * a.rep) * a.q_head + c * 8;
                    const uint32_t dst = to + uint32_t(c / 8) * (kRows * 128) + uint32_t(r) * 128 + uint32_t(((c % 8) ^ (r & 7)) << 4);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.query_full[buffer]);
            }
        }
    } else {
        // ---- softmax: group g, one query row a thread ----
        const int g = warp / 4, row = threadIdx.x % 128;
        const uint32_t lanes = tmem + (uint32_t(warp & 3) << 21);
        const uint32_t s_at = lanes + uint32_t(g) * kKeys, o_at = lanes + 2 * kKeys + uint32_t(g) * HD;
        uint32_t n = 0, done = 0, pieces = 0;  // loads, tasks of this group and pieces with any before this one
        while (ok && walk.step(a, share, p)) {
            const int live = p.both ? min(a.tile_rows, p.rows - g * a.tile_rows) * a.rep : p.rows * a.rep;
            const bool any = (warp & 3) * 32 < live;  // of this warp's rows
            const int first = p.both ? 0 : g, stride = p.both ? 1 : 2;
            float m = -INFINITY, l = 0.0f;
            for (int tile = first; tile < p.tiles && ok; tile += stride) {
                ok = wait(&bars.scores[g], done & 1, 48);
                if (!ok) break;
                ++done;
                tc_fence_after();
                const int valid = p.keys - tile * kKeys;  // keys of the tile, and more
                if (any) {
                    uint32_t v[kKeys];
#pragma unroll
                    for (int i = 0; i < 4; ++i) tmem_ask_32(v + 32 * i, s_at + 32 * i);
#pragma unroll
                    for (int i = 0; i < 4; ++i) tmem_arrived(v + 32 * i);
                    if (valid < kKeys) {
#pragma unroll
                        for (int i = 0; i < kKeys; ++i)
                            if (i >= valid) v[i] = 0xFF800000u;
                    }
                    float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < kKeys; i += 4)
#pragma unroll
                        for (int j = 0; j < 4; ++j) most[j] = fmaxf(most[j], __uint_as_float(v[i + j]));
                    const float here = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * a.scale_log2;
                    if (tile == first) {
                        m = here == -INFINITY ? 0.0f : here;
                    } else if (__any_sync(0xFFFFFFFFu, row < live && here > m + kStale)) {
                        const float next = here > m + kStale ? here : m, by = exp2_approx(m - next);
                        m = next;
                        l *= by;
#pragma unroll
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            tmem_ask_32(o, o_at + c);
                            tmem_arrived(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
                            tmem_put_32(o_at + c, o);
                        }
                    }
                    const float2 scale = make_float2(a.scale_log2, a.scale_log2), minus = make_float2(-m, -m);
                    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t w[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int at = 64 * h + 2 * i;
                            const float2 t = fma2(make_float2(__uint_as_float(v[at]), __uint_as_float(v[at + 1])), scale, minus);
                            const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
                            sum = add2(sum, e);
                            w[i] = H::pack(e.x, e.y);
                        }
                        tmem_put_32(s_at + 32 * h, w);
                    }
                    l += sum.x + sum.y;
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                if (valid < kKeys && (!p.both || g == 0)) {
                    // Rows of V past the last key may hold anything, and 0 * NaN is no 0.
                    const uint32_t load = n + uint32_t(place_of_v(p, tile)), slot = load % S::kSlots;
                    ok = wait(&bars.full[slot], (load / S::kSlots) & 1, 49);
                    if (!ok) break;
                    uint8_t* tail = slots + slot * S::kSlot;
                    for (int i = row; i < (kKeys - valid) * 8 * S::kHalves; i += 128) {
                        const int h = i / ((kKeys - valid) * 8), rest = i - h * (kKeys - valid) * 8;
                        *reinterpret_cast<uint4*>(tail + h * S::kHalf + valid * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.weights[g]);
            }
            if (!ok) break;
            // ---- the piece's result ----
            const int span = p.prefix ? kRows : a.rep;  // rows of a group in the scratch memory
            float* to = a.scratch + (p.prefix ? 0 : a.own_at) + (2 * int64_t(p.place) + g) * group_floats(span, HD);
            const bool worked = first < p.tiles;
            if (worked) {
                ok = wait(&bars.result[g], pieces & 1, 50);
                if (!ok) break;
                ++pieces;
                tc_fence_after();
                if (any) {
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tmem_ask_32(o, o_at + c);
                        tmem_arrived(o);
                        if (row < live) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                reinterpret_cast<uint4*>(to)[((c + i) / 4) * span + row] = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        }
                    }
                }
            }
            if (row < live) {
                to[int64_t(HD) * span + row] = worked ? m : -INFINITY;
                to[int64_t(HD + 1) * span + row] = l;
            }
            n += 2 * uint32_t(p.tiles);
        }
    }

    // Every role falls through to here, also after an expired wait.
    tc_fence_before();
    __syncthreads();
    if (warp == kIssuerWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
    }
}

// ---- joining the pieces of a row ----------------------------------------------------------------
// One query row a lane; the D / 4 columns of four numbers are dealt among warps and blocks, two a
// thread.  out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i in f32; a row without any key is 0.
constexpr int kJoinWarps = 4, kJoinColumns = 2;

template <typename T, int HD>
__global__ void __launch_bounds__(32 * kJoinWarps)
prefix_join_kernel(const __grid_constant__ PrefixArgs a, int blocks) {
    using H = Half16<T>;
    pdl_launch_dependents();
    pdl_wait();
    const int head = blockIdx.y, row = blockIdx.x * 32 + threadIdx.x % 32;  // batch row * rep + head of the group
    const int column = (blockIdx.z * kJoinWarps + threadIdx.x / 32) * kJoinColumns;
    if (row >= a.batch * a.rep) return;
    const int b = row / a.rep, r = row - b * a.rep;
    auto word = [&](int i) { return int(ld_mutable(reinterpret_cast<const uint32_t*>(a.cum) + i)); };
    const int total = word(a.batch), prefix_tiles = word(a.batch + 1);

    struct Item {              // the prefix, and the row's own keys
        const float* base;     // of the first group that has the row, in the first piece
        int parts, groups;     // groups that have the row: over all pieces, and of a piece
        int span, at;          // rows of a group in the scratch memory, and which one this is
    } items[2] = {};
    if (prefix_tiles > 0) {
        const int pair = b / (2 * a.tile_rows), within = b - pair * 2 * a.tile_rows;
        const bool both = min(2 * a.tile_rows, a.batch - pair * 2 * a.tile_rows) > a.tile_rows;
        const int item = head * a.row_tiles + pair, first = item * prefix_tiles;
        const int from = block_of(first, total, blocks), to = block_of(first + prefix_tiles - 1, total, blocks);
        const int g = both && within >= a.tile_rows;
        items[0].base = a.scratch + (2 * int64_t(item + from) + g) * group_floats(kRows, HD);
        items[0].groups = both ? 1 : 2, items[0].parts = (to - from + 1) * items[0].groups;
        items[0].span = kRows, items[0].at = (within - g * a.tile_rows) * a.rep + r;
    }
    const int each = own_tiles(a, ld_mutable(a.positions + b));
    if (each > 0) {
        const int first = a.items * prefix_tiles + word(b) * a.nkv + head * each;
        const int from = block_of(first, total, blocks), to = block_of(first + each - 1, total, blocks);
        items[1].base = a.scratch + a.own_at + 2 * int64_t(b * a.nkv + head + from) * group_floats(a.rep, HD);
        items[1].groups = 2, items[1].parts = (to - from + 1) * 2;
        items[1].span = a.rep, items[1].at = r;
    }
    auto part = [&](const Item& it, int k) {
        return it.base + (it.groups == 2 ? k : 2 * k) * group_floats(it.span, HD);
    };
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll 8
        for (int k = 0; k < items[i].parts; ++k) m = fmaxf(m, ld_mutable(part(items[i], k) + HD * items[i].span + items[i].at));
    float l = 0.0f, o[4 * kJoinColumns] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const Item& it = items[i];
#pragma unroll 4
        for (int k = 0; k < it.parts; ++k) {
            const float* from = part(it, k);
            const float theirs = ld_mutable(from + HD * it.span + it.at);
            if (theirs == -INFINITY) continue;  // a group that had no tile of the piece: nothing else is there
            const float weight = exp2_approx(theirs - m);
            l += weight * ld_mutable(from + (HD + 1) * it.span + it.at);
#pragma unroll
            for (int c = 0; c < kJoinColumns; ++c) {
                const uint4 v = ld_mutable(reinterpret_cast<const uint4*>(from) + (column + c) * it.span + it.at);
                o[4 * c] += weight * __uint_as_float(v.x), o[4 * c + 1] += weight * __uint_as_float(v.y);
                o[4 * c + 2] += weight * __uint_as_float(v.z), o[4 * c + 3] += weight * __uint_as_float(v.w);
            }
        }
    }
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* to = a.out + (int64_t(b) * a.nq + head * a.rep + r) * HD + column * 4;
    *reinterpret_cast<uint4*>(to) = make_uint4(H::pack(o[0] * by, o[1] * by), H::pack(o[2] * by, o[3] * by),
                                               H::pack(o[4] * by, o[5] * by), H::pack(o[6] * by, o[7] * by));
}

// ---- host -----------------------------------------------------------------------------------------

struct PrefixPlan {
    int tile_rows, row_tiles, items, blocks;
    int64_t own_at, cum_at, floats;
};

PrefixPlan plan_of(int64_t batch, int64_t nkv, int64_t rep, int64_t hd, int64_t prefix, int64_t slots) {
    PrefixPlan p;
    p.tile_rows = int(kRows / rep);
    p.row_tiles = prefix > 0 ? int((batch + 2 * p.tile_rows - 1) / (2 * p.tile_rows)) : 0;
    p.items = int(nkv) * p.row_tiles;
    p.blocks = sm_count();
    const int64_t tiles = p.items * ((prefix + kKeys - 1) / kKeys) + batch * nkv * ((slots + kKeys - 1) / kKeys);
    if (tiles < p.blocks) p.blocks = tiles < 1 ? 1 : int(tiles);
    p.own_at = (p.items > 0 ? p.items + p.blocks : 0) * 2 * group_floats(kRows, int(hd));
    p.cum_at = p.own_at + (batch * nkv + p.blocks) * 2 * group_floats(int(rep), int(hd));
    p.floats = p.cum_at + (batch + 2 + 3) / 4 * 4;
    return p;
}

int32_t check_prefix(int64_t batch, int64_t nq, int64_t nkv, int64_t hd, int64_t prefix, int64_t slots) {
    B200Q_REQUIRE(batch >= 0 && batch <= 65536 && nq > 0 && nkv > 0 && nkv <= 65535 && nq % nkv == 0 && nq / nkv <= kRows,
                  "prefix_attention: up to 65536 rows, heads / kv_heads a whole number up to 128; not %lld rows of %lld / %lld",
                  (long long)batch, (long long)nq, (long long)nkv);
    B200Q_REQUIRE(hd == 64 || hd == 128, "prefix_attention: head_dim is 64 or 128, not %lld", (long long)hd);
    B200Q_REQUIRE(prefix >= 0 && prefix < (int64_t(1) << 30) && slots >= 0 && slots < (int64_t(1) << 30),
                  "prefix_attention: bad length of the prefix or the cache");
    const int64_t row_tiles = batch / (2 * (kRows / (nq / nkv))) + 1;
    B200Q_REQUIRE(nkv * row_tiles * (prefix / kKeys + 1) + batch * nkv * (slots / kKeys + 1) < (int64_t(1) << 30) &&
                      batch * nq < (int64_t(1) << 30),
                  "prefix_attention: more than 2^30 tiles of 128 keys, or rows times heads");
    return B200Q_OK;
}

// A map of keys or values [extents][hd], 64 numbers x 128 keys a box; strides in numbers.
CUresult make_map(EncodeTiled encode, CUtensorMap* map, const void* base, int32_t dtype, int rank, const int64_t* extents,
                  const int64_t* strides) {
    cuuint64_t dims[4], bytes[3];
    cuuint32_t box[4] = {64, cuuint32_t(kKeys), 1, 1}, elem[4] = {1, 1, 1, 1};
    int64_t dense = extents[0];
    for (int d = 0; d < rank; ++d) {
        dims[d] = cuuint64_t(extents[d]);
        if (d == 0) continue;
        bytes[d - 1] = cuuint64_t(extents[d] > 1 ? strides[d - 1] : dense) * 2;  // (one of them: the stride means nothing)
        dense *= extents[d];
    }
    return encode(map, dtype == B200Q_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, cuuint32_t(rank),
                  const_cast<void*>(base), dims, bytes, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

template <typename T, int HD>
cudaError_t launch_prefix(const CUtensorMap (&maps)[4], const PrefixArgs& a, int blocks, cudaStream_t stream) {
    constexpr size_t kSmem = Shape<HD>::kBytes + 1024;
    cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(prefix_attention_kernel<T, HD>), kSmem);
    if (err != cudaSuccess) return err;
    err = launch_overlapped(prefix_attention_kernel<T, HD>, dim3(unsigned(blocks)), dim3(kThreads), kSmem, stream, maps[0],
                            maps[1], maps[2], maps[3], a);
    if (err != cudaSuccess) return err;
    const dim3 grid{unsigned((a.batch * a.rep + 31) / 32), unsigned(a.nkv), unsigned(HD / (4 * kJoinWarps * kJoinColumns))};
    return launch_overlapped(prefix_join_kernel<T, HD>, grid, dim3(32 * kJoinWarps), 0, stream, a, blocks);
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int64_t b200q_prefix_attention_scratch_bytes(int64_t batch, int64_t nq, int64_t nkv, int64_t head_dim, int64_t prefix,
                                                        int64_t max_seq) {
    if (check_prefix(batch, nq, nkv, head_dim, prefix, max_seq) != B200Q_OK) return -1;
    return plan_of(batch, nkv, nq / nkv, head_dim, prefix, max_seq).floats * int64_t(sizeof(float));
}

extern "C" int32_t b200q_prefix_attention(const void* q, const void* prefix_k, const void* prefix_v, const void* cache_k,
                                          const void* cache_v, const int64_t* positions, const int64_t* prefix_at, void* out,
                                          void* scratch, int64_t batch, int64_t nq, int64_t nkv, int64_t head_dim, int64_t prefix,
                                          int64_t max_seq, const int64_t* strides, float scale, int32_t dtype, void* stream) {
    const int32_t checked = check_prefix(batch, nq, nkv, head_dim, prefix, max_seq);
    if (checked != B200Q_OK) return checked;
    B200Q_REQUIRE(dtype == B200Q_BF16 || dtype == B200Q_F16, "prefix_attention: bf16 or f16");
    // (masked scores are -inf before the scale, and the largest score is looked for there)
    B200Q_REQUIRE(scale > 0.0f && scale <= 3.0e38f, "prefix_attention: the scale is a positive number, not %g", double(scale));
    if (batch == 0) return B200Q_OK;
    B200Q_REQUIRE(q && positions && out && scratch && strides && (prefix == 0 || (prefix_k && prefix_v)) &&
                      (max_seq == 0 || (cache_k && cache_v)) && aligned(q, 16) && aligned(prefix_k, 16) && aligned(prefix_v, 16) &&
                      aligned(cache_k, 16) && aligned(cache_v, 16) && aligned(out, 16) && aligned(scratch, 16) &&
                      aligned(positions, 8) && aligned(prefix_at, 8),
                  "prefix_attention: tensors must be 16-byte aligned (positions and the prefix length: int64)");
    for (int i = 0; i < 12; ++i)
        B200Q_REQUIRE(strides[i] % 8 == 0 && strides[i] >= 0, "prefix_attention: strides must be whole 16-byte steps");
    EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return unavailable("prefix_attention: the driver has no cuTensorMapEncodeTiled");

    const PrefixPlan p = plan_of(batch, nkv, nq / nkv, head_dim, prefix, max_seq);
    CUtensorMap maps[4] = {};
    // strides: q (row, head), then (key, head) of the prefix's keys and values, (key, head, row) of the caches'
    for (int v = 0; v < 2; ++v) {
        const int64_t shared[3] = {head_dim, prefix, nkv}, alone[4] = {head_dim, max_seq, nkv, batch};
        CUresult made = CUDA_SUCCESS;
        if (prefix > 0) made = make_map(encode, &maps[v], v ? prefix_v : prefix_k, dtype, 3, shared, strides + 2 + 2 * v);
        if (made == CUDA_SUCCESS && max_seq > 0)
            made = make_map(encode, &maps[2 + v], v ? cache_v : cache_k, dtype, 4, alone, strides + 6 + 3 * v);
        B200Q_REQUIRE(made == CUDA_SUCCESS, "prefix_attention: cuTensorMapEncodeTiled failed (%d)", int(made));
    }
    PrefixArgs a = {};
    a.q = static_cast<const uint16_t*>(q), a.q_row = strides[0], a.q_head = strides[1];
    a.positions = positions, a.prefix_at = prefix_at, a.out = static_cast<uint16_t*>(out);
    a.scratch = static_cast<float*>(scratch), a.cum = static_cast<int*>(scratch) + p.cum_at;
    a.batch = int(batch), a.nq = int(nq), a.nkv = int(nkv), a.rep = int(nq / nkv);
    a.prefix = int(prefix), a.slots = int(max_seq);
    a.tile_rows = p.tile_rows, a.row_tiles = p.row_tiles, a.items = p.items, a.own_at = p.own_at;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.status = decoder_error_word(), a.error = gemm_error_word();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t err;
    if (dtype == B200Q_BF16)
        err = head_dim == 128 ? launch_prefix<__nv_bfloat16, 128>(maps, a, p.blocks, s) : launch_prefix<__nv_bfloat16, 64>(maps, a, p.blocks, s);
    else
        err = head_dim == 128 ? launch_prefix<__half, 128>(maps, a, p.blocks, s) : launch_prefix<__half, 64>(maps, a, p.blocks, s);
    return launch_status("prefix_attention", err);
}
