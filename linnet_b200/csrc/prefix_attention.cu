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
constexpr int kPart = 64;                  // keys of one turn of scores, weights and sums: half a tile
constexpr int kRows = 128;                 // of a group's products
constexpr int kProducerWarp = 8, kIssuerWarp = 9, kQueryWarp = 11;  // 9 and 10: an issuer for each group
constexpr int kThreads = 12 * 32;
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

__device__ __forceinline__ int own_keys(const PrefixArgs& a, int64_t position) {
    return position < -1 || position >= a.slots ? 0 : int(position) + 1;  // outside the cache: none
}
__device__ __forceinline__ int own_tiles(const PrefixArgs& a, int64_t position) {
    return (own_keys(a, position) + kKeys - 1) / kKeys;
}
__device__ __forceinline__ int prefix_length(const PrefixArgs& a) {
    if (a.prefix_at == nullptr) return a.prefix;
    const int64_t given = ld_mutable(a.prefix_at);
    return int(given < 0 ? 0 : given > a.prefix ? a.prefix : given);
}
// The first tile of block c, and the block that takes tile t, of `total` over `blocks`: no more of
// them than tiles, so that none between two has nothing.  (total * c / blocks in 32 bits; its inverse
// from an estimate that is a block off at most.)
__device__ __forceinline__ int first_tile(int c, int total, int blocks) {
    if (total <= blocks) return min(c, total);
    const int whole = total / blocks;
    return whole * c + (total - whole * blocks) * c / blocks;
}
__device__ __forceinline__ int block_of(int t, int total, int blocks) {
    if (total <= blocks) return t;
    int c = min(int(float(t) * (float(blocks) / float(total))), blocks - 1);
    while (first_tile(c, total, blocks) > t) --c;
    while (first_tile(c + 1, total, blocks) <= t) ++c;
    return c;
}

struct Share {  // of a block; in shared memory
    int total, first, last;              // tiles
    int prefix_keys, prefix_tiles, own_first;
    int own_row, own_row_tile;           // the batch row that holds the first own tile of the share, and its first tile
};

// A piece, as the scheduling warp writes it down for the other roles.
enum Who : unsigned char { kGroup0, kGroup1, kAlternate, kBoth };  // whose the tiles are: one group's, each group's in turn, all both's
struct __align__(16) Piece {
    int place;                // item + block: of the scratch memory
    int head, row;            // KV head, first batch row
    int key, keys, tiles;     // first key, keys to the end of the item, tiles (0: the share is at its end)
    int before;               // tiles of the share before it
    short rows;               // batch rows
    unsigned char who;
    bool prefix;
    // of a group: its first tile of the piece, and how far on the next one is
    __device__ __forceinline__ int first(int g) const { return who == kAlternate ? g : who == kBoth || who == g ? 0 : tiles; }
    __device__ __forceinline__ int step() const { return who == kAlternate ? 2 : 1; }
    __device__ __forceinline__ int queries() const { return who == kBoth ? 2 : 1; }  // buffers
};
constexpr int kBatch = 16;    // pieces that are written down at a time; there are two such batches

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
__device__ __forceinline__ float exp2_approx(float x) {  // relative error 2^-22
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
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
__device__ __forceinline__ void tmem_take_8(uint32_t (&v)[8], uint32_t taddr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_put_8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map)); }

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {  // does not suspend the thread
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

struct Barriers {
    uint64_t full[10], empty[10];          // tiles of K and V
    uint64_t query_full[2], query_empty[2];
    uint64_t scores[2][2], weights[2][2];  // of the groups' halves of a tile: S is there, P is there
    uint64_t summed[2], result[2];         // of the groups: P . V of a half is done; O of a piece is complete
    uint64_t list_full[2], list_empty[2];  // batches of pieces
    Piece list[2 * kBatch];
    Share share;
    uint32_t tmem_base;
    int warp_tiles[kThreads / 32];
};
constexpr int kListReaders = 3 + 8;        // producer, issuers, warps of the groups

// One role's way through the pieces.  Every batch is waited for and handed back.
struct Pieces {
    Barriers* bars;
    uint32_t i;               // pieces read
    __device__ __forceinline__ explicit Pieces(Barriers* b) : bars(b), i(0) {}
    // One thread's: the next piece; one without tiles at the end (or when a wait has expired).
    __device__ __forceinline__ Piece next(bool* ok, int* error) {
        const uint32_t batch = i / kBatch;
        if (i % kBatch == 0) {
            if (batch > 0) mbar_arrive(&bars->list_empty[(batch - 1) & 1]);
            *ok = *ok && mbar_wait(&bars->list_full[batch & 1], (batch >> 1) & 1, error, 51);
        }
        Piece p = bars->list[i % (2 * kBatch)];
        if (!*ok) p.tiles = 0;
        ++i;
        return p;
    }
    // A whole warp's.
    __device__ __forceinline__ Piece next_of_warp(bool* ok, int* error) {
        const uint32_t batch = i / kBatch;
        if (i % kBatch == 0) {
            __syncwarp();
            if (batch > 0 && threadIdx.x % 32 == 0) mbar_arrive(&bars->list_empty[(batch - 1) & 1]);
            *ok = *ok && __all_sync(0xFFFFFFFFu, mbar_wait(&bars->list_full[batch & 1], (batch >> 1) & 1, error, 51));
        }
        Piece p = bars->list[i % (2 * kBatch)];
        if (!*ok) p.tiles = 0;
        ++i;
        return p;
    }
};

// A group's tiles, one after the other through the pieces.
struct Tasks {
    Pieces pieces;
    Piece p;
    int g, tile;
    uint32_t query;           // query buffers filled before the piece
    // `leave` is called for every piece that is left behind, the group's or not, with the buffers filled up to its end.
    template <typename Leave>
    __device__ __forceinline__ Tasks(Barriers* bars, int group, bool* ok, int* error, Leave leave) : pieces(bars) {
        g = group, query = 0;
        p = pieces.next(ok, error);
        tile = p.first(g);
        settle(ok, error, leave);
    }
    __device__ __forceinline__ bool valid() const { return p.tiles > 0; }
    template <typename Leave>
    __device__ __forceinline__ void settle(bool* ok, int* error, Leave leave) {
        while (p.tiles > 0 && tile >= p.tiles) {
            query += p.queries();
            leave(p, query);
            p = pieces.next(ok, error);
            tile = p.first(g);
        }
    }
    template <typename Leave>
    __device__ __forceinline__ void advance(bool* ok, int* error, Leave leave) {
        tile += p.step();
        settle(ok, error, leave);
    }
    __device__ __forceinline__ bool starts() const { return tile == p.first(g); }
    __device__ __forceinline__ bool ends() const { return tile + p.step() >= p.tiles; }
};
// K and V of a tile are these loads of the share, in the order in which each group's products want them;
// where the groups alternate, K of the tile after next comes before V of the next one.
__device__ __forceinline__ uint32_t load_of_k(const Piece& p, int tile) {
    return uint32_t(2 * (p.before + tile) - (p.who == kAlternate && tile > 0 ? 1 : 0));
}
__device__ __forceinline__ uint32_t load_of_v(const Piece& p, int tile) {
    return uint32_t(2 * (p.before + tile) + (p.who == kAlternate && tile < p.tiles - 1 ? 2 : 1));
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
prefix_attention_kernel(const __grid_constant__ CUtensorMap prefix_k, const __grid_constant__ CUtensorMap prefix_v,
                        const __grid_constant__ CUtensorMap cache_k, const __grid_constant__ CUtensorMap cache_v,
                        const __grid_constant__ CUtensorMap prefix_q, const __grid_constant__ CUtensorMap own_q,
                        const __grid_constant__ PrefixArgs a) {
    using H = Half16<T>;
    using S = Shape<HD>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* slots = smem + 2 * S::kQuery;
    Barriers& bars = *reinterpret_cast<Barriers*>(smem + S::kBytes);
    Share& share = bars.share;
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) / 32, 0), lane = threadIdx.x % 32;

    if (threadIdx.x == kProducerWarp * 32) {
        if (a.prefix > 0) prefetch_map(&prefix_k), prefetch_map(&prefix_v), prefetch_map(&prefix_q);
        if (a.slots > 0) prefetch_map(&cache_k), prefetch_map(&cache_v), prefetch_map(&own_q);
    }
    if (threadIdx.x == 0) {
        // (empty: the two issuers)
        for (int s = 0; s < S::kSlots; ++s) mbar_init(&bars.full[s], 1), mbar_init(&bars.empty[s], 2);
        for (int g = 0; g < 2; ++g) {
            mbar_init(&bars.query_full[g], 1), mbar_init(&bars.query_empty[g], 2);
            for (int h = 0; h < 2; ++h) mbar_init(&bars.scores[g][h], 1), mbar_init(&bars.weights[g][h], 4);
            mbar_init(&bars.summed[g], 1), mbar_init(&bars.result[g], 1);
            mbar_init(&bars.list_full[g], 1), mbar_init(&bars.list_empty[g], kListReaders);
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
        const int keys = prefix_length(a), tiles = (keys + kKeys - 1) / kKeys;
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
        if (lane == 31) bars.warp_tiles[warp] = before;
        before -= mine;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += bars.warp_tiles[w];
            all += bars.warp_tiles[w];
        }
        if (a.prefix_at != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
            const int64_t given = ld_mutable(a.prefix_at);
            if (given < 0 || given > a.prefix) record_bad_position(a.status, 0);
        }
        const int own_first = a.items * tiles, total = own_first + all * a.nkv;
        const int first = first_tile(blockIdx.x, total, gridDim.x), last = first_tile(blockIdx.x + 1, total, gridDim.x);
        const int look = max(first, own_first);  // the first own tile this block can have
        if (threadIdx.x == 0) {
            share.total = total, share.first = first, share.last = last;
            share.prefix_keys = keys, share.prefix_tiles = tiles, share.own_first = own_first;
        }
        const int begin = own_first + before * a.nkv, end = begin + mine * a.nkv;
        if (look >= begin && look < end) {
            int row = from, at = begin;
            for (; per > 1; ++row) {  // (one row a thread: it is this one)
                const int each = own_tiles(a, ld_mutable(a.positions + row));
                if (look < at + each * a.nkv) break;
                at += each * a.nkv;
            }
            share.own_row = row, share.own_row_tile = at;
        }
        if (blockIdx.x == 0) {  // for the joining kernel
            int c = before;
            for (int b = from; b < to; ++b) {
                a.cum[b] = c;
                if (b + 1 < to) c += own_tiles(a, ld_mutable(a.positions + b));
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
    bool ok = true;

    if (warp == kProducerWarp) {
        if (lane == 0) {
            Pieces pieces(&bars);
            uint32_t n = 0, slot = 0, lap = 0;
            auto load = [&](const Piece& p, int tile, const CUtensorMap* shared, const CUtensorMap* own) {
                ok = ok && (lap == 0 || mbar_wait(&bars.empty[slot], (lap - 1) & 1, a.error, 41));
                if (!ok) return;
                mbar_expect_tx(&bars.full[slot], S::kSlot);
#pragma unroll
                for (int c = 0; c < S::kHalves; ++c) {
                    const uint32_t dst = smem_u32(slots) + slot * S::kSlot + c * S::kHalf;
                    const int key = p.key + tile * kKeys;
                    if (p.prefix) tma_load_3d(dst, shared, c * 64, key, p.head, &bars.full[slot]);
                    else tma_load_4d(dst, own, c * 64, key, p.head, p.row, &bars.full[slot]);
                }
                ++n;
                if (++slot == S::kSlots) slot = 0, ++lap;
            };
            for (;;) {
                const Piece p = pieces.next(&ok, a.error);
                if (p.tiles == 0) break;
                load(p, 0, &prefix_k, &cache_k);
                for (int tile = 0; tile < p.tiles && ok; ++tile) {
                    const bool ahead = p.who == kAlternate && tile + 1 < p.tiles;
                    if (ahead) load(p, tile + 1, &prefix_k, &cache_k);
                    load(p, tile, &prefix_v, &cache_v);
                    if (!ahead && tile + 1 < p.tiles) load(p, tile + 1, &prefix_k, &cache_k);
                }
            }
            if (!ok)  // what is in flight lands before the block leaves
                for (uint32_t i = n > S::kSlots ? n - S::kSlots : 0; i < n; ++i) mbar_wait(&bars.full[i % S::kSlots], (i / S::kSlots) & 1, a.error, 42);
        }
        __syncwarp();
    } else if (warp == kIssuerWarp || warp == kIssuerWarp + 1) {
        // ---- the products of group g, from one thread ----
        if (elect_one()) {
            constexpr uint32_t kType = H::kDtype == B200Q_BF16 ? 1u : 0u;
            constexpr uint32_t kScores = (1u << 4) | (kType << 7) | (kType << 10) | (uint32_t(kPart >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
            constexpr uint32_t kValues = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | (uint32_t(HD >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
            const int g = warp - kIssuerWarp;
            const uint32_t s_at = tmem + uint32_t(g) * kKeys, o_at = tmem + 2 * kKeys + uint32_t(g) * HD;
            // Both issuers see every load and every buffer of queries, piece by piece in order, and hand it back: a
            // waiter that left one out could not tell a barrier's phase from the one after next.
            uint32_t loads = 0, queries = 0;  // those handed back
            auto take_load = [&](uint32_t load) {  // waits for it, hands back those before it; its slot
                for (; ok && loads < load; ++loads) {
                    ok = mbar_wait(&bars.full[loads % S::kSlots], (loads / S::kSlots) & 1, a.error, 44);
                    if (ok) mbar_arrive(&bars.empty[loads % S::kSlots]);
                }
                const uint32_t slot = load % S::kSlots;
                ok = ok && mbar_wait(&bars.full[slot], (load / S::kSlots) & 1, a.error, 44);
                loads = load + 1;
                return slot;
            };
            auto pass_queries = [&](uint32_t before) {
                for (; ok && queries < before; ++queries) {
                    ok = mbar_wait(&bars.query_full[queries & 1], (queries >> 1) & 1, a.error, 43);
                    if (ok) mbar_arrive(&bars.query_empty[queries & 1]);
                }
            };
            auto pass_piece = [&](const Piece& p, uint32_t filled) {
                pass_queries(filled);
                const uint32_t end = uint32_t(2 * (p.before + p.tiles));
                if (ok && loads < end) mbar_arrive(&bars.empty[take_load(end - 1)]);
            };
            Tasks task(&bars, g, &ok, a.error, pass_piece);
            const Piece& p = task.p;
            int ahead = 0;            // the tile whose scores are issued next; one ahead of the tile that is summed
            uint32_t k_slot = 0, k_query = 0;
            auto issue_scores = [&](int h) {  // of half h; after its last half, on to the next tile
                if (h == 0) k_slot = take_load(load_of_k(p, ahead));
                if (!ok) return;
                tc_fence_after();
                const uint64_t qd = smem_desc(smem_u32(smem) + k_query * S::kQuery);
                const uint64_t kd = smem_desc(smem_u32(slots) + k_slot * S::kSlot + uint32_t(h) * (kPart * 128));
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const uint32_t step = uint32_t(k / 4) * (S::kHalf >> 4) + uint32_t(k % 4) * 2;
                    umma_f16_ss(s_at + uint32_t(h) * kPart, qd + step, kd + step, kScores, k > 0);
                }
                umma_commit(&bars.scores[g][h]);
                if (h == 0 && p.keys - ahead * kKeys > kPart) return;
                umma_commit(&bars.empty[k_slot]);
                ahead += p.step();
                if (ahead >= p.tiles) umma_commit(&bars.query_empty[k_query]);
            };
            auto issue_rest = [&](int h) {  // of the next tile, from half h on
                for (const int tile = ahead; ok && ahead == tile; ++h) issue_scores(h);
            };
            uint32_t given[2] = {0, 0};
            while (ok && task.valid()) {
                const bool begun = !task.starts();
                if (!begun) {
                    const uint32_t query = task.query + (p.who == kBoth ? uint32_t(g) : 0u);
                    k_query = query & 1;
                    pass_queries(query);
                    ok = ok && mbar_wait(&bars.query_full[k_query], (query >> 1) & 1, a.error, 43);
                    queries = query + 1;
                    ahead = task.tile;
                    issue_rest(0);
                }
                const int valid = p.keys - task.tile * kKeys;
                const uint32_t slot = take_load(load_of_v(p, task.tile));
                const uint64_t vd = value_desc(smem_u32(slots) + slot * S::kSlot, S::kHalf);
                const int next = task.tile + p.step();
                int issued = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h * kPart >= valid) break;
                    ok = ok && mbar_wait(&bars.weights[g][h], given[h]++ & 1, a.error, 45);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 4 * h; k < 4 * h + 4; ++k)
                        if (k == 0 || k * 16 < valid)
                            umma_f16_ts(o_at, s_at + h * kPart + (k - 4 * h) * 8, vd + uint32_t(k) * (2048 >> 4), kValues, k > 0 || begun);
                    umma_commit(&bars.summed[g]);
                    // the next tile's first half, unless it would have to be waited for
                    if (h == 0 && next < p.tiles) {
                        const uint32_t load = load_of_k(p, next);
                        if (loads == load && mbar_test(&bars.full[load % S::kSlots], (load / S::kSlots) & 1)) issue_scores(0), issued = 1;
                    }
                }
                if (!ok) break;
                umma_commit(&bars.empty[slot]);
                if (task.ends()) umma_commit(&bars.result[g]);
                if (ahead == next && next < p.tiles) issue_rest(issued);
                task.advance(&ok, a.error, pass_piece);
            }
        }
        __syncwarp();
    } else if (warp == kQueryWarp) {
        // ---- the pieces, a batch at a time, and their queries ----
        int t = share.first, row = share.own_row, at = share.own_row_tile;
        int keys_of = 0, held = -1;            // own keys of rows 32 * held + lane
        const int prefix_end = min(share.own_first, share.last);
        uint32_t query = 0;
        for (uint32_t batch = 0; ok; ++batch) {
            if (batch >= 2) ok = wait(&bars.list_empty[batch & 1], ((batch >> 1) - 1) & 1, 52);
            if (!ok) break;
            Piece* list = bars.list + (batch & 1) * kBatch;
            int n = 0;
            bool over = false;
            while (n < kBatch && !over) {
                Piece p;
                int begin, end;                // tiles of this lane's piece
                if (t < prefix_end) {          // an item a lane
                    const int item = t / share.prefix_tiles + lane, head = item / a.row_tiles, tile = item - head * a.row_tiles;
                    const int first = item * share.prefix_tiles;
                    begin = max(t, first), end = min(first + share.prefix_tiles, prefix_end);
                    p.head = head, p.row = tile * 2 * a.tile_rows;
                    p.rows = short(min(2 * a.tile_rows, a.batch - p.row));
                    p.who = p.rows > a.tile_rows ? kBoth : kAlternate, p.prefix = true;
                    p.key = (begin - first) * kKeys, p.keys = share.prefix_keys - p.key;
                    p.place = item + int(blockIdx.x);
                } else if (t < share.last) {   // a head of the row a lane
                    int keys, each;
                    for (;; ++row) {           // (t is before the end of the sequence: some row has it)
                        if (row / 32 != held) {
                            held = row / 32;
                            const int r = held * 32 + lane;
                            keys_of = r < a.batch ? own_keys(a, ld_mutable(a.positions + r)) : 0;
                        }
                        keys = __shfl_sync(0xFFFFFFFFu, keys_of, row % 32);
                        each = (keys + kKeys - 1) / kKeys;
                        if (t < at + each * a.nkv) break;
                        at += each * a.nkv;
                    }
                    const int head = (t - at) / each + lane, first = at + head * each;
                    begin = max(t, first), end = head < a.nkv ? min(first + each, share.last) : begin;
                    // (one group's: the other is done with the piece before meanwhile, or begins the next)
                    p.head = head, p.row = row, p.rows = 1, p.who = (n + lane) & 1 ? kGroup1 : kGroup0, p.prefix = false;
                    p.key = (begin - first) * kKeys, p.keys = keys - p.key;
                    p.place = row * a.nkv + head + int(blockIdx.x);
                } else {
                    over = true;
                    begin = end = t;
                    if (lane == 0) list[n].tiles = 0;
                }
                const bool there = begin < end && n + lane < kBatch;
                const int count = __popc(__ballot_sync(0xFFFFFFFFu, there));
                if (there) {
                    p.tiles = end - begin, p.before = begin - share.first;
                    list[n + lane] = p;
                }
                if (count > 0) t = __shfl_sync(0xFFFFFFFFu, end, count - 1);
                n += count;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.list_full[batch & 1]);
            for (int i = 0; i < n && ok; ++i) {
                const Piece& p = list[i];
                for (int half = 0; half < p.queries(); ++half, ++query) {
                    const uint32_t buffer = query & 1;
                    ok = query < 2 || wait(&bars.query_empty[buffer], ((query >> 1) - 1) & 1, 47);
                    if (!ok) break;
                    if (lane == 0) {
                        // (batch rows past the last one read as zeros; rows of the buffer past the box are never looked at)
                        mbar_expect_tx(&bars.query_full[buffer], uint32_t(S::kHalves * 128 * a.rep * (p.prefix ? a.tile_rows : 1)));
#pragma unroll
                        for (int h = 0; h < S::kHalves; ++h)
                            tma_load_4d(smem_u32(smem) + buffer * S::kQuery + h * (kRows * 128), p.prefix ? &prefix_q : &own_q, h * 64, 0,
                                        p.head, p.row + half * a.tile_rows, &bars.query_full[buffer]);
                    }
                    __syncwarp();
                }
            }
            if (over) break;
        }
        if (!ok && lane == 0)
            for (uint32_t i = query > 2 ? query - 2 : 0; i < query; ++i) mbar_wait(&bars.query_full[i & 1], (i >> 1) & 1, a.error, 42);
        __syncwarp();
    } else if (warp < kProducerWarp) {
        // ---- softmax: group g, one query row a thread ----
        const int g = warp / 4, row = threadIdx.x % 128;
        const uint32_t lanes = tmem + (uint32_t(warp & 3) << 21);
        const uint32_t s_at = lanes + uint32_t(g) * kKeys, o_at = lanes + 2 * kKeys + uint32_t(g) * HD;
        Pieces list(&bars);
        uint32_t pieces = 0;                      // that this group has had
        uint32_t had = 0, had_first = 0;          // halves of tiles that this group has had, and first halves
        const float2 scale = make_float2(a.scale_log2, a.scale_log2);
        for (;;) {
            const Piece p = list.next_of_warp(&ok, a.error);
            if (p.tiles == 0) break;
            const int first = p.first(g), step = p.step();
            if (p.who <= kGroup1 && p.who != g) continue;
            const int live = p.who == kBoth ? min(a.tile_rows, p.rows - g * a.tile_rows) * a.rep : p.rows * a.rep;
            const bool any = (warp & 3) * 32 < live;  // of this warp's rows
            float m = 0.0f, l = 0.0f;
            for (int tile = first; tile < p.tiles && ok; tile += step) {
                const int valid = p.keys - tile * kKeys;  // keys of the tile, and more
#pragma unroll 1
                for (int h = 0; h * kPart < min(valid, kKeys); ++h) {
                    const int keys = valid - h * kPart;   // of this half, and more
                    const uint32_t at = s_at + uint32_t(h) * kPart;
                    const uint32_t turn = h == 0 ? had_first++ : had - had_first;
                    ok = wait(&bars.scores[g][h], turn & 1, 48);
                    if (!ok) break;
                    ++had;
                    tc_fence_after();
                    if (any) {
                        // Few warps run here, so every step is written as independent instructions in a row.
                        uint32_t v[kPart];
                        tmem_ask_32(v, at), tmem_ask_32(v + 32, at + 32);
                        tmem_arrived(v), tmem_arrived(v + 32);
                        if (keys < kPart) {
#pragma unroll
                            for (int i = 0; i < kPart; ++i) v[i] = i < keys ? v[i] : 0xFF800000u;
                        }
                        float most[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) most[i] = __uint_as_float(v[i]);
#pragma unroll
                        for (int i = 8; i < kPart - 8; i += 16)
#pragma unroll
                            for (int k = 0; k < 8; ++k) most[k] = max3(most[k], __uint_as_float(v[i + k]), __uint_as_float(v[i + 8 + k]));
#pragma unroll
                        for (int k = 0; k < 8; ++k) most[k] = fmaxf(most[k], __uint_as_float(v[kPart - 8 + k]));
                        const float here = a.scale_log2 * fmaxf(max3(max3(most[0], most[1], most[2]), most[3], most[4]),
                                                                max3(most[5], most[6], most[7]));
                        if (tile == first && h == 0) {
                            m = here == -INFINITY ? 0.0f : here;
                        } else if (__any_sync(0xFFFFFFFFu, row < live && here > m + kStale)) {
                            const float next = here > m + kStale ? here : m, by = exp2_approx(m - next);
                            m = next;
                            l *= by;
                            // (these scores were asked for behind the sums before the last ones)
                            ok = wait(&bars.summed[g], (had - 2) & 1, 53);
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < HD; c += 8) {
                                uint32_t o[8];
                                tmem_take_8(o, o_at + c);
#pragma unroll
                                for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
                                tmem_put_8(o_at + c, o);
                            }
                        }
                        const float2 minus = make_float2(-m, -m);
                        // Scaled scores run kAhead pairs ahead of the exponentials and the sums as far behind, so that
                        // the exponential unit, which takes eight clocks an instruction, always has one to do.
                        constexpr int kPairs = kPart / 2, kAhead = 4;
                        float2 e[kPairs], sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                        auto scaled = [&](int i) { e[i] = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), scale, minus); };
                        auto added = [&](int i) {
                            sum[i & 1] = add2(sum[i & 1], e[i]);
                            v[i] = H::pack(e[i].x, e[i].y);
                        };
#pragma unroll
                        for (int i = 0; i < kAhead; ++i) scaled(i);
#pragma unroll
                        for (int i = 0; i < kPairs; ++i) {
                            if (i + kAhead < kPairs) scaled(i + kAhead);
                            e[i] = make_float2(exp2_approx(e[i].x), exp2_approx(e[i].y));
                            if (i >= kAhead) added(i - kAhead);
                        }
#pragma unroll
                        for (int i = kPairs - kAhead; i < kPairs; ++i) added(i);
                        tmem_put_32(at, v);
                        const float2 pair = add2(sum[0], sum[1]);
                        l += pair.x + pair.y;
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                    if (keys < kPart) {
                        // Rows of V past the last key may hold anything, and 0 * NaN is no 0: those that the last
                        // step of 16 keys takes in are cleared (by either group where both use the tile).
                        const uint32_t load = load_of_v(p, tile), slot = load % S::kSlots;
                        ok = ok && wait(&bars.full[slot], (load / S::kSlots) & 1, 49);
                        if (!ok) break;
                        uint8_t* tail = slots + slot * S::kSlot;
                        const int rows = (16 - valid % 16) % 16;
                        for (int i = row; i < rows * 8 * S::kHalves; i += 128) {
                            const int c = S::kHalves == 1 ? 0 : (i >> 3) & 1, r = valid + (i >> 3) / S::kHalves;
                            *reinterpret_cast<uint4*>(tail + c * S::kHalf + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.weights[g][h]);
                }
            }
            if (!ok) break;
            // ---- the piece's result ----
            const int span = p.prefix ? kRows : a.rep;  // rows of a group in the scratch memory
            float* to = a.scratch + (p.prefix ? 0 : a.own_at) + (p.prefix ? 2 * int64_t(p.place) + g : int64_t(p.place)) * group_floats(span, HD);
            const bool worked = first < p.tiles;
            if (worked) {
                ok = wait(&bars.result[g], pieces & 1, 50);
                if (!ok) break;
                ++pieces;
                tc_fence_after();
                if (any) {
                    uint4* column = reinterpret_cast<uint4*>(to) + row;
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tmem_ask_32(o, o_at + c);
                        tmem_arrived(o);
                        if (row < live) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4, column += span) *column = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        }
                    }
                }
            }
            if (row < live) {
                to[int64_t(HD) * span + row] = worked ? m : -INFINITY;
                to[int64_t(HD + 1) * span + row] = l;
            }
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
// out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i in f32 over a row's parts (a piece has one, or
// one of each group); a row without any key is 0.  One query row a lane.  What the kernel waits for is
// the way to the L2 cache, so a thread has several parts in flight.  Few parts a row: a block has all
// columns of its rows, four columns of four numbers a warp.  Many (a long prefix for few rows and heads):
// the parts are dealt among the warps too, and their sums meet in shared memory.
constexpr int kJoinWarps = 8, kJoinHeld = 4;
constexpr int kManyParts = 12;  // more than this many parts of a row are dealt among the warps

template <typename T, int HD, bool MANY>
__global__ void __launch_bounds__(32 * kJoinWarps)
prefix_join_kernel(const __grid_constant__ PrefixArgs a, int blocks) {
    using H = Half16<T>;
    constexpr int kSlices = MANY ? kJoinWarps : 1;     // warps that share a row's parts
    constexpr int kColumns = MANY ? 2 : HD / 4 / kJoinWarps, kSums = 4 * kColumns;
    __shared__ float sums[MANY ? kJoinWarps : 1][kSums + 2][32];  // O, m and l
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int head = blockIdx.y, row = blockIdx.x * 32 + lane;  // row: batch row * rep + head of the group
    const int slice = MANY ? warp : 0, column = (MANY ? int(blockIdx.z) : warp) * kColumns;
    const bool live = row < a.batch * a.rep;
    const int b = live ? row / a.rep : 0, r = row - b * a.rep;
    auto word = [&](int i) { return int(ld_mutable(reinterpret_cast<const uint32_t*>(a.cum) + i)); };
    const int total = word(a.batch), prefix_tiles = word(a.batch + 1), before = word(b);
    const int each = own_tiles(a, ld_mutable(a.positions + b));

    struct Item {              // the prefix, and the row's own keys
        const float* base;     // of the first group that has the row, in the first piece
        int parts, skip;       // groups that have the row: over all pieces; and the floats from one to the next
        int span, at;          // rows of a group in the scratch memory, and which one this is
    } shared = {}, own = {};
    if (live && prefix_tiles > 0) {
        const int pair = b / (2 * a.tile_rows), within = b - pair * 2 * a.tile_rows;
        const bool both = min(2 * a.tile_rows, a.batch - pair * 2 * a.tile_rows) > a.tile_rows;
        const int item = head * a.row_tiles + pair, first = item * prefix_tiles;
        const int from = block_of(first, total, blocks), to = block_of(first + prefix_tiles - 1, total, blocks);
        const int g = both && within >= a.tile_rows, groups = both ? 1 : 2;
        shared.base = a.scratch + (2 * int64_t(item + from) + g) * group_floats(kRows, HD);
        shared.parts = (to - from + 1) * groups, shared.skip = int(group_floats(kRows, HD)) * (2 / groups);
        shared.span = kRows, shared.at = (within - g * a.tile_rows) * a.rep + r;
    }
    if (live && each > 0) {
        const int first = a.items * prefix_tiles + before * a.nkv + head * each;
        const int from = block_of(first, total, blocks), to = block_of(first + each - 1, total, blocks);
        own.base = a.scratch + a.own_at + int64_t(b * a.nkv + head + from) * group_floats(a.rep, HD);
        own.parts = to - from + 1, own.skip = int(group_floats(a.rep, HD));
        own.span = a.rep, own.at = r;
    }
    const int parts = shared.parts + own.parts;
    float m = -INFINITY, l = 0.0f, o[kSums] = {};
    for (int k0 = slice; k0 < parts; k0 += kSlices * kJoinHeld) {
        float ms[kJoinHeld], ls[kJoinHeld];
        uint4 os[kJoinHeld][kColumns];
#pragma unroll
        for (int u = 0; u < kJoinHeld; ++u) {
            const int k = k0 + u * kSlices;
            ms[u] = -INFINITY;
            if (k >= parts) continue;
            const Item& it = k < shared.parts ? shared : own;
            const float* from = it.base + int64_t(k < shared.parts ? k : k - shared.parts) * it.skip;
            ms[u] = ld_mutable(from + HD * it.span + it.at);
            ls[u] = ld_mutable(from + (HD + 1) * it.span + it.at);
#pragma unroll
            for (int c = 0; c < kColumns; ++c) os[u][c] = ld_mutable(reinterpret_cast<const uint4*>(from) + (column + c) * it.span + it.at);
        }
        float most = m;
#pragma unroll
        for (int u = 0; u < kJoinHeld; ++u) most = fmaxf(most, ms[u]);
        if (most == -INFINITY) continue;
        const float by = exp2_approx(m - most);
        m = most, l *= by;
#pragma unroll
        for (int i = 0; i < kSums; ++i) o[i] *= by;
#pragma unroll
        for (int u = 0; u < kJoinHeld; ++u) {
            if (ms[u] == -INFINITY) continue;  // a group that had no tile of the piece: the rest of it was not stored
            const float weight = exp2_approx(ms[u] - m);
            l += weight * ls[u];
#pragma unroll
            for (int c = 0; c < kColumns; ++c) {
                o[4 * c] += weight * __uint_as_float(os[u][c].x), o[4 * c + 1] += weight * __uint_as_float(os[u][c].y);
                o[4 * c + 2] += weight * __uint_as_float(os[u][c].z), o[4 * c + 3] += weight * __uint_as_float(os[u][c].w);
            }
        }
    }
    if (MANY) {
#pragma unroll
        for (int i = 0; i < kSums; ++i) sums[slice][i][lane] = o[i];
        sums[slice][kSums][lane] = m, sums[slice][kSums + 1][lane] = l;
        __syncthreads();
        if (warp != 0) return;
#pragma unroll
        for (int w = 1; w < kSlices; ++w) m = fmaxf(m, sums[w][kSums][lane]);
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < kSums; ++i) o[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < kSlices; ++w) {
            const float theirs = sums[w][kSums][lane], weight = theirs == -INFINITY ? 0.0f : exp2_approx(theirs - m);
            l += weight * sums[w][kSums + 1][lane];
#pragma unroll
            for (int i = 0; i < kSums; ++i) o[i] += weight * sums[w][i][lane];
        }
    }
    if (!live) return;
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    uint4* to = reinterpret_cast<uint4*>(a.out + (int64_t(b) * a.nq + head * a.rep + r) * HD + column * 4);
#pragma unroll
    for (int i = 0; i < kSums; i += 8)
        *to++ = make_uint4(H::pack(o[i] * by, o[i + 1] * by), H::pack(o[i + 2] * by, o[i + 3] * by),
                           H::pack(o[i + 4] * by, o[i + 5] * by), H::pack(o[i + 6] * by, o[i + 7] * by));
}

// ---- host -----------------------------------------------------------------------------------------

struct PrefixPlan {
    int tile_rows, row_tiles, items, blocks;
    bool many;                             // parts of a row
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
    // Parts of a row, were all rows' caches full: blocks an item's tiles are spread over, and a block at either end.
    const int64_t share = tiles < 1 ? 1 : (tiles + p.blocks - 1) / p.blocks, of_prefix = ((prefix + kKeys - 1) / kKeys + share - 1) / share + 1;
    const int64_t of_own = ((slots + kKeys - 1) / kKeys + share - 1) / share + 1;
    p.many = (p.items > 0 ? of_prefix * (batch > p.tile_rows ? 1 : 2) : 0) + of_own > kManyParts;
    p.own_at = (p.items > 0 ? p.items + p.blocks : 0) * 2 * group_floats(kRows, int(hd));
    p.cum_at = p.own_at + (batch * nkv + p.blocks) * group_floats(int(rep), int(hd));
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

// A map of boxes of 64 numbers x `rows` x 1 x `last` (keys and values: 128 keys); strides in numbers.
CUresult make_map(EncodeTiled encode, CUtensorMap* map, const void* base, int32_t dtype, int rank, const int64_t* extents,
                  const int64_t* strides, int rows, int last) {
    cuuint64_t dims[4], bytes[3];
    cuuint32_t box[4] = {64, cuuint32_t(rows), 1, cuuint32_t(last)}, elem[4] = {1, 1, 1, 1};
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
cudaError_t launch_prefix(const CUtensorMap (&maps)[6], const PrefixArgs& a, int blocks, bool many, cudaStream_t stream) {
    constexpr size_t kSmem = Shape<HD>::kBytes + sizeof(Barriers) + 1024;
    static_assert(kSmem <= 227 * 1024, "shared memory of a block");
    cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(prefix_attention_kernel<T, HD>), kSmem);
    if (err != cudaSuccess) return err;
    err = launch_overlapped(prefix_attention_kernel<T, HD>, dim3(unsigned(blocks)), dim3(kThreads), kSmem, stream, maps[0],
                            maps[1], maps[2], maps[3], maps[4], maps[5], a);
    if (err != cudaSuccess) return err;
    const dim3 grid{unsigned((a.batch * a.rep + 31) / 32), unsigned(a.nkv), unsigned(many ? HD / 8 : 1)};
    return many ? launch_overlapped(prefix_join_kernel<T, HD, true>, grid, dim3(32 * kJoinWarps), 0, stream, a, blocks)
                : launch_overlapped(prefix_join_kernel<T, HD, false>, grid, dim3(32 * kJoinWarps), 0, stream, a, blocks);
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
    CUtensorMap maps[6] = {};
    // strides: q (row, head), then (key, head) of the prefix's keys and values, (key, head, row) of the caches'
    for (int v = 0; v < 2; ++v) {
        const int64_t shared[3] = {head_dim, prefix, nkv}, alone[4] = {head_dim, max_seq, nkv, batch};
        CUresult made = CUDA_SUCCESS;
        if (prefix > 0) made = make_map(encode, &maps[v], v ? prefix_v : prefix_k, dtype, 3, shared, strides + 2 + 2 * v, kKeys, 1);
        if (made == CUDA_SUCCESS && max_seq > 0)
            made = make_map(encode, &maps[2 + v], v ? cache_v : cache_k, dtype, 4, alone, strides + 6 + 3 * v, kKeys, 1);
        // queries of a KV head: of as many batch rows as a group takes, and of one
        const int64_t rep = nq / nkv, queries[4] = {head_dim, rep, nkv, batch}, steps[3] = {strides[1], rep * strides[1], strides[0]};
        if (made == CUDA_SUCCESS && (v ? max_seq : prefix) > 0)
            made = make_map(encode, &maps[4 + v], q, dtype, 4, queries, steps, int(rep), v ? 1 : p.tile_rows);
        B200Q_REQUIRE(made == CUDA_SUCCESS, "prefix_attention: cuTensorMapEncodeTiled failed (%d)", int(made));
    }
    PrefixArgs a = {};
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
        err = head_dim == 128 ? launch_prefix<__nv_bfloat16, 128>(maps, a, p.blocks, p.many, s) : launch_prefix<__nv_bfloat16, 64>(maps, a, p.blocks, p.many, s);
    else
        err = head_dim == 128 ? launch_prefix<__half, 128>(maps, a, p.blocks, p.many, s) : launch_prefix<__half, 64>(maps, a, p.blocks, p.many, s);
    return launch_status("prefix_attention", err);
}
