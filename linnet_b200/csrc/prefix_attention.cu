// Single-query attention of a batch whose rows share a long prefix (many answers to one prompt):
//     out[b, head] = sum_j softmax_j(scale * q[b, head] . k_j) v_j
// over the prefix's keys (one copy for the batch) and then the row's own, 0 .. positions[b] of its
// cache.  Row by row the prefix would be read once a row; here all rows of a KV head that share it are
// the 128 rows of a tcgen05 product, so its keys and values cross HBM once.
//
// Work is cut into tiles of 64 keys.  An ITEM is the prefix of one KV head for up to 256 query rows
// (rep = heads / kv_heads rows a batch row), or one batch row's own keys of one KV head.  The items'
// tiles stand in one sequence, prefix first, and block c of G takes the c-th G-th of it, so blocks have
// equal work whatever the lengths; where a block's share begins and ends, an item is cut into PIECES,
// each with its own softmax statistics, and a second kernel joins the pieces of a row.  (An item of own
// keys counts one tile more than it has, for its start: 256 rows of 1024 + 128 keys take 41.8 us so,
// 46.7 without, 46.8 with two; of 16384 + 128 keys 104, 152 and 103.  One of the prefix counts two more: 256 rows
// of 64 + 128 keys 38.2 us so, 50.8 with one, 84.1 without, 37.9 with three; 33 rows of 5001, 2 KV heads, 13.0,
// 13.6, 14.2 and 13.6.)  An item and a block have at most one piece in common, and
// (item + block) grows along the sequence: that is a piece's place in the scratch memory.
//
// A block has two groups, each a pipeline of its own: a TMA producer, an issuer of products and four
// warps of softmax with one query row a thread.  Per task, a tile for one group:
//   S [128 rows x 64 keys] = Q . K^T       Q and K in shared memory as TMA's 128-byte swizzle has them
//   P = 2^(scale' S - m), l += sum P       one row a thread: no exchange between threads
//   O [128 rows x D] += P . V              P in tensor memory over S's columns; V's rows are the keys, so
//                                          it is the MN-major operand as it lies in memory
// S has two buffers a group, so that the next tile's scores are there while this one's weights are made.
// A prefix item of more than 128 rows gives each group half of the rows and both every tile (each is
// loaded once); one of fewer gives the groups the same rows and a half of the keys each; own keys are one
// group's, the other is at the piece before or after.  A last warp, the lister, works out the pieces
// ahead of all roles and writes them down: with that arithmetic in every role the kernel's code was 80 KB
// and its short turns went by instruction fetches.
//
// m is a row's maximum of the first tile; a later tile whose own exceeds it by more than 2^8 moves it
// and rescales O and l in tensor memory (rare: P stays below 2^8, and the sums are f32 anyway).
// P is rounded to the tensors' type, as the product takes it; l sums P before that rounding.
//
// Registers are handed out to four warps at a time, so that 13 warps leave a thread 128: some 40 bytes of it are spilled.
//
// What bounds it, measured on a B200 (nq 32, nkv 8, D 128, bf16; join included): few rows, HBM and the
// start of the pipeline: 8 rows of 65536 keys 56 us, 4.8 TB/s; 64 rows of 8192 + up to 512 own keys
// 37 us where the bytes take 15.6; 2 rows of 100 keys 8.5 us, two launches and their latencies.  Many
// rows, the chain from scores to weights to the next scores: 256 rows of 16384 + up to 128 own keys 108 us, 640 TFLOP/s,
// and 117 in a run of a second, which the power limit takes to 1.8 GHz; of 65536 keys 313 us, 880 TFLOP/s (53 % of
// measured).  A tile of both groups takes some 2000 clocks there; its products alone take 1300, its 16384
// exponentials 1024, its 32 KB 700.
#include "mma.cuh"
#include "umma.cuh"

namespace b200q {
namespace {

using namespace umma;

constexpr int kKeys = 64;                  // of a tile
constexpr int kRows = 128;                 // of a group's products
constexpr int kProducerWarp = 8, kIssuerWarp = 10, kListWarp = 12;  // a producer and an issuer for each group
constexpr int kThreads = 13 * 32;
constexpr uint32_t kTmemColumns = 512;     // S of both groups, O of both groups
constexpr float kStale = 8.0f;             // how far (log2) a tile's maximum may exceed the row's before it moves
constexpr float kLowest = -3.0e38f;        // the maximum of scores that are all -inf (2^(-inf - m) is 0, and any other exceeds it) or NaN
constexpr int kOwnStart = 1;               // what an item of own keys costs beside its tiles, in tiles
constexpr int kPrefixStart = 2;            // and what one of the prefix does

template <int HD>
struct Shape {
    static constexpr int kHalves = HD / 64;                    // 128-byte columns of a tile
    static constexpr uint32_t kHalf = kKeys * 128;             // bytes of one
    static constexpr uint32_t kSlot = kHalves * kHalf;         // a tile of K or V
    static constexpr int kSlots = HD == 128 ? 10 : 20;
    static constexpr uint32_t kQuery = kHalves * kRows * 128;  // a group's queries; two of them
    static constexpr uint32_t kBytes = 2 * kQuery + kSlots * kSlot;
};

struct PrefixArgs {
    const int64_t* positions;
    const int64_t* prefix_at;              // its length on the device, or null: `prefix`
    uint16_t* out;
    float* scratch;
    int* cum;                              // [batch]: units of a KV head before row b; then their total, then tiles of an item's prefix
    int batch, nq, nkv, rep, prefix, slots;  // slots: of a row's own cache
    int tile_rows;                         // batch rows of a group's products: 128 / rep
    int row_tiles, items;                  // of the prefix: ceil(batch / 2 tile_rows), that times nkv
    int weight;                            // units of a tile of the prefix
    int64_t own_at;                        // where the scratch memory of own pieces begins, in floats
    float scale_log2;
    int* status;
    int* error;
};

// ---- the sequence of tiles ---------------------------------------------------------------------

__device__ __forceinline__ int own_keys(const PrefixArgs& a, int64_t position) {
    return position < -1 || position >= a.slots ? 0 : int(position) + 1;  // outside the cache: none
}
__device__ __forceinline__ int tiles_of(int keys) { return (keys + kKeys - 1) / kKeys; }
// Units of an item of the prefix.
__device__ __forceinline__ int prefix_units(const PrefixArgs& a, int tiles) { return tiles > 0 ? (tiles + kPrefixStart) * a.weight : 0; }
// Units of one head of a row.
__device__ __forceinline__ int own_units(int keys) { return keys > 0 ? tiles_of(keys) + kOwnStart : 0; }
__device__ __forceinline__ int prefix_length(const PrefixArgs& a) {
    if (a.prefix_at == nullptr) return a.prefix;
    const int64_t given = ld_mutable(a.prefix_at);
    return int(given < 0 ? 0 : given > a.prefix ? a.prefix : given);
}
// How `total` units are dealt to blocks: no more of them than half the units, so that every block between two of
// an item's has a tile of it.  The first unit of block c is total * c / blocks, in 32 bits and without a division
// a call: rest * c is less than blocks^2, so that with a half added its quotient is further from any whole number
// than f32 is off.  block_of inverts it from an estimate that is a block off at most.
struct Deal {
    int total, blocks, whole, rest;
    float inverse, share;
    __device__ __forceinline__ Deal(int units, int most) : total(units), blocks(max(1, min(units / 2, most))) {
        whole = total / blocks, rest = total - whole * blocks;
        inverse = __fdividef(1.0f, float(blocks)), share = __fdividef(float(blocks), float(total));
    }
    __device__ __forceinline__ int first(int c) const {
        return c >= blocks ? total : whole * c + int((float(rest * c) + 0.5f) * inverse);
    }
    __device__ __forceinline__ int block_of(int t) const {
        int c = min(int(float(t) * share), blocks - 1);
        while (first(c) > t) --c;
        while (first(c + 1) <= t) ++c;
        return c;
    }
};

// t / d of numbers below 2^30, by an estimate and its correction: the compiler's integer division is some hundred
// clocks of one thread, which the short turns of the roles are made of.
__device__ __forceinline__ int quotient(int t, int d) {
    const float inverse = __fdividef(1.0f, float(d));
    int q = int(float(t) * inverse);          // off by 2^-21 of it at most, and one
    q += int(float(t - q * d) * inverse);     // off by one at most
    const int left = t - q * d;
    return left < 0 ? q - 1 : left >= d ? q + 1 : q;
}

struct Share {  // of a block; in shared memory
    int first, last, own_first;          // units; of the rows' own keys
    int prefix_keys;
    int own_row, own_row_unit;           // the batch row that holds the first own unit of the share, and its first unit
};

// A piece, as the listing warp writes it down for the other roles.
enum Who : unsigned char { kGroup0, kGroup1, kBoth, kNobody, kEnd };
enum Kind : unsigned char { kRowsOfBoth, kHalves, kOwn };  // both groups its rows; its keys halved between them; own keys, one group's
struct __align__(16) Piece {
    int place;                // item + block: of the scratch memory
    int row, key, keys;       // first batch row, first key, keys to the end of the item
    int tiles;
    uint32_t base;            // loads before it in its ring: of both groups, or of its group
    unsigned short head, rows;    // KV head, batch rows
    unsigned char who, kind;
    unsigned char epoch;      // changes of kind before it
    unsigned char query;      // where its queries are, of group 0 in bits 0..2, of group 1 in bits 4..6: see Query
    __device__ __forceinline__ bool of(int g) const { return who == g || who == kBoth; }
};
// A group's two buffers of queries: which one, whether it has been filled an odd number of times before, or at all.
// Queries of up to 64 rows take half of a group's memory, so that the next piece's can be there early.
struct Query {
    uint32_t bits;
    __device__ __forceinline__ Query(const Piece& p, int g) { bits = uint32_t(p.query) >> (4 * g); }
    __device__ __forceinline__ uint32_t buffer() const { return bits & 1; }
    __device__ __forceinline__ uint32_t parity() const { return (bits >> 1) & 1; }
    __device__ __forceinline__ bool first() const { return (bits & 4) == 0; }
};
constexpr int kBatch = 8;     // pieces that are written down at a time; there are two such batches (even: pairs stay together)

// ---- scratch memory: of a piece, per group, O as [D / 4][rows] float4, then m [rows] and l [rows] ----

// (a whole number of 16-byte steps)
__host__ __device__ constexpr int64_t group_floats(int rows, int hd) { return (int64_t(rows) * (hd + 2) + 3) / 4 * 4; }

// ---- instructions --------------------------------------------------------------------------------

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
// Descriptors by halves: the address (in 16 bytes) is in the low one, all else stays.
__device__ __forceinline__ uint64_t desc_of(uint32_t low, uint32_t high) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(high));
    return d;
}
__device__ __forceinline__ void commit_at(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map)); }

__device__ __forceinline__ bool test_at(uint32_t bar, uint32_t parity) {  // does not suspend the thread
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) { return test_at(smem_u32(bar), parity); }

// The bounded wait, once in the code for all roles: with its slow path written out at every use the
// kernel was 80 KB, and its short turns went by the instruction cache.
__device__ __noinline__ bool mbar_wait_long(uint64_t* bar, uint32_t parity, int* error, int code) {
    return mbar_wait(bar, parity, error, code);
}
__device__ __forceinline__ bool mbar_watch(uint64_t* bar, uint32_t parity, int* error, int code) {
    return mbar_try_wait(bar, parity) || mbar_wait_long(bar, parity, error, code);
}

// The same by the barrier's address in shared memory.
__device__ __forceinline__ bool watch_at(uint32_t bar, uint32_t parity, int* error, int code) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kSuspendNs)
        : "memory");
    return ok != 0 || mbar_wait_long(static_cast<uint64_t*>(__cvta_shared_to_generic(bar)), parity, error, code);
}

// A way through a ring of slots: addresses of its barriers and its memory (that in 16 bytes), and where it stands.
struct Walk {
    uint32_t full, empty, memory, slots;
    uint32_t slot, parity;
    __device__ __forceinline__ void start(uint32_t load, uint32_t lap) { slot = load - lap * slots, parity = lap & 1; }
    __device__ __forceinline__ void step(uint32_t loads) {  // fewer than there are slots
        slot += loads;
        if (slot >= slots) slot -= slots, parity ^= 1;
    }
};

struct Barriers {
    uint64_t full[20], empty[20];              // tiles of K and V that both groups take
    uint64_t own_full[2][10], own_empty[2][10];    // ... that one takes: half of the slots each
    uint64_t query_full[2][2], query_empty[2][2];  // of the groups: two buffers
    uint64_t scores[2][2], weights[2][2], summed[2][2];  // of the groups' two buffers: S is there, P is there, P . V is done
    uint64_t result[2];                        // of the groups: O of a piece is complete
    uint64_t changed;                          // the pieces of one kind are done, those of another begin
    uint64_t list_full[2], list_empty[2];      // batches of pieces
    Piece list[2 * kBatch];
    Share share;
    uint32_t tmem_base;
    int warp_units[kThreads / 32];
};
constexpr int kListReaders = 4 + 8;            // producers, issuers, warps of the groups

// One role's way through the pieces.  Every batch is waited for and handed back.
struct Pieces {
    Barriers* bars;
    uint32_t i;               // pieces read
    __device__ __forceinline__ explicit Pieces(Barriers* b) : bars(b), i(0) {}
    // One thread's: the next piece, or the end (also when a wait has expired), after which there is none.
    __device__ __forceinline__ Piece next(bool* ok, int* error) {
        const uint32_t batch = i / kBatch;
        if (i % kBatch == 0) {
            if (batch > 0) mbar_arrive(&bars->list_empty[(batch - 1) & 1]);
            *ok = *ok && mbar_watch(&bars->list_full[batch & 1], (batch >> 1) & 1, error, 51);
        }
        Piece p = bars->list[i % (2 * kBatch)];
        if (!*ok) p.who = kEnd;
        ++i;
        return p;
    }
    // A whole warp's.
    __device__ __forceinline__ Piece next_of_warp(bool* ok, int* error) {
        const uint32_t batch = i / kBatch;
        if (i % kBatch == 0) {
            __syncwarp();
            if (batch > 0 && threadIdx.x % 32 == 0) mbar_arrive(&bars->list_empty[(batch - 1) & 1]);
            *ok = *ok && __all_sync(0xFFFFFFFFu, mbar_watch(&bars->list_full[batch & 1], (batch >> 1) & 1, error, 51));
        }
        Piece p = bars->list[i % (2 * kBatch)];
        if (!*ok) p.who = kEnd;
        ++i;
        return p;
    }
};

// K and V of a tile are these loads of the piece, in the order in which the products want them: S of the tile
// after next comes before P . V of the next one.
__device__ __forceinline__ uint32_t load_of_k(int tile) { return tile == 0 ? 0u : uint32_t(2 * tile - 1); }
__device__ __forceinline__ uint32_t load_of_v(int tile, int tiles) { return uint32_t(2 * tile + (tile == tiles - 1 ? 1 : 2)); }

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
    constexpr int kOwnSlots = S::kSlots / 2;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kSlots; ++s) mbar_init(&bars.full[s], 1), mbar_init(&bars.empty[s], 2);
        for (int g = 0; g < 2; ++g) {
            for (int s = 0; s < kOwnSlots; ++s) mbar_init(&bars.own_full[g][s], 1), mbar_init(&bars.own_empty[g][s], 1);
            for (int b = 0; b < 2; ++b) {
                mbar_init(&bars.query_full[g][b], 1), mbar_init(&bars.query_empty[g][b], 1);
                mbar_init(&bars.scores[g][b], 1), mbar_init(&bars.weights[g][b], 4), mbar_init(&bars.summed[g][b], 1);
            }
            mbar_init(&bars.result[g], 1);
            mbar_init(&bars.list_full[g], 1), mbar_init(&bars.list_empty[g], kListReaders);
        }
        mbar_init(&bars.changed, 4);  // producers and issuers
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

    // ---- this block's share: every thread sums some rows' own units ----
    {
        const int per = (a.batch + kThreads - 1) / kThreads, from = min(int(threadIdx.x) * per, a.batch), to = min(from + per, a.batch);
        int mine = 0;
        const int keys = prefix_length(a);
#pragma unroll 1
        for (int b = from; b < to; ++b) {
            const int64_t position = ld_mutable(a.positions + b);
            if (blockIdx.x == 0 && (position < -1 || position >= a.slots)) record_bad_position(a.status, b);
            mine += own_units(own_keys(a, position));
        }
        int before = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int other = __shfl_up_sync(0xFFFFFFFFu, before, d);
            if (lane >= d) before += other;
        }
        if (lane == 31) bars.warp_units[warp] = before;
        before -= mine;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += bars.warp_units[w];
            all += bars.warp_units[w];
        }
        const int own_first = a.items * prefix_units(a, tiles_of(keys)), total = own_first + all * a.nkv;
        const Deal deal(total, gridDim.x);
        const int first = deal.first(blockIdx.x), last = deal.first(blockIdx.x + 1);
        const int look = max(first, own_first);  // the first own unit this block can have
        if (threadIdx.x == 0) share.first = first, share.last = last, share.own_first = own_first, share.prefix_keys = keys;
        const int begin = own_first + before * a.nkv, end = begin + mine * a.nkv;
        if (look >= begin && look < end) {
            int row = from, at = begin;
#pragma unroll 1
            for (; per > 1; ++row) {  // (one row a thread: it is this one)
                const int each = own_units(own_keys(a, ld_mutable(a.positions + row)));
                if (look < at + each * a.nkv) break;
                at += each * a.nkv;
            }
            share.own_row = row, share.own_row_unit = at;
        }
        if (blockIdx.x == 0) {  // for the joining kernel
            int c = before;
#pragma unroll 1
            for (int b = from; b < to; ++b) {
                a.cum[b] = c;
                if (b + 1 < to) c += own_units(own_keys(a, ld_mutable(a.positions + b)));
            }
            if (threadIdx.x == 0) {
                a.cum[a.batch] = total, a.cum[a.batch + 1] = tiles_of(keys);
                const int64_t given = a.prefix_at != nullptr ? ld_mutable(a.prefix_at) : 0;
                if (given < 0 || given > a.prefix) record_bad_position(a.status, 0);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem_base);

    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {  // of a whole warp; bounded
        return __all_sync(0xFFFFFFFFu, mbar_watch(bar, parity, a.error, code));
    };
    bool ok = true;

    if (warp == kProducerWarp || warp == kProducerWarp + 1) {
        // ---- group g's queries, and its tiles of K and V (producer 0: those of both, too) ----
        if (lane == 0) {
            const int g = warp - kProducerWarp;
            Pieces pieces(&bars);
            uint32_t changes = 0, both_end = 0, own_end = 0;  // loads so far
            uint32_t filled = 0;                              // query buffers that were ever filled, and the last fills' parities
            for (;;) {
                const Piece p = pieces.next(&ok, a.error);
                if (p.who == kEnd) break;
                for (; ok && changes != p.epoch; changes = (changes + 1) & 255) {  // the memory is divided anew
                    mbar_arrive(&bars.changed);
                    ok = mbar_watch(&bars.changed, changes & 1, a.error, 40);
                }
                if (!ok) break;
                if (!p.of(g) || p.tiles == 0) continue;
                const Query query(p, g);
                const uint32_t buffer = query.buffer();
                ok = query.first() || mbar_watch(&bars.query_empty[g][buffer], query.parity() ^ 1, a.error, 47);
                if (!ok) break;
                const bool own = p.kind == kOwn, both = p.who == kBoth;
                // (batch rows past the last one read as zeros; rows of the buffer past the box are never looked at)
                mbar_expect_tx(&bars.query_full[g][buffer], uint32_t(S::kHalves * 128 * a.rep * (own ? 1 : a.tile_rows)));
#pragma unroll
                for (int c = 0; c < S::kHalves; ++c)
                    tma_load_4d(smem_u32(smem) + g * S::kQuery + c * (kRows * 128) + buffer * (64 * 128), own ? &own_q : &prefix_q, c * 64, 0,
                                p.head, p.row + (both && g == 1 ? a.tile_rows : 0), &bars.query_full[g][buffer]);
                filled = (filled & ~(0x11u << buffer)) | (1u << buffer) | (query.parity() << (4 + buffer));
                if (both && g == 1) continue;
                uint64_t* const full = both ? bars.full : bars.own_full[g];
                uint64_t* const empty = both ? bars.empty : bars.own_empty[g];
                const uint32_t memory = smem_u32(slots) + (both ? 0 : g * kOwnSlots * S::kSlot), ring = both ? S::kSlots : kOwnSlots;
                uint32_t lap = both ? p.base / S::kSlots : p.base / kOwnSlots, slot = p.base - lap * ring;
                const int loads = 2 * p.tiles;
#pragma unroll 1
                for (int i = 0; i < loads; ++i) {
                    const bool value = i > 0 && ((i & 1) == 0 || i == loads - 1);
                    const int tile = i == 0 ? 0 : i == loads - 1 ? p.tiles - 1 : value ? i / 2 - 1 : (i + 1) / 2;
                    ok = lap == 0 || mbar_watch(&empty[slot], (lap - 1) & 1, a.error, 41);
                    if (!ok) break;
                    mbar_expect_tx(&full[slot], S::kSlot);
                    const CUtensorMap* map = own ? (value ? &cache_v : &cache_k) : value ? &prefix_v : &prefix_k;
#pragma unroll
                    for (int c = 0; c < S::kHalves; ++c)
                        tma_load_4d(memory + slot * S::kSlot + c * S::kHalf, map, c * 64, p.key + tile * kKeys, p.head, own ? p.row : 0, &full[slot]);
                    ++(both ? both_end : own_end);
                    if (++slot == ring) slot = 0, ++lap;
                }
                if (!ok) break;
            }
            if (!ok) {  // what is in flight lands before the block leaves
                for (uint32_t i = both_end > S::kSlots ? both_end - S::kSlots : 0; i < both_end; ++i)
                    mbar_watch(&bars.full[i % S::kSlots], (i / S::kSlots) & 1, a.error, 42);
                for (uint32_t i = own_end > kOwnSlots ? own_end - kOwnSlots : 0; i < own_end; ++i)
                    mbar_watch(&bars.own_full[g][i % kOwnSlots], (i / kOwnSlots) & 1, a.error, 42);
                for (int b = 0; b < 2; ++b)
                    if (filled >> b & 1) mbar_watch(&bars.query_full[g][b], filled >> (4 + b) & 1, a.error, 42);
            }
        }
        __syncwarp();
    } else if (warp == kIssuerWarp || warp == kIssuerWarp + 1) {
        // ---- the products of group g, from one thread ----
        if (elect_one()) {
            constexpr uint32_t kType = H::kDtype == B200Q_BF16 ? 1u : 0u;
            constexpr uint32_t kScores = (1u << 4) | (kType << 7) | (kType << 10) | (uint32_t(kKeys >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
            constexpr uint32_t kValues = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | (uint32_t(HD >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
            const int g = warp - kIssuerWarp;
            const uint32_t s_at = tmem + uint32_t(g) * 2 * kKeys, o_at = tmem + 4 * kKeys + uint32_t(g) * HD;
            const uint32_t scores = smem_u32(&bars.scores[g][0]), weights = smem_u32(&bars.weights[g][0]), summed = smem_u32(&bars.summed[g][0]),
                           result = smem_u32(&bars.result[g]), query_full = smem_u32(&bars.query_full[g][0]),
                           query_empty = smem_u32(&bars.query_empty[g][0]), queries = (smem_u32(smem) + g * S::kQuery) >> 4;
            const uint32_t k_high = uint32_t(smem_desc(0) >> 32), k_low = uint32_t(smem_desc(0));
            const uint32_t v_high = uint32_t(value_desc(0, S::kHalf) >> 32), v_low = uint32_t(value_desc(0, S::kHalf));
            auto walk = [&](const Piece& p, uint32_t load) {
                const bool both = p.who == kBoth;
                Walk w;
                w.full = smem_u32(both ? bars.full : bars.own_full[g]), w.empty = smem_u32(both ? bars.empty : bars.own_empty[g]);
                w.memory = (smem_u32(slots) + (both ? 0 : g * kOwnSlots) * S::kSlot) >> 4, w.slots = both ? S::kSlots : kOwnSlots;
                w.start(p.base + load, both ? (p.base + load) / S::kSlots : (p.base + load) / kOwnSlots);
                return w;
            };
            // Two ways through the group's tiles: the sums', and the scores' up to two tiles ahead of it.
            Pieces pieces(&bars);
            Piece p, q;                           // the sums' and the scores' piece
            Walk vs = {}, ks = {};                // their loads
            int tile = 0, q_tile = 0;
            uint32_t task = 0, q_task = 0, q_index = 0, changes = 0;
            bool found = false;                   // q is the scores' next piece, or the end
            bool any_change = false;
            auto next_piece = [&]() {             // of the sums
                do {
                    p = pieces.next(&ok, a.error);
                    if (p.who == kEnd) break;
                    for (; changes != p.epoch; changes = (changes + 1) & 255) {  // the memory of one kind is free (not twice before all know)
                        if (any_change) ok = ok && mbar_watch(&bars.changed, (changes - 1) & 1, a.error, 40);
                        umma_commit(&bars.changed);
                        any_change = true;
                    }
                } while (!p.of(g) || p.tiles == 0);
                tile = 0;
                vs = walk(p, load_of_v(0, p.tiles));
            };
            // The next scores' operands, where they are to be had: their keys and queries are there (and are waited for
            // only if the sums have nothing to do without), and they lie neither beyond a change of kind that the sums
            // have not come to nor two batches on.
            uint32_t buffer = 0, query_parity = 0;
            auto scores_ready = [&]() {
                const bool wanted = q_task == task;
                while (!found) {
                    if (wanted) {
                        q = p, q_index = pieces.i, found = true;
                    } else {
                        const uint32_t batch = q_index / kBatch;
                        if (q_index % kBatch == 0 && (batch > (pieces.i - 1) / kBatch + 1 || !mbar_test(&bars.list_full[batch & 1], (batch >> 1) & 1))) return false;
                        q = bars.list[q_index++ % (2 * kBatch)];
                        found = q.who == kEnd || (q.of(g) && q.tiles > 0);
                    }
                    if (found && q.who != kEnd) {
                        const Query query(q, g);
                        q_tile = 0, buffer = query.buffer(), query_parity = query.parity();
                        ks = walk(q, load_of_k(0));
                    }
                }
                if (q.who == kEnd || q.epoch != p.epoch) return false;
                if (!wanted) return (q_tile > 0 || test_at(query_full + 8 * buffer, query_parity)) && test_at(ks.full + 8 * ks.slot, ks.parity);
                ok = (q_tile > 0 || watch_at(query_full + 8 * buffer, query_parity, a.error, 43)) &&
                     watch_at(ks.full + 8 * ks.slot, ks.parity, a.error, 44);
                return ok;
            };
            auto issue_scores = [&]() {
                const uint32_t b = q_task & 1, at = s_at + b * kKeys;
                const uint32_t qd = k_low + queries + buffer * (64 * 128 >> 4), kd = k_low + ks.memory + ks.slot * (S::kSlot >> 4);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)
                    umma_f16_ss(at, desc_of(qd + uint32_t(k / 4) * ((kRows * 128) >> 4) + uint32_t(k % 4) * 2, k_high),
                                desc_of(kd + uint32_t(k / 4) * (S::kHalf >> 4) + uint32_t(k % 4) * 2, k_high), kScores, k > 0);
                commit_at(scores + 8 * b);
                commit_at(ks.empty + 8 * ks.slot);
                ++q_task;
                ks.step(q_tile == 0 ? 1 : 2);
                if (++q_tile == q.tiles) {
                    commit_at(query_empty + 8 * buffer);
                    found = false;
                }
            };
            next_piece();
            while (ok && p.who != kEnd) {
                while (q_task < task + 2 && scores_ready()) {
                    tc_fence_after();
                    issue_scores();
                }
                // The scores after those follow the sums at once, in the buffer that the sums read their weights from.
                const bool follows = ok && q_task == task + 2 && scores_ready();
                const uint32_t b = task & 1, from = s_at + b * kKeys, vd = v_low + vs.memory + vs.slot * (S::kSlot >> 4);
                const int keys = p.keys - tile * kKeys;
                const bool last = tile + 1 == p.tiles;
                ok = ok && watch_at(vs.full + 8 * vs.slot, vs.parity, a.error, 44) && watch_at(weights + 8 * b, (task >> 1) & 1, a.error, 45);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k)
                    if (k == 0 || k * 16 < keys) umma_f16_ts(o_at, from + k * 8, desc_of(vd + uint32_t(k) * (2048 >> 4), v_high), kValues, k > 0 || tile > 0);
                if (last) commit_at(result);
                commit_at(summed + 8 * b);
                if (follows) issue_scores();
                commit_at(vs.empty + 8 * vs.slot);
                ++task, ++tile;
                if (last) next_piece();
                else vs.step(tile + 1 == p.tiles ? 1 : 2);
            }
        }
        __syncwarp();
    } else if (warp == kListWarp) {
        // ---- the pieces, a batch at a time ----
        int t = share.first, row = share.own_row, at = share.own_row_unit;
        int keys_of = 0, held = -1;            // own keys of rows 32 * held + lane
        const int prefix_end = min(share.own_first, share.last), prefix_tiles = tiles_of(share.prefix_keys);
        const int item_units = prefix_units(a, prefix_tiles);
        uint32_t loads_both = 0, loads_0 = 0, loads_1 = 0;     // before the batch's next piece: loads of the rings,
        uint32_t fills = 0, own_fills = 0;                     // pieces of the groups (16 bits each): of a prefix, of own keys
        int kind = -1;
        uint32_t epoch = 0;
        for (uint32_t batch = 0; ok; ++batch) {
            // (of the counts only "any" and the last two bits are asked for: long ones are kept from running into one another)
            fills -= (fills & 0x80008000u) >> 1, own_fills -= (own_fills & 0x80008000u) >> 1;
            if (batch >= 2) ok = wait(&bars.list_empty[batch & 1], ((batch >> 1) - 1) & 1, 52);
            if (!ok) break;
            Piece* list = bars.list + (batch & 1) * kBatch;
            int n = 0;
            while (n < kBatch && t < share.last) {
                Piece p;
                int first_tile, end_tile, count;  // this lane's tiles of its item; lanes that write
                if (t < prefix_end) {             // two lanes an item: both groups' piece, or a group's half of the keys each
                    const int item0 = quotient(t, item_units), item = item0 + lane / 2, head = quotient(item, a.row_tiles), tile = item - head * a.row_tiles;
                    const int first = item * item_units;
                    first_tile = max(0, ((max(t, first) - first + a.weight - 1) >> (a.weight - 1)) - kPrefixStart);  // (a weight is 1 or 2)
                    end_tile = max(first_tile, ((min(first + item_units, prefix_end) - first + a.weight - 1) >> (a.weight - 1)) - kPrefixStart);
                    p.head = static_cast<unsigned short>(head), p.row = tile * 2 * a.tile_rows;
                    p.rows = static_cast<unsigned short>(max(0, min(2 * a.tile_rows, a.batch - p.row)));
                    p.place = item + int(blockIdx.x);
                    const bool both = p.rows > a.tile_rows;
                    p.kind = both ? kRowsOfBoth : kHalves;
                    p.who = both ? (lane & 1 ? kNobody : kBoth) : (lane & 1 ? kGroup1 : kGroup0);
                    if (!both) {
                        const int middle = first_tile + (end_tile - first_tile + 1) / 2;
                        (lane & 1 ? first_tile : end_tile) = middle;
                    } else if (end_tile <= first_tile) {
                        p.who = kNobody;
                    }
                    p.key = first_tile * kKeys, p.keys = share.prefix_keys - p.key;
                    const int items = quotient(prefix_end - item0 * item_units + item_units - 1, item_units);
                    count = min(kBatch - n, 2 * items);
                    t = min(prefix_end, (item0 + count / 2) * item_units);
                } else {                          // a head of the row a lane; one group's: the other is at the piece before or after
                    int keys, each;
                    for (;; ++row) {              // (t is before the end of the sequence: some row has it)
                        if (row / 32 != held) {
                            held = row / 32;
                            const int r = held * 32 + lane;
                            keys_of = r < a.batch ? own_keys(a, ld_mutable(a.positions + r)) : 0;
                        }
                        keys = __shfl_sync(0xFFFFFFFFu, keys_of, row % 32);
                        each = own_units(keys);
                        if (t < at + each * a.nkv) break;
                        at += each * a.nkv;
                    }
                    const int head0 = quotient(t - at, each), head = head0 + lane, first = at + head * each;
                    first_tile = max(0, t - first - kOwnStart), end_tile = min(tiles_of(keys), share.last - first - kOwnStart);
                    p.head = static_cast<unsigned short>(head), p.row = row, p.rows = 1, p.kind = kOwn;
                    p.who = end_tile <= first_tile ? kNobody : (n + lane) & 1 ? kGroup1 : kGroup0;
                    p.key = first_tile * kKeys, p.keys = keys - p.key;
                    p.place = row * a.nkv + head + int(blockIdx.x);
                    const int left = min(a.nkv - head0, quotient(share.last - (at + head0 * each) + each - 1, each));
                    count = min(kBatch - n, left);
                    t = min(share.last, at + (head0 + count) * each);
                }
                p.tiles = max(0, end_tile - first_tile);
                // Sums over the pieces before: of the lanes before this one, and of those written before.
                const bool counts = lane < count && p.tiles > 0 && p.who <= kBoth, own = p.kind == kOwn;
                const uint32_t n_loads = counts ? 2 * p.tiles : 0, which = !counts ? 0u : p.who == kBoth ? 0x10001u : p.who == kGroup0 ? 1u : 0x10000u;
                uint32_t sum_both = p.who == kBoth ? n_loads : 0, sum_0 = p.who == kGroup0 ? n_loads : 0, sum_1 = p.who == kGroup1 ? n_loads : 0;
                uint32_t sum_fills = own ? 0 : which, sum_own = own ? which : 0;
                const uint32_t mine_both = sum_both, mine_0 = sum_0, mine_1 = sum_1, mine_fills = sum_fills, mine_own = sum_own;
                auto before = [&](uint32_t& sum, uint32_t mine, uint32_t& total) {  // exclusive over the lanes; adds up the total
#pragma unroll
                    for (int d = 1; d < kBatch; d <<= 1) {
                        const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, sum, d);
                        if (lane >= d) sum += other;
                    }
                    const uint32_t all = __shfl_sync(0xFFFFFFFFu, sum, count - 1);
                    sum = total + sum - mine;
                    total += all;
                };
                before(sum_both, mine_both, loads_both), before(sum_0, mine_0, loads_0), before(sum_1, mine_1, loads_1);
                before(sum_fills, mine_fills, fills), before(sum_own, mine_own, own_fills);
                p.base = p.who == kBoth ? sum_both : p.who == kGroup0 ? sum_0 : sum_1;
                p.query = 0;
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const uint32_t f = sum_fills >> (16 * g) & 0xFFFFu, o = sum_own >> (16 * g) & 0xFFFFu;
                    const uint32_t buffer = own && a.rep <= 64 ? o & 1 : 0, times = buffer ? o / 2 : f + (a.rep <= 64 ? (o + 1) / 2 : o);
                    p.query |= static_cast<unsigned char>((buffer | (times & 1) << 1 | (times > 0 ? 4 : 0)) << (4 * g));
                }
                // a change of kind: against the lane before, and of the first lane against what was written last
                const int kind_up = __shfl_up_sync(0xFFFFFFFFu, int(p.kind), 1);
                const bool changes = lane < count && (lane == 0 ? kind >= 0 && p.kind != kind : int(p.kind) != kind_up);
                const uint32_t change_mask = __ballot_sync(0xFFFFFFFFu, changes);
                p.epoch = static_cast<unsigned char>(epoch + __popc(change_mask & (0xFFFFFFFFu >> (31 - lane))));
                epoch += __popc(change_mask);
                kind = __shfl_sync(0xFFFFFFFFu, int(p.kind), count - 1);
                if (lane < count) list[n + lane] = p;
                n += count;
            }
            const bool over = n < kBatch;
            if (over && lane == 0) list[n].who = kEnd;
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.list_full[batch & 1]);
            if (over) break;
        }
    } else {
        // ---- softmax: group g, one query row a thread ----
        const int g = warp / 4, row = threadIdx.x % 128;
        const uint32_t lanes = tmem + (uint32_t(warp & 3) << 21);
        const uint32_t s_at = lanes + uint32_t(g) * 2 * kKeys, o_at = lanes + 4 * kKeys + uint32_t(g) * HD;
        Pieces list(&bars);
        uint32_t task = 0, pieces = 0;            // that this group has had
        // f16 has no weights below 2^-24: the largest is made 2^7 there (and 2^15 at most, before its maximum moves), so that
        // those of 2^-21 of it still are normal numbers, and what is lost of any is 2^-32 of it at most.
        constexpr float kLift = H::kDtype == B200Q_F16 ? 7.0f : 0.0f;
        for (;;) {
            const Piece p = list.next_of_warp(&ok, a.error);
            if (p.who == kEnd) break;
            if (!p.of(g)) continue;
            const int live = p.who == kBoth ? min(a.tile_rows, p.rows - g * a.tile_rows) * a.rep : p.rows * a.rep;
            const bool any = (warp & 3) * 32 < live;  // of this warp's rows
            float m = 0.0f, l = 0.0f;
            for (int tile = 0; tile < p.tiles && ok; ++tile, ++task) {
                const int keys = p.keys - tile * kKeys;   // of the tile, and more
                const uint32_t b = task & 1, at = s_at + b * kKeys;
                ok = wait(&bars.scores[g][b], (task >> 1) & 1, 48);
                // The sums of two tiles ago, which these scores stood behind, but by a commit of their own: every phase of
                // `summed` is waited for in order (no later one of this barrier can be over, its weights are not made yet),
                // or the wait for the sums of the last tile, below, could take the phase before theirs for it.
                if (ok && task >= 2) ok = wait(&bars.summed[g][b], ((task - 2) >> 1) & 1, 53);
                if (!ok) break;
                tc_fence_after();
                if (any) {
                    uint32_t v[kKeys];
                    tmem_ask_32(v, at), tmem_ask_32(v + 32, at + 32);
                    tmem_arrived(v), tmem_arrived(v + 32);
                    if (keys < kKeys) {
#pragma unroll
                        for (int i = 0; i < kKeys; ++i) v[i] = i < keys ? v[i] : 0xFF800000u;
                    }
                    float most[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) most[i] = __uint_as_float(v[i]);
#pragma unroll
                    for (int i = 8; i < kKeys - 8; i += 16)
#pragma unroll
                        for (int k = 0; k < 8; ++k) most[k] = max3(most[k], __uint_as_float(v[i + k]), __uint_as_float(v[i + 8 + k]));
#pragma unroll
                    for (int k = 0; k < 8; ++k) most[k] = fmaxf(most[k], __uint_as_float(v[kKeys - 8 + k]));
                    const float here = a.scale_log2 * fmaxf(max3(max3(most[0], most[1], most[2]), most[3], most[4]),
                                                            max3(most[5], most[6], most[7]));
                    if (tile == 0) {
                        m = here > -INFINITY ? here - kLift : kLowest;  // (NaN too: l is NaN then, and m says that it was stored)
                    } else if (__any_sync(0xFFFFFFFFu, row < live && here - kLift > m + kStale)) {
                        const float next = here - kLift > m + kStale ? here - kLift : m, by = exp2_approx(m - next);
                        m = next;
                        l *= by;
                        ok = wait(&bars.summed[g][b ^ 1], ((task - 1) >> 1) & 1, 53);
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
                    // Scaled scores run kAhead pairs ahead of the exponentials and the sums as far behind, so that
                    // the exponential unit, which takes eight clocks an instruction, always has one to do.
                    constexpr int kPairs = kKeys / 2, kAhead = 4;
                    uint32_t weights[kPairs];
                    float2 e[kPairs], sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                    auto scaled = [&](int i) {
                        e[i].x = fmaf(__uint_as_float(v[2 * i]), a.scale_log2, -m), e[i].y = fmaf(__uint_as_float(v[2 * i + 1]), a.scale_log2, -m);
                    };
                    auto added = [&](int i) {
                        sum[i & 1] = add2(sum[i & 1], e[i]);
                        weights[i] = H::pack(e[i].x, e[i].y);
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
                    tmem_put_32(at, weights);
                    const float2 pair = add2(sum[0], sum[1]);
                    l += pair.x + pair.y;
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                if (keys < kKeys) {
                    // Rows of V past the last key may hold anything, and 0 * NaN is no 0: those that the last
                    // step of 16 keys takes in are cleared (by either group where both use the tile).
                    const bool both = p.who == kBoth;
                    const uint32_t load = p.base + load_of_v(tile, p.tiles), lap = both ? load / S::kSlots : load / kOwnSlots,
                                   slot = load - lap * (both ? S::kSlots : kOwnSlots);
                    ok = ok && wait((both ? bars.full : bars.own_full[g]) + slot, lap & 1, 49);
                    if (!ok) break;
                    uint8_t* tail = slots + ((both ? 0 : g * kOwnSlots) + slot) * S::kSlot;
                    const int rows = (16 - keys % 16) % 16;
#pragma unroll 1
                    for (int i = row; i < rows * 8 * S::kHalves; i += 128) {
                        const int c = S::kHalves == 1 ? 0 : (i >> 3) & 1, r = keys + (i >> 3) / S::kHalves;
                        *reinterpret_cast<uint4*>(tail + c * S::kHalf + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.weights[g][b]);
            }
            if (!ok) break;
            // ---- the piece's result ----
            const int span = p.kind == kOwn ? a.rep : kRows;  // rows of a group in the scratch memory
            float* to = a.scratch + (p.kind == kOwn ? a.own_at + p.place * group_floats(a.rep, HD) : (2 * int64_t(p.place) + g) * group_floats(kRows, HD));
            if (p.tiles > 0) {
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
                to[int64_t(HD) * span + row] = p.tiles > 0 ? m : -INFINITY;
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
// the way to the L2 cache, so a thread has several parts in flight: 8 of two columns (of four numbers), or
// where there are rows enough for a block on every multiprocessor, 4 of four.  (64 rows of 8192 + 512 keys
// 35.7 us so and 38.0 with four columns; 256 of 16384 + 128, 104.3 with four and 106.6 with two.)  Few parts a
// row: the warps share its columns.  Many (a long prefix for few rows and heads): the parts are dealt
// among the warps, and their sums meet in shared memory.
constexpr int kJoinWarps = 8;
// More than so many parts of a row are dealt among the warps, where there are fewer than so many blocks of rows
// and heads: 33 rows of 5001 keys, 2 KV heads (16 blocks), 12.8 us so and 21.1 otherwise; 64 of 16384 + 64, 8 KV heads
// (64 blocks), 43.5 so and 39.6 otherwise; 256 of 1024 + 128, few parts, 71.6 so and 41.8 otherwise.
constexpr int kManyParts = 12, kFewBlocks = 32;

template <typename T, int HD, bool MANY, int COLUMNS>
__global__ void __launch_bounds__(32 * kJoinWarps)
prefix_join_kernel(const __grid_constant__ PrefixArgs a, int blocks) {
    using H = Half16<T>;
    constexpr int kSlices = MANY ? kJoinWarps : 1;     // warps that share a row's parts
    constexpr int kSums = 4 * COLUMNS, kJoinHeld = 16 / COLUMNS;
    __shared__ float sums[MANY ? kJoinWarps : 1][kSums + 2][32];  // O, m and l
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int head = blockIdx.y, row = blockIdx.x * 32 + lane;  // row: batch row * rep + head of the group
    const int slice = MANY ? warp : 0, column = (MANY ? int(blockIdx.z) : int(blockIdx.z) * kJoinWarps + warp) * COLUMNS;
    const bool live = row < a.batch * a.rep;
    const int b = live ? quotient(row, a.rep) : 0, r = row - b * a.rep;
    auto word = [&](int i) { return int(ld_mutable(reinterpret_cast<const uint32_t*>(a.cum) + i)); };
    const int total = word(a.batch), prefix_tiles = word(a.batch + 1), before = word(b);
    const int keys = own_keys(a, ld_mutable(a.positions + b));
    const Deal deal(total, blocks);

    struct Item {              // the prefix, and the row's own keys
        const float* base;     // of the first group that has the row, in the first piece
        int parts, skip;       // groups that have the row: over all pieces; and the floats from one to the next
        int span, at;          // rows of a group in the scratch memory, and which one this is
    } shared = {}, own = {};
    if (live && prefix_tiles > 0) {
        const int pair = quotient(b, 2 * a.tile_rows), within = b - pair * 2 * a.tile_rows;
        const bool both = min(2 * a.tile_rows, a.batch - pair * 2 * a.tile_rows) > a.tile_rows;
        const int item = head * a.row_tiles + pair, first = item * prefix_units(a, prefix_tiles) + kPrefixStart * a.weight;
        const int from = deal.block_of(first), to = deal.block_of(first + (prefix_tiles - 1) * a.weight);
        const int g = both && within >= a.tile_rows, groups = both ? 1 : 2;
        shared.base = a.scratch + (2 * int64_t(item + from) + g) * group_floats(kRows, HD);
        shared.parts = (to - from + 1) * groups, shared.skip = int(group_floats(kRows, HD)) * (2 / groups);
        shared.span = kRows, shared.at = (within - g * a.tile_rows) * a.rep + r;
    }
    if (live && keys > 0) {
        const int first = a.items * prefix_units(a, prefix_tiles) + before * a.nkv + head * own_units(keys) + kOwnStart;
        const int from = deal.block_of(first), to = deal.block_of(first + tiles_of(keys) - 1);
        own.base = a.scratch + a.own_at + int64_t(b * a.nkv + head + from) * group_floats(a.rep, HD);
        own.parts = to - from + 1, own.skip = int(group_floats(a.rep, HD));
        own.span = a.rep, own.at = r;
    }
    const int parts = shared.parts + own.parts;
    float m = -INFINITY, l = 0.0f, o[kSums] = {};
    for (int k0 = slice; k0 < parts; k0 += kSlices * kJoinHeld) {
        float ms[kJoinHeld], ls[kJoinHeld];
        uint4 os[kJoinHeld][COLUMNS];
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
            for (int c = 0; c < COLUMNS; ++c) os[u][c] = ld_mutable(reinterpret_cast<const uint4*>(from) + (column + c) * it.span + it.at);
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
            for (int c = 0; c < COLUMNS; ++c) {
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
    int tile_rows, row_tiles, items, weight, blocks;
    bool many;                             // parts of a row
    int64_t own_at, cum_at, floats;
};

PrefixPlan plan_of(int64_t batch, int64_t nkv, int64_t rep, int64_t hd, int64_t prefix, int64_t slots) {
    PrefixPlan p;
    p.tile_rows = int(kRows / rep);
    p.row_tiles = prefix > 0 ? int((batch + 2 * p.tile_rows - 1) / (2 * p.tile_rows)) : 0;
    p.items = int(nkv) * p.row_tiles;
    p.weight = batch > p.tile_rows ? 2 : 1;
    p.blocks = sm_count();
    const int64_t of_prefix = (prefix + kKeys - 1) / kKeys, of_own = (slots + kKeys - 1) / kKeys;
    const int64_t units = p.items * (of_prefix + kPrefixStart) * p.weight + batch * nkv * (of_own + kOwnStart);
    if (units / 2 < p.blocks) p.blocks = units < 2 ? 1 : int(units / 2);
    // Parts of a row, were all rows' caches full: blocks an item's tiles are spread over, and a block at either end.
    const int64_t share = units < 1 ? 1 : (units + p.blocks - 1) / p.blocks;
    const int64_t parts = (p.items > 0 ? ((of_prefix * p.weight + share - 1) / share + 1) * (batch > p.tile_rows ? 1 : 2) : 0) + (of_own + share - 1) / share + 1;
    p.many = parts > kManyParts && (batch * rep + 31) / 32 * nkv < kFewBlocks;
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
    // (a multiprocessor's share of these takes a third of a second, so that no role waits for the second that ends a wait)
    B200Q_REQUIRE(2 * nkv * row_tiles * (prefix / kKeys + 1 + kPrefixStart) + batch * nkv * (slots / kKeys + 2) < (int64_t(1) << 26) &&
                      batch * nq < (int64_t(1) << 30),
                  "prefix_attention: 2^26 tiles of 64 keys or more (those of the prefix counted for every 128 rows), or 2^30 rows times heads");
    return B200Q_OK;
}

// A map of boxes of 64 numbers x `rows` x 1 x `last` (keys and values: the keys of a tile); strides in numbers.
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
    const unsigned rows = unsigned((a.batch * a.rep + 31) / 32);
    constexpr int warps = HD / 4 / (4 * kJoinWarps);  // of four columns: 1, or none where a warp has no more than two
    auto join = [&](auto kernel, unsigned parts) {
        return launch_overlapped(kernel, dim3(rows, unsigned(a.nkv), parts), dim3(32 * kJoinWarps), 0, stream, a, blocks);
    };
    if (many) return join(prefix_join_kernel<T, HD, true, 2>, HD / 8);
    if constexpr (warps > 0)
        if (int64_t(rows) * a.nkv >= sm_count()) return join(prefix_join_kernel<T, HD, false, 4>, warps);
    return join(prefix_join_kernel<T, HD, false, 2>, HD / 8 / kJoinWarps);
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
    const int64_t extents[12] = {batch, nq, prefix, nkv, prefix, nkv, max_seq, nkv, batch, max_seq, nkv, batch};
    for (int i = 0; i < 12; ++i)
        B200Q_REQUIRE(extents[i] <= 1 || (strides[i] % 8 == 0 && strides[i] > 0),
                      "prefix_attention: strides must be whole 16-byte steps");
    EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return unavailable("prefix_attention: the driver has no cuTensorMapEncodeTiled");

    const PrefixPlan p = plan_of(batch, nkv, nq / nkv, head_dim, prefix, max_seq);
    CUtensorMap maps[6] = {};
    // strides: q (row, head), then (key, head) of the prefix's keys and values, (key, head, row) of the caches'
    for (int v = 0; v < 2; ++v) {
        const int64_t shared[4] = {head_dim, prefix, nkv, 1}, alone[4] = {head_dim, max_seq, nkv, batch};
        CUresult made = CUDA_SUCCESS;
        if (prefix > 0) made = make_map(encode, &maps[v], v ? prefix_v : prefix_k, dtype, 4, shared, strides + 2 + 2 * v, kKeys, 1);
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
    a.tile_rows = p.tile_rows, a.row_tiles = p.row_tiles, a.items = p.items, a.weight = p.weight, a.own_at = p.own_at;
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
