// Attention of packed tables (tah_attend_packed): every table's queries over its own rows, causal or not, grouped heads, at f32's
// precision on the fp16 matrix cores.
//
// Keys and values become split-fp16 tiles first, one per (block of 64 of a table's rows, key/value head), laid out as the LDS
// images that the attention reads: tables begin at tiles of their own, short blocks are filled with zeros. Tables that few workgroups
// read get none: those make the images themselves. The attention then takes a tile of queries of one table and head a workgroup.
#include "common.hpp"
#include "device_math.hpp"
#include "tiles.hpp"

namespace tah {

namespace {

// What the attention's workgroups do (k_packed): of each head's units (of each 2^log_share heads'), `own` are a workgroup's each; the
// blocks of the others, `rest` of a head from block own_blocks on, go in `runs` runs of `per`.
struct PackedPlan {
    uint32_t own, own_blocks, rest, per, runs;
};

// A unit that several runs have parts of, from the one it begins in (slot) to last_run: `live` columns, queries from row on and heads
// from head on. live 0: there is none.
struct CutUnit {
    uint32_t slot, last_run;
    int row, live, head;
};

struct Packed {
    const float *q, *k, *v;
    const int32_t *qo, *ko;
    int tables, nq, nkv, heads, kv_heads, hd, causal;
    size_t q_ld, kv_ld;
    float *out;
    int log_share;  // a tile's columns are its queries' 2^log_share heads that share their keys
    // working memory: the tiles, per tile the keys' and the values' power of two (four times it, 2 if each row has one of its own, 1
    // if a value is not finite), the rows' own (64 of the keys, 64 of the values), which keys of each coordinate hold values that are
    // not finite; the attention's plan, and per table its first block of rows, and for one head the tiles of queries of the tables
    // before it and those tiles' blocks (tables + 1)
    int blocks;  // room for so many tiles of a head
    uint8_t *tiles;
    int *shifts;
    int8_t *row_shifts;
    uint64_t *odd;
    PackedPlan *plan;
    uint32_t *first, *tile_sums, *block_sums;
    // the attention's runs of blocks, and per slot (two a run) [queries][hd] outputs and [queries] (maximum, sum); per run the unit
    // that begins in it and ends in a later one
    int waves, runs;
    int direct;  // tables that few workgroups read are read where they stand (few_readers)
    float *part_o;
    float2 *part_ml;
    CutUnit *cut;
};

// rows [a, a + n) of table t, cut to what there are
__device__ __forceinline__ int rows_of(const int32_t *offsets, int t, int rows, int &a) {
    a = min(max(offsets[t], 0), rows);
    return min(max(offsets[t + 1], a), rows) - a;
}

// What beginning and ending a unit costs, in blocks of heads padded to D (8,000 rows in order, 8 heads of 64 that share their keys, 260,
// 237 and 225 us with 1, 2 and 3; three tables of up to 2,500, heads of 128, 99, 91 and 94). A unit of WHOLE blocks is not cut
// (30 tables of 350 to 380 rows 56 us, with 5 66; 20 of 400 to 700, in order, 60 and 57).
template <int D>
constexpr int BEGIN_OF = D == 128 ? 2 : 3;
constexpr int WHOLE = 8;

// A table's tiles of queries in the order in which they are taken (causal: the last first, which have the most to do), the blocks of
// tile i and of all tiles before it (BEGIN more for each). A tile has 2^log_queries queries.
template <int BEGIN>
struct Tiles {
    int n_q, n_k, causal, log_queries;
    __device__ __forceinline__ int count() const { return (n_q + (1 << log_queries) - 1) >> log_queries; }
    __device__ __forceinline__ int first_query(int i) const { return (causal ? count() - 1 - i : i) << log_queries; }
    __device__ __forceinline__ int all() const { return (n_k + KB - 1) / KB; }
    // causal, by place: tile j's last query sees the rows but those of the queries behind it, so its blocks are (seen() + j
    // 2^log_queries) / 64, none below 0, but for the last tile, which ends with the last query
    __device__ __forceinline__ int seen() const { return n_k - n_q + KB - 1 + (1 << log_queries); }
    __device__ __forceinline__ int blocks(int i) const {
        return !causal || i == 0 ? all() : max(0, (seen() + ((count() - 1 - i) << log_queries)) >> 6);
    }
    // sum of k >> log from 0 to n - 1
    __device__ __forceinline__ static long quotients(long n, int log) {
        const long q = n >> log;
        return ((q * (q - 1) / 2) << log) + q * (n - (q << log));
    }
    __device__ __forceinline__ uint64_t before(int i) const {
        if (!causal || i == 0) return (uint64_t)i * (all() + BEGIN);
        // places count() - i .. count() - 2, from the first that has blocks on, and the last
        const long c = seen(), j1 = count() - 1, low = count() - i;
        const long j0 = c >= KB ? low : max(low, min(j1, (KB - c + (1 << log_queries) - 1) >> log_queries));
        long sum;
        if (log_queries >= 6) {
            sum = (j1 - j0) * (c >> 6) + (((j1 * (j1 - 1) - j0 * (j0 - 1)) / 2) << (log_queries - 6));
        } else {
            const long f = c >> log_queries;
            sum = j0 < j1 ? quotients(f + j1, 6 - log_queries) - quotients(f + j0, 6 - log_queries) : 0;
        }
        return (uint64_t)(sum + all() + (long)i * BEGIN);
    }
};

// Whether a table's blocks are split by the workgroups that read them, without tiles: where up to three do (200 tables of 50 to 100
// rows 80 -> 56 us, 100 of 200 to 250, causal, 101 -> 87, 32 of 100 to 300 41 -> 39). More find the tiles as fast or faster (64 of 500
// to 1,000, causal, 257, without 268; 8 of 1,000 to 2,000 150 and 171).
constexpr int READERS = 3;
__device__ __forceinline__ bool few_readers(const Packed &p, int n_q) {
    const int log = 7 - p.log_share;  // of a tile's queries
    return p.direct && (int64_t)((n_q + (1 << log) - 1) >> log) * ((p.heads / p.kv_heads) >> p.log_share) <= READERS;
}

// Blocks that are made into tiles, of a table of n_q queries and n_k rows.
__device__ __forceinline__ uint32_t tiled_blocks(const Packed &p, int n_q, int n_k) {
    return few_readers(p, n_q) ? 0 : (uint32_t)((n_k + KB - 1) / KB);
}
// `first` of a table whose tiles are past the room that the offsets' promise gives: its queries see no rows
constexpr uint32_t NO_ROOM = 0x7fffffff;

// The table that tile `at` of all is of: its number (-1 if there are fewer), and the block of its rows. Every lane of a wavefront calls it.
__device__ __forceinline__ int table_with(const Packed &p, uint32_t at, uint32_t &block) {
    const int lane = threadIdx.x & 63;
    uint64_t before = 0;
    for (int t0 = 0; t0 < p.tables; t0 += 64) {
        int a = 0;
        const int t = min(t0 + lane, p.tables - 1);
        const uint32_t c = t0 + lane < p.tables ? tiled_blocks(p, rows_of(p.qo, t, p.nq, a), rows_of(p.ko, t, p.nkv, a)) : 0;
        const uint64_t sum = before + wave_scan(c);  // of 64 tables: below 2^32
        const uint64_t past = __ballot(sum > at);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            block = at - (uint32_t)__shfl(sum - c, l);
            return __builtin_amdgcn_readfirstlane(t0 + l);
        }
        before = __shfl(sum, 63);
    }
    return -1;
}

__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {  // of numbers below 2^50
    const uint32_t lo = wave_scan((uint32_t)v & 0x1ffffffu), hi = wave_scan((uint32_t)(v >> 25));
    return ((uint64_t)hi << 25) + lo;
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int l) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), l) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, l);
}

// One wavefront: the attention's plan for tiles of QT columns. As many units of each head as make whole rounds of p.runs workgroups are
// a workgroup's each. All of them where units are short, where they are of different lengths in two rounds or more (their ends
// overlap by themselves: ten tables of 1,000 to 5,000 rows 675 us, with runs 710; four of up to 8,000, in order, 452 and 460), or
// where blocks are too many for 32 bits.
template <int QT, int BEGIN>
__device__ void make_plan(const Packed &p) {
    const int lane = threadIdx.x & 63, heads = p.heads >> p.log_share, log_queries = (QT == 256 ? 8 : 7) - p.log_share;
    uint64_t rows = 0, units = 0, blocks = 0;
    int longest = 0, shortest = 0x7fffff;
    for (int t0 = 0; t0 < p.tables; t0 += 64) {
        const int t = min(t0 + lane, p.tables - 1);
        const bool in = t0 + lane < p.tables;
        int qa = 0, ka = 0;
        const int n_q = rows_of(p.qo, t, p.nq, qa), n_t = rows_of(p.ko, t, p.nkv, ka);
        const uint32_t nb = in ? tiled_blocks(p, n_q, n_t) : 0;
        const uint64_t before = rows + wave_scan(nb) - nb;  // of 64 tables: below 2^32
        const bool room = before + nb <= (uint64_t)p.blocks;
        if (in) p.first[t] = room ? (uint32_t)before : NO_ROOM;
        rows = lane64(before + nb, 63);
        const Tiles<BEGIN> ts{n_q, room ? n_t : 0, p.causal, log_queries};
        const uint64_t tiles = in ? ts.count() : 0, cost = in ? ts.before(ts.count()) : 0;
        const uint64_t tile_sum = units + wave_scan64(tiles), block_sum = blocks + wave_scan64(cost);
        if (in) {
            p.tile_sums[t] = (uint32_t)(tile_sum - tiles);
            p.block_sums[t] = (uint32_t)min(block_sum - cost, (uint64_t)0xffffffff);
        }
        units = lane64(tile_sum, 63);
        blocks = lane64(block_sum, 63);
        if (tiles) {
            longest = max(longest, ts.all());
            shortest = min(shortest, ts.all());
        }
    }
    longest = (int)wave_max((float)longest);
    shortest = (int)-wave_max(-(float)shortest);
    const uint64_t rounds = units * heads / p.runs;
    const bool even = !p.causal && shortest + 1 >= longest;
    uint64_t own = rounds * p.runs / heads;
    if (longest <= WHOLE || (!even && rounds >= 2) || blocks * heads >> 32) own = units;
    uint64_t own_blocks = own < units ? 0 : blocks;
    if (own > 0 && own < units)
        for (int t0 = 0; t0 < p.tables; t0 += 64) {
            const int t = min(t0 + lane, p.tables - 1);
            int qa = 0, ka = 0;
            const int n_q = rows_of(p.qo, t, p.nq, qa), n_t = rows_of(p.ko, t, p.nkv, ka);
            const Tiles<BEGIN> ts{n_q, p.first[t] != NO_ROOM ? n_t : 0, p.causal, log_queries};
            const uint64_t a = p.tile_sums[t];
            const uint64_t here = __ballot(t0 + lane < p.tables && own >= a && own < a + ts.count());
            if (here) {
                const int l = __ffsll((unsigned long long)here) - 1;
                own_blocks = lane64(p.block_sums[t] + ts.before((int)min(max(own, a) - a, (uint64_t)ts.count())), l);
                break;
            }
        }
    if (lane == 0) {
        const uint64_t rest = blocks - own_blocks, total = rest * heads;
        const uint64_t per = max((uint64_t)WHOLE, (total + p.runs - 1) / p.runs);
        p.tile_sums[p.tables] = (uint32_t)units;
        p.block_sums[p.tables] = (uint32_t)min(blocks, (uint64_t)0xffffffff);
        *p.plan = PackedPlan{(uint32_t)own, (uint32_t)own_blocks, (uint32_t)rest, (uint32_t)per, (uint32_t)((total + per - 1) / per)};
    }
}

// Bytes of half a tile of D coordinates, keys or values: keys by 64 coordinates, hi then lo [64 keys][64] each (D 32: [64 keys], a
// key's hi then its lo), values hi then lo [D][64 keys], rows of 128 bytes in swizzled chunks of 16 (swz).
template <int D>
constexpr int HALF_BYTES = D * 256;

// Where rows of a block lie further apart than this, each row takes a power of two of its own. One for all would cost a
// row 2^-39 of the block's largest number, so less than 2^-26 of its own within this; and rows that a query does not see would
// count, in order, for the rows before them. Layer norms leave rows within a few powers of two of each other.
constexpr float APART = 0x1p-12f;
__device__ __forceinline__ bool rows_apart(float least, float most) { return least < most * APART; }  // least: not of zeros

// the largest of LANES lanes next to each other, in each
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
    v = fmaxf(v, dpp<0xb1>(v));
    v = fmaxf(v, dpp<0x4e>(v));
    if constexpr (LANES >= 8) v = fmaxf(v, dpp<0x141>(v));
    if constexpr (LANES >= 16) v = fmaxf(v, dpp<0x140>(v));
    return v;
}

// the same of floats' bits, which NaN pass
template <int LANES>
__device__ __forceinline__ uint32_t lanes_most(uint32_t v) {
    auto step = [](uint32_t a, int b) { return max(a, (uint32_t)b); };
    v = step(v, __builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, false));
    v = step(v, __builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, false));
    if constexpr (LANES >= 8) v = step(v, __builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, false));
    if constexpr (LANES >= 16) v = step(v, __builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, false));
    return v;
}

// grid (blocks, key/value heads, keys and values); 256 threads: one half tile. Scaled by the power of two that brings its own
// largest finite number below 2^14, or each row by one of its own (APART). A value that is not finite is a zero in the tile, and its
// bit is set in `odd`. Bound by bytes: 10,000 rows of 8 heads of 64, 41 MB read and 41 written, 16.7 us at least (median 17.9), 4.9 TB/s.
template <int D>
__global__ __launch_bounds__(256) void k_packed_tiles(Packed p) {
    __shared__ float x[KB][D + 1];
    constexpr int LANES = D / 4 < 16 ? D / 4 : 16, PARTS = D / 4 / LANES;  // of a row
    __shared__ uint32_t rows_most[KB][PARTS];
    __shared__ float scale_here[4][KB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = blockIdx.y;
    const bool values = blockIdx.z == 1;
    if (blockIdx.x == 0 && h == 0 && !values && tid < 64) p.waves == 8 ? make_plan<256, BEGIN_OF<D>>(p) : make_plan<128, BEGIN_OF<D>>(p);
    uint32_t kb = 0;
    const int t = table_with(p, blockIdx.x, kb);
    if (t < 0) return;
    int a = 0;
    const int n = min(rows_of(p.ko, t, p.nkv, a) - (int)kb * KB, KB);
    const float *src = (values ? p.v : p.k) + (size_t)(a + (int)kb * KB) * p.kv_ld + (size_t)h * p.hd;
#pragma unroll
    for (int i = 0; i < KB * D / 4 / 256; i++) {
        const int u = tid + 256 * i, r = u / (D / 4), dim = 4 * (u % (D / 4));
        const floatx4 w = r < n && dim < p.hd ? (floatx4) * reinterpret_cast<const floatx4u *>(src + (size_t)r * p.kv_ld + dim)
                                              : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t raw = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float f = w[j];
            raw = max(raw, __float_as_uint(f) & 0x7fffffffu);
            x[r][dim + j] = f;
        }
        raw = lanes_most<LANES>(raw);
        if (dim % (4 * LANES) == 0) rows_most[r][dim / (4 * LANES)] = raw;
    }
    __syncthreads();
    // a row a lane
    uint32_t raw = rows_most[lane][0];
#pragma unroll
    for (int i = 1; i < PARTS; i++) raw = max(raw, rows_most[lane][i]);
    const bool any = __any(raw >= 0x7f800000u), odd = values && any;
    if (any) {
        raw = 0;
        for (int j = 0; j < D; j++) raw = max(raw, finite_bits(__float_as_uint(x[lane][j])));
    }
    const float mine = __uint_as_float(raw), most = wave_max(mine), least = -wave_max(raw ? -mine : -INFINITY);
    const bool apart = rows_apart(least, most);
    const int shift = shift_below(most), own = apart ? shift_below(mine) : shift;
    scale_here[wave][lane] = pow2(own);  // each wavefront reads what it wrote
    const float *scale = scale_here[wave];
    const size_t at = (size_t)blockIdx.x * p.kv_heads + h;
    if (tid == 0) p.shifts[2 * at + (values ? 1 : 0)] = 4 * shift + (apart ? 2 : 0) + (odd ? 1 : 0);
    if (tid < KB) p.row_shifts[(2 * at + (values ? 1 : 0)) * KB + tid] = (int8_t)own;
    uint8_t *tile = p.tiles + at * (2 * HALF_BYTES<D>);
    if (odd && tid < D) {
        uint64_t bits = 0;
        for (int r = 0; r < KB; r++) {
            const bool b = (__float_as_uint(x[r][tid]) & 0x7fffffffu) >= 0x7f800000u;
            bits |= (uint64_t)b << r;
        }
        p.odd[at * D + tid] = bits;
    }
#pragma unroll
    for (int i = 0; i < D * 8 / 256; i++) {
        const int u = tid + 256 * i;
        float w[8];
        uint8_t *hi, *lo;
        if (values) {
            const int c = u & 7, r = u >> 3;  // coordinate r, keys 8 c ..
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = x[8 * c + e][r];
                w[e] = (odd && (__float_as_uint(y) & 0x7fffffffu) >= 0x7f800000u ? 0.0f : y) * scale[8 * c + e];
            }
            hi = tile + HALF_BYTES<D> + r * 128 + swz(r, c) * 16;
            lo = hi + D * 128;
        } else {
            constexpr int CHUNKS = D < 64 ? D / 8 : 8;
            const int c = u % CHUNKS, r = (u / CHUNKS) & 63, part = u / (64 * CHUNKS);  // key r, coordinates 64 part + 8 c ..
            const float f = scale[r];
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = x[r][64 * part + 8 * c + e] * f;
            hi = tile + part * 16384 + r * 128 + swz(r, c) * 16;
            lo = D < 64 ? tile + r * 128 + swz(r, c + CHUNKS) * 16 : hi + 8192;
        }
        halfx8 wh, wl;
        split8(w, 1.0f, wh, wl);
        *reinterpret_cast<halfx8 *>(hi) = wh;
        *reinterpret_cast<halfx8 *>(lo) = wl;
    }
}

// what load instructions read from p on, zeros from its `bytes` on
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_from(const float *p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(p), 0, bytes, 0x00027000);
}

// grid: a workgroup for each unit, and p.runs; 64 WAVES threads, 32 columns a wavefront.
//
// A unit is (heads that share keys, table, tile of 32 WAVES columns, each a query and one of those heads); its blocks are the 64-row
// tiles that its queries see. 50 tables of 250 to 500 rows, in order, 16 heads of 32 over 4: 63 us, with a head a unit 70; 95 of 11
// rows, 8 heads of 128 over one, 20 and 35. p.runs workgroups are what the card holds at once. As many units of each head as make whole
// rounds of them are a workgroup's each (all of them where units are short); the blocks of the others, one unit after the other, are
// cut into equal runs, which end together, for tables of any lengths, causal or not. A run that is not a whole unit leaves a state for
// k_packed_join. One table of 10,000 rows and 8 heads, 632 units on 512 places: two rounds 720 us, everything in runs 840 (workgroups
// of an XCD then read different keys at a time, more than its cache holds; whole units read the same ones), as it is 619 (564 with what
// follows).
//
// S^T = K Q^T and O^T += V^T P^T by v_mfma_f32_32x32x16_f16, three products of halves a term, the keys in sigma32 order so that
// the weights of a block are the values' operand where they stand. Tiles come by DMA into two LDS buffers each for keys and values,
// a block ahead (one each where two would leave one workgroup of four wavefronts a compute unit), or are made here from rows read a
// block ahead (few_readers). The softmax is in log2 units against a reference that is raised when a block passes it by more than 3;
// weights stay below 2^15. A column's sums of values are held in units of their own, 2^(unit - 12): the unit is raised, as the
// reference is, when a block's largest weight times its values' power of two passes it by more than 3, so that what a column does not
// see, or gives no weight, takes none of its precision; the block's weights are taken smaller or larger by the difference.
//
// In a long table the matrix pipes are busy 60% of the time and the vector pipes 49%, hardly ever at once: 10,000 rows, 8 heads of 64,
// 564 us or 1,089 TFLOP/s of the three products, what a large fp16 product reaches here (1,109). Short tables are bound by their start
// (plan, rows and queries on their way: about 9 us) and by memory. Columns' own units cost a long table 1% (558 us without), looking
// for rows that lie apart a short one in order 3% (200 of 50 to 100 rows 58 and 60 us; heads of 32 38 and 41, registers).
// Heads of up to 32 keep to the registers of three workgroups of four wavefronts a compute unit (10,000 rows in order 209 us, at two
// 226), or two of eight (10,000 rows 350, at one 361).
template <int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, D == 32 ? (WAVES == 4 ? 3 : 4) : 2) void k_packed(Packed p) {
    constexpr int QT = 32 * WAVES, HALF = HALF_BYTES<D>, DC = D / 16, DB = D / 32, BEGIN = BEGIN_OF<D>;
    constexpr bool DIRECT = WAVES == 4 && D <= 64, SINGLE = WAVES == 4 && D == 128;
    __shared__ __align__(16) uint8_t kt0[HALF], kt1[SINGLE ? 16 : HALF], vt0[HALF], vt1[SINGLE ? 16 : HALF];
    __shared__ int4 rows_here[64];
    __shared__ uint32_t first_here[64];
    __shared__ floatx4 most_here[4];
    __shared__ __align__(8) uint8_t odd_here[64][8];
    __shared__ uint32_t rows_most[DIRECT ? KB : 1];  // values'
    __shared__ __align__(8) int8_t shifts_here[2][DIRECT ? KB : 8];  // the rows' own powers of two, keys' and values'
    const int thread = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(thread >> 6);

    // the first 64 tables, one a lane, read beside the plan
    const int t64 = min(thread & 63, p.tables - 1);
    const uint32_t tiles64 = p.tile_sums[t64 + 1], blocks64 = p.block_sums[t64 + 1];
    {
        int qa = 0, ka = 0;
        const int n_q = rows_of(p.qo, t64, p.nq, qa), n_t = rows_of(p.ko, t64, p.nkv, ka);
        first_here[thread & 63] = p.first[t64];  // every wavefront writes the same and reads what it wrote
        rows_here[thread & 63] = make_int4(qa, n_q, ka, n_t);
    }
    const PackedPlan plan = *p.plan;
    const int heads = p.heads >> p.log_share, log_queries = (WAVES == 8 ? 8 : 7) - p.log_share;
    // Workgroup i runs on XCD i % 8. So many XCDs as a head has, where there are fewer heads than XCDs, take turns at its units or runs
    // (else an XCD has whole heads): an XCD reads few heads' keys, and all have long and short units alike.
    const int log_turns = 3 - min(3, __builtin_ctz(heads)), turns = 1 << log_turns, sets = 8 >> log_turns;
    const uint32_t set_units = plan.own * (uint32_t)(heads / sets), set_runs = (plan.runs + sets - 1) / sets;
    const uint32_t share = (set_units + turns - 1) >> log_turns;
    const bool whole = blockIdx.x < 8 * share;
    const uint32_t idx = whole ? blockIdx.x : blockIdx.x - 8 * share, xcd = idx & 7, size = whole ? set_units : set_runs;
    const uint32_t in_set = (idx >> 3 << log_turns) + (xcd & (turns - 1)), run = (xcd >> log_turns) * size + in_set;
    const uint32_t total = plan.rest * heads;
    if (in_set >= size || (!whole && run >= plan.runs)) return;
    const uint32_t mine = whole ? run : run * plan.per, end = whole ? run + 1 : min(total, mine + plan.per);
    const uint32_t a_head = whole ? plan.own : plan.rest;
    const uint32_t *sums = whole ? p.tile_sums : p.block_sums;
    const uint32_t sum64 = whole ? tiles64 : blocks64;

    for (uint32_t at = mine; at < end;) {
    if (at != mine) __syncthreads();  // the unit before's buffers are no longer read
    int tid = thread;
    asm volatile("" : "+v"(tid));  // what follows from it is formed for each unit, not held for all
    const int lane = tid & 63, r32 = lane & 31, g = lane >> 5;
    const uint32_t shared = at / a_head, in_head = at - shared * a_head + (whole ? 0 : plan.own_blocks);
    const int h0 = (int)(shared << p.log_share), hk = h0 / (p.heads / p.kv_heads);
    // the table: so many end at or before here (those without queries among them)
    int t = __popcll(__ballot(lane < p.tables - 1 && sum64 <= in_head));
    for (int t0 = 64; t == t0 && t0 < p.tables - 1; t0 += 64)
        t += __popcll(__ballot(t0 + lane < p.tables - 1 && sums[t0 + lane + 1] <= in_head));
    t = __builtin_amdgcn_readfirstlane(t);
    int qa, ka, n_q, n_t;
    uint32_t first, local;
    if (t < 64) {
        const int4 rows = rows_here[t];
        qa = __builtin_amdgcn_readfirstlane(rows.x);
        n_q = __builtin_amdgcn_readfirstlane(rows.y);
        ka = __builtin_amdgcn_readfirstlane(rows.z);
        n_t = __builtin_amdgcn_readfirstlane(rows.w);
        first = __builtin_amdgcn_readfirstlane(first_here[t]);
        local = in_head - (t ? __builtin_amdgcn_readlane(sum64, t - 1) : 0);
    } else {
        n_q = rows_of(p.qo, t, p.nq, qa);
        n_t = rows_of(p.ko, t, p.nkv, ka);
        first = p.first[t];
        local = in_head - sums[t];
    }
    const int n_k = first != NO_ROOM ? n_t : 0;
    const Tiles<BEGIN> ts{n_q, n_k, p.causal, log_queries};
    int tile = 0;
    if (whole) {
        tile = (int)local;
    } else if (!p.causal) {
        tile = (int)(local / (uint32_t)(ts.all() + BEGIN));
    } else {
        int hi = ts.count();
        while (hi - tile > 1) {
            const int mid = (tile + hi) >> 1;
            if (ts.before(mid) <= local)
                tile = mid;
            else
                hi = mid;
        }
    }
    const int nb = ts.blocks(tile), b0 = whole ? 0 : (int)(local - (uint32_t)ts.before(tile));
    const int b1 = whole ? nb + BEGIN : min(nb + BEGIN, b0 + (int)(end - at));
    const bool done = b0 == 0 && b1 == nb + BEGIN;
    const size_t slot = 2 * (size_t)run + (at == mine ? 0 : 1);
    const uint32_t last_run = done ? run : (at - b0 + nb + BEGIN - 1) / plan.per;
    at += whole ? 1 : b1 - b0;
    // a column is a query and one of the heads that share its keys; w0, w1 the wavefront's first and last query
    const int row0 = ts.first_query(tile), w0 = row0 + ((32 * wave) >> p.log_share), w1 = row0 + ((32 * wave + 31) >> p.log_share);
    const int qi = row0 + ((32 * wave + r32) >> p.log_share), h = h0 + ((32 * wave + r32) & ((1 << p.log_share) - 1));
    auto limit_of = [&](int i) { return p.causal ? max(0, n_k - (n_q - 1 - i)) : n_k; };
    const bool live = qi < n_q;
    if (!whole && at >= end && tid == 0)
        p.cut[run] = b0 == 0 && !done ? CutUnit{(uint32_t)slot, last_run, qa + row0, min(QT >> p.log_share, n_q - row0) << p.log_share, h0}
                                      : CutUnit{};
    if (b0 > 0 && b0 >= nb) {  // behind the unit's blocks
        if (g == 0) p.part_ml[slot * QT + 32 * wave + r32] = make_float2(-INFINITY, 0.0f);
        continue;
    }
    // the rows that this lane's query sees, and those that all and any of the wavefront's see
    const int limit = live ? limit_of(qi) : n_k, least = w0 < n_q ? limit_of(w0) : n_k;
    const int most_seen = w0 < n_q ? limit_of(min(w1, n_q - 1)) : 0;
    const int kb0 = b0, kb1 = min(b1, nb);
    const uint8_t *tiles = p.tiles + ((size_t)first * p.kv_heads + hk) * (2 * HALF);
    const int *shifts = p.shifts + 2 * ((size_t)first * p.kv_heads + hk);
    const size_t kb_bytes = (size_t)p.kv_heads * (2 * HALF);
    // half a tile, 16 bytes a lane: in copy i wavefront w fills the 1 KB at 1024 (WAVES i + w), from a scalar address on
    const uint32_t lane16 = 16 * lane;
    auto copy = [&](const uint8_t *src, uint8_t *dst) {
#pragma unroll
        for (int i = 0; i < HALF / (1024 * WAVES); i++)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint4 *>(src + 1024 * (WAVES * i + wave) + lane16),
                                             dst + 1024 * (WAVES * i + wave), 16, 0, 0);
    };
    // the powers of two of 64 blocks, one a lane
    int shifts_at = kb0, key_shifts = 0, value_shifts = 0;
    auto hold_shifts = [&] {
        const int *at = shifts + 2 * (size_t)min(shifts_at + lane, kb1 - 1) * p.kv_heads;
        key_shifts = at[0];
        value_shifts = at[1];
    };
    const bool direct = DIRECT && few_readers(p, n_q);
    // direct: a block's rows in registers, the next one's while a block is worked on: 8 coordinates of a key, 8 keys' value of a
    // coordinate a lane
    constexpr int HELD = DIRECT ? D / 32 : 1, CHUNKS = D < 64 ? D / 8 : 8;
    u32x4 key_rows[HELD][2];
    uint32_t value_rows[HELD][8];
    const uint32_t ld4 = 4 * (uint32_t)p.kv_ld, past = 0x80000000u;  // past: behind all of a block's rows
    const uint32_t key_at = 8 * (tid % CHUNKS) < p.hd ? (tid / CHUNKS) * ld4 + 32 * (tid % CHUNKS) : past;
    const uint32_t value_at = tid % D < p.hd ? 8 * (tid / D) * ld4 + 4 * (tid % D) : past;
    auto load_rows = [&](int kb) __attribute__((always_inline)) {
        // rows behind the table's and coordinates behind the head's are zeros
        const size_t at = (size_t)(ka + kb * KB) * p.kv_ld + (size_t)hk * p.hd;
        const uint32_t bytes = (uint32_t)(min(n_k - kb * KB, KB) - 1) * ld4 + 4 * p.hd;
        const auto ks = rows_from(p.k + at, bytes), vs = rows_from(p.v + at, bytes);
#pragma unroll
        for (int i = 0; i < HELD; i++) {
#pragma unroll
            for (int j = 0; j < 2; j++)
                key_rows[i][j] = __builtin_amdgcn_raw_buffer_load_b128(ks, key_at + i * (256 / CHUNKS) * ld4 + 16 * j, 0, 0);
#pragma unroll
            for (int e = 0; e < 8; e++)
                value_rows[i][e] = __builtin_amdgcn_raw_buffer_load_b32(vs, value_at + (i * 8 * (256 / D) + e) * ld4, 0, 0);
        }
    };
    if (kb0 < kb1) {
        if (direct) {
            load_rows(kb0);
        } else {
            hold_shifts();
            copy(tiles + kb0 * kb_bytes, kt0);
            copy(tiles + kb0 * kb_bytes + HALF, vt0);
        }
    }
    // this lane's query coordinates 16 dc + 8 g + t, at a maximum near 2^14, split
    halfx8 qh[DC], ql[DC];
    float to_log2;
    {
        float qv[DC][8], most = 0.0f;
        const float *src = p.q + (size_t)(qa + (live ? qi : 0)) * p.q_ld + (size_t)h * p.hd;
#pragma unroll
        for (int dc = 0; dc < DC; dc++) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const floatx4 w = live && 16 * dc < p.hd ? (floatx4) * reinterpret_cast<const floatx4u *>(src + 16 * dc + 8 * g + 4 * j)
                                                         : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float f = w[e];
                    qv[dc][4 * j + e] = f;
                    most = fmaxf(most, __uint_as_float(finite_bits(__float_as_uint(f))));
                }
            }
        }
        most = half_max(most);
        const int eq = shift_below(most);
        const float f = pow2(eq);
#pragma unroll
        for (int dc = 0; dc < DC; dc++) split8(qv[dc], f, qh[dc], ql[dc]);
        to_log2 = LOG2E * pow2(-eq);
    }
    // where a lane's operands begin in a buffer: key row sigma(r32), value row r32, and the four chunks of each; rows 32 further on are
    // in the same chunks
    const int krow = sigma32(r32);
    int kat[4], vat[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        kat[i] = krow * 128 + swz(krow, 2 * i + g) * 16;
        vat[i] = r32 * 128 + swz(r32, 2 * i + g) * 16;
    }
    // whole numbers: the weights' sum is in units of 2^(ref - 12), the values' sums in 2^(unit - 12)
    float ref = -INFINITY, unit = -INFINITY, l = 0.0f;
    floatx16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[db][v] = 0.0f;
    floatx16 zero;
#pragma unroll
    for (int v = 0; v < 16; v++) zero[v] = 0.0f;

    // Block kb in the buffers kc and vc, with its powers of two as k_packed_tiles leaves them.
    // With is_apart rows may have powers of two of their own.
    auto block_of = [&](auto here, auto is_apart, const uint8_t *kc, const uint8_t *vc, int kb, int eko,
                        int evo) __attribute__((always_inline)) {
        constexpr bool apart = decltype(is_apart)::value;
        if (kb * KB >= most_seen) return;  // a wavefront whose queries see none of it: its part of the copies is all it does
        const int eb = evo >> 2;
        auto in_log2 = [&](int shift) { return fminf(fmaxf(to_log2 * pow2(-shift), 0x1p-126f), 0x1p126f); };
        const float f = in_log2(eko >> 2);  // from raw scores to log2 units
        floatx16 sc[2];
#pragma unroll
        for (int dc = 0; dc < DC; dc++)
#pragma unroll
            for (int kh = 0; kh < 2; kh++) {
                const uint8_t *at = kc + (dc >> 2) * 16384 + kh * 4096 + kat[dc & 3];
                const halfx8 hi = *reinterpret_cast<const halfx8 *>(at);
                const halfx8 lo = *reinterpret_cast<const halfx8 *>(D < 64 ? kc + kh * 4096 + kat[dc + 2] : at + 8192);
                sc[kh] = mfma16(hi, qh[dc], dc == 0 ? zero : sc[kh]);
                sc[kh] = mfma16(hi, ql[dc], sc[kh]);
                sc[kh] = mfma16(lo, qh[dc], sc[kh]);
            }
        if ((kb + 1) * KB > least) {
            const int lim = limit - kb * KB - 8 * g;  // accumulator v of half kh is seen while 32 kh + 16 (v / 8) + v % 8 < lim
#pragma unroll
            for (int kh = 0; kh < 2; kh++)
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (32 * kh + 16 * (v >> 3) + (v & 7) >= lim) sc[kh][v] = -INFINITY;
        }
        float mb = -INFINITY;
#pragma unroll
        for (int kh = 0; kh < 2; kh++)
#pragma unroll
            for (int v = 0; v < 16; v++) mb = fmaxf(mb, sc[kh][v]);
        mb = half_max(mb) * f;
        float top = mb - (float)eb;  // of weights times values, in log2
        // eight rows' own powers of two, keys' or values', from row 32 kh + 16 hh + 8 g on
        auto rows_shifts = [&](int which, int kh, int hh) {
            const int8_t *at = decltype(here)::value ? shifts_here[which]
                                                     : p.row_shifts + (2 * (((size_t)first + kb) * p.kv_heads + hk) + which) * KB;
            return *reinterpret_cast<const uint2 *>(at + 32 * kh + 16 * hh + 8 * g);
        };
        auto byte_of = [](uint2 w, int e) { return (int)(int8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3))); };
        if constexpr (apart) {  // scores in log2, and what they come to with their values
            mb = top = -INFINITY;
#pragma unroll
            for (int kh = 0; kh < 2; kh++)
#pragma unroll
                for (int hh = 0; hh < 2; hh++) {
                    __builtin_amdgcn_sched_barrier(0);  // eight rows at a time: there are no registers for more
                    const uint2 ks = rows_shifts(0, kh, hh), vs = rows_shifts(1, kh, hh);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float x = sc[kh][8 * hh + e] * in_log2(byte_of(ks, e));
                        sc[kh][8 * hh + e] = x;
                        mb = fmaxf(mb, x);
                        top = fmaxf(top, x - (float)byte_of(vs, e));
                    }
                }
            mb = half_max(mb);
            top = half_max(top);
        }
        const bool grow = mb > ref + 3.0f, grow_unit = top > unit + 3.0f;
        if (__any(grow || grow_unit)) {
            const float nref = grow ? floorf(mb) : ref, nunit = grow_unit ? floorf(top) : unit;
            l *= grow ? pow2((int)fmaxf(ref - nref, -200.0f)) : 1.0f;
            const float beta = grow_unit ? pow2((int)fmaxf(unit - nunit, -200.0f)) : 1.0f;
#pragma unroll
            for (int db = 0; db < DB; db++) acc[db] *= beta;
            ref = nref;
            unit = nunit;
        }
        // what the block's weights are taken larger by (below 2^-60 they are zeros as halves; their sum is taken of them)
        const float less = ref == -INFINITY ? 0.0f : apart ? ref - unit : fmaxf(ref - unit - (float)eb, -60.0f);
        const float off_sum = ref == -INFINITY ? 0.0f : 12.0f - ref, off = off_sum + less;
        float ps = 0.0f;
#pragma unroll
        for (int kh = 0; kh < 2; kh++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
                u32x4 hw, lw;
                const uint2 vs = apart ? rows_shifts(1, kh, hh) : make_uint2(0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x0 = sc[kh][8 * hh + 2 * i], x1 = sc[kh][8 * hh + 2 * i + 1];
                    float p0, p1;
                    if constexpr (apart) {  // the weights for their sum, and times the values' powers of two
                        ps += exp2_hw(x0 + off_sum) + exp2_hw(x1 + off_sum);
                        p0 = exp2_hw(x0 - (float)byte_of(vs, 2 * i) + off);
                        p1 = exp2_hw(x1 - (float)byte_of(vs, 2 * i + 1) + off);
                    } else {
                        p0 = exp2_hw(fmaf(x0, f, off));
                        p1 = exp2_hw(fmaf(x1, f, off));
                        ps += p0 + p1;
                    }
                    uint32_t hi, lo;
                    split2(p0, p1, hi, lo);
                    hw[i] = hi;
                    lw[i] = lo;
                }
                const halfx8 ph = __builtin_bit_cast(halfx8, hw), pl = __builtin_bit_cast(halfx8, lw);
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    const uint8_t *at = vc + db * 4096 + vat[2 * kh + hh];
                    const halfx8 hi = *reinterpret_cast<const halfx8 *>(at), lo = *reinterpret_cast<const halfx8 *>(at + D * 128);
                    acc[db] = mfma16(hi, ph, acc[db]);
                    acc[db] = mfma16(hi, pl, acc[db]);
                    acc[db] = mfma16(lo, ph, acc[db]);
                }
            }
        l = apart ? l + ps : fmaf(ps, pow2(-(int)less), l);
        if (evo & 1) {  // values that are not finite, zeros in the tile: what sees one is no number
            const int left = limit - kb * KB;
            const uint64_t sees = left >= 64 ? ~uint64_t(0) : (left > 0 ? (uint64_t(1) << left) - 1 : 0);
            const uint64_t *odd;
            if constexpr (decltype(here)::value)
                odd = reinterpret_cast<const uint64_t *>(odd_here);
            else
                odd = p.odd + (((size_t)first + kb) * p.kv_heads + hk) * D;
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (odd[32 * db + 8 * (v >> 2) + 4 * g + (v & 3)] & sees) acc[db][v] = NAN;
        }
    };
    // The powers of two of block kb, and whether one serves all of its rows.
    int eko = 0, evo = 0;
    auto even = [&](int kb) {
        if (kb >= shifts_at + 64) {
            shifts_at += 64;
            hold_shifts();
        }
        eko = __builtin_amdgcn_readlane(key_shifts, kb - shifts_at);
        evo = __builtin_amdgcn_readlane(value_shifts, kb - shifts_at);
        return !((eko | evo) & 2);
    };
    // Block kb from the buffers kc and vc, the next one on its way into kn and vn: four arrays, so that the compiler sees that it need
    // not wait for the copies before it reads.
    auto step = [&](const uint8_t *kc, const uint8_t *vc, uint8_t *kn, uint8_t *vn, int kb, int eko,
                    int evo) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0);  // this wavefront's copies of block kb have landed
        __syncthreads();                // everyone's have, and block kb - 1's buffers are no longer read
        if (kb + 1 < kb1) {
            copy(tiles + (kb + 1) * kb_bytes, kn);
            copy(tiles + (kb + 1) * kb_bytes + HALF, vn);
        }
        block_of(Flag<false>{}, Flag<false>{}, kc, vc, kb, eko, evo);
    };
    int kb = kb0;
    if (direct) {
        if constexpr (DIRECT) {
            // the rows in registers as halves in the buffers, with these powers of two
            auto split_rows = [&](const float (&fk)[HELD], float fv, bool odd) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < HELD; i++) {
                    const int u = tid + 256 * i, c = u % CHUNKS, r = u / CHUNKS, dim = u % D, kc = u / D;
                    float w[8];
                    halfx8 wh, wl;
#pragma unroll
                    for (int e = 0; e < 8; e++) w[e] = __uint_as_float(key_rows[i][e >> 2][e & 3]);
                    split8(w, fk[i], wh, wl);
                    *reinterpret_cast<halfx8 *>(kt0 + r * 128 + swz(r, c) * 16) = wh;
                    *reinterpret_cast<halfx8 *>(kt0 + r * 128 + (D < 64 ? swz(r, c + CHUNKS) * 16 : 8192 + swz(r, c) * 16)) = wl;
                    uint32_t bits = 0;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        w[e] = __uint_as_float(value_rows[i][e]);
                        if (odd && (value_rows[i][e] & 0x7fffffffu) >= 0x7f800000u) {
                            bits |= 1u << e;
                            w[e] = 0.0f;
                        }
                    }
                    if (odd) odd_here[dim][kc] = (uint8_t)bits;
                    split8(w, fv, wh, wl);
                    *reinterpret_cast<halfx8 *>(vt0 + dim * 128 + swz(dim, kc) * 16) = wh;
                    *reinterpret_cast<halfx8 *>(vt0 + D * 128 + dim * 128 + swz(dim, kc) * 16) = wl;
                }
            };
            for (; kb < kb1; kb++) {
                uint32_t big_k = 0, big_v = 0;
#pragma unroll
                for (int i = 0; i < HELD; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        big_k = max(big_k, key_rows[i][e >> 2][e & 3] & 0x7fffffffu);
                        big_v = max(big_v, value_rows[i][e] & 0x7fffffffu);
                    }
                const bool any = __any(big_v >= 0x7f800000u);
                if (__any(max(big_k, big_v) >= 0x7f800000u)) {  // of the finite ones, then
                    big_k = big_v = 0;
#pragma unroll
                    for (int i = 0; i < HELD; i++)
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            big_k = max(big_k, finite_bits(key_rows[i][e >> 2][e & 3]));
                            big_v = max(big_v, finite_bits(value_rows[i][e]));
                        }
                }
                const float most_k = wave_max(__uint_as_float(big_k)), most_v = wave_max(__uint_as_float(big_v));
                // Where a query of the tile does not see all of the block: the least of its rows by parts that quads of lanes have, four
                // coordinates of a value, 32 of a key (a row of parts of several sizes then merely has its own power of two). Less one as
                // an int, so that zeros are not the least.
                uint32_t least_k = 0x7f7fffffu, least_v = 0x7f7fffffu;
                if ((kb + 1) * KB > limit_of(row0)) {
#pragma unroll
                    for (int i = 0; i < HELD; i++) {
                        float m = 0.0f;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const uint32_t w = key_rows[i][e >> 2][e & 3];
                            m = fmaxf(m, fabsf(__uint_as_float(w)));
                            least_v = min(least_v, __float_as_uint(lanes_max<4>(fabsf(__uint_as_float(value_rows[i][e])))) - 1);
                        }
                        least_k = min(least_k, __float_as_uint(lanes_max<4>(m)) - 1);
                    }
                    least_k = __float_as_uint(-wave_max(-__uint_as_float(least_k)));
                    least_v = __float_as_uint(-wave_max(-__uint_as_float(least_v)));
                    if (any) least_v = 0;
                }
                if (lane == 0)
                    most_here[wave] = floatx4{any ? -most_k : most_k, most_v, __uint_as_float(least_k), __uint_as_float(least_v)};
                __syncthreads();  // everyone's maxima are there, and block kb - 1's buffers are no longer read
                floatx4 m = {0.0f, 0.0f, INFINITY, INFINITY};
                bool odd = false;
#pragma unroll
                for (int w = 0; w < WAVES; w++) {
                    const floatx4 o = most_here[w];
                    odd = odd || __builtin_signbitf(o[0]);
                    m = floatx4{fmaxf(m[0], fabsf(o[0])), fmaxf(m[1], o[1]), fminf(m[2], o[2]), fminf(m[3], o[3])};
                }
                if (__builtin_amdgcn_readfirstlane(rows_apart(m[2], m[0]) || rows_apart(m[3], m[1]))) break;
                const int ek = __builtin_amdgcn_readfirstlane(shift_below(m[0]));
                const int ev = __builtin_amdgcn_readfirstlane(shift_below(m[1]));
                odd = __builtin_amdgcn_readfirstlane(odd);
                float fk[HELD];
#pragma unroll
                for (int i = 0; i < HELD; i++) fk[i] = pow2(ek);
                split_rows(fk, pow2(ev), odd);
                if (kb + 1 < kb1) load_rows(kb + 1);
                __syncthreads();
                block_of(Flag<true>{}, Flag<false>{}, kt0, vt0, kb, 4 * ek, 4 * ev + (odd ? 1 : 0));
            }
            // from the first block whose rows lie apart on: a power of two for each row
            for (; kb < kb1; kb++) {
                __syncthreads();  // the buffers are no longer read
                if (tid < KB) rows_most[tid] = 0;
                if (tid == 0) most_here[0][2] = 0.0f;
                __syncthreads();
                float fk[HELD];
                uint32_t raw_v = 0;
#pragma unroll
                for (int i = 0; i < HELD; i++) {
                    const int u = tid + 256 * i;
                    uint32_t big = 0;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        big = max(big, finite_bits(key_rows[i][e >> 2][e & 3]));
                        raw_v = max(raw_v, value_rows[i][e] & 0x7fffffffu);
                        atomicMax(&rows_most[8 * (u / D) + e], finite_bits(value_rows[i][e]));
                    }
                    const int shift = shift_below(lanes_max<CHUNKS>(__uint_as_float(big)));
                    fk[i] = pow2(shift);
                    if (u % CHUNKS == 0) shifts_here[0][u / CHUNKS] = (int8_t)shift;
                }
                if (raw_v >= 0x7f800000u) most_here[0][2] = 1.0f;
                __syncthreads();
                if (tid < KB) shifts_here[1][tid] = (int8_t)shift_below(__uint_as_float(rows_most[tid]));
                const bool odd = __builtin_amdgcn_readfirstlane(most_here[0][2] != 0.0f);
#pragma unroll
                for (int i = 0; i < HELD; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        __builtin_amdgcn_sched_barrier(0);
                        const float most = __uint_as_float(rows_most[8 * ((tid + 256 * i) / D) + e]);
                        value_rows[i][e] = __float_as_uint(__uint_as_float(value_rows[i][e]) * pow2(shift_below(most)));
                    }
                split_rows(fk, 1.0f, odd);
                if (kb + 1 < kb1) load_rows(kb + 1);
                __syncthreads();
                block_of(Flag<true>{}, Flag<true>{}, kt0, vt0, kb, 2, 2 + (odd ? 1 : 0));
            }
        }
    } else {
        if constexpr (SINGLE) {
            for (; kb < kb1 && even(kb); kb++) {
                __builtin_amdgcn_s_waitcnt(0);  // as in step
                __syncthreads();
                block_of(Flag<false>{}, Flag<false>{}, kt0, vt0, kb, eko, evo);
                if (kb + 1 < kb1) {
                    __syncthreads();  // the buffers are no longer read; the compute unit's other workgroup works meanwhile
                    copy(tiles + (kb + 1) * kb_bytes, kt0);
                    copy(tiles + (kb + 1) * kb_bytes + HALF, vt0);
                }
            }
        } else {
            for (; kb + 1 < kb1 && even(kb); kb += 2) {  // two steps a turn: the buffers' places are constants
                const int eko0 = eko, evo0 = evo;
                if (!even(kb + 1)) break;
                step(kt0, vt0, kt1, vt1, kb, eko0, evo0);
                step(kt1, vt1, kt0, vt0, kb + 1, eko, evo);
            }
            if (kb + 1 == kb1 && even(kb)) {
                step(kt0, vt0, kt1, vt1, kb, eko, evo);
                kb++;
            }
        }
        // from the first block whose rows lie apart on, a block after the other
        for (; kb < kb1; kb++) {
            even(kb);
            __builtin_amdgcn_s_waitcnt(0);  // what is on its way has landed
            __syncthreads();                // and is no longer read
            copy(tiles + kb * kb_bytes, kt0);
            copy(tiles + kb * kb_bytes + HALF, vt0);
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            block_of(Flag<false>{}, Flag<true>{}, kt0, vt0, kb, eko, evo);
        }
    }
    l = half_sum(l);  // lanes l and l ^ 32 have the same queries' sums over different keys
    const float inv = l > 0.0f ? 1.0f / l : l;  // 0 and NaN stay
    const float back = ref == -INFINITY ? 1.0f : pow2((int)(unit - ref));
    if (!done || live) {
        float *dst = done ? p.out + ((size_t)(qa + qi) * p.heads + h) * p.hd : p.part_o + (slot * QT + 32 * wave + r32) * p.hd;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int v4 = 0; v4 < 4; v4++) {
                const int dim = 32 * db + 8 * v4 + 4 * g;
                if (dim < p.hd) {
                    floatx4 o;
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = acc[db][4 * v4 + e] * inv * back;
                    *reinterpret_cast<floatx4u *>(dst + dim) = o;
                }
            }
        if (!done && g == 0) p.part_ml[slot * QT + 32 * wave + r32] = make_float2(ref, l);
    }
    }
}

// grid (runs, tiles' queries / 16); 256 threads: the states that runs left of a unit's sixteen columns, together: sixteen lanes a
// column, four of each 64 coordinates a lane. Bound by bytes where all is in runs: three tables of up to 2,500 rows, heads of 128, 13 us
// for up to 64 MB of states.
template <int C, int QT>
__global__ __launch_bounds__(256) void k_packed_join(Packed p) {
    constexpr int AHEAD = 4;
    if (blockIdx.x >= p.plan->runs) return;
    const CutUnit unit = p.cut[blockIdx.x];
    const int r = 16 * blockIdx.y + (threadIdx.x >> 4), dim = 4 * (threadIdx.x & 15);
    if (r >= unit.live) return;
    float M = -INFINITY, L = 0.0f;
    floatx4 o[C];
#pragma unroll
    for (int c = 0; c < C; c++) o[c] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t e = blockIdx.x; e <= unit.last_run; e += AHEAD) {
        float2 ml[AHEAD];
        floatx4 x[AHEAD][C];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            // past the last: the last again, without weight
            const uint32_t run = min(e + j, unit.last_run);
            const size_t at = (size_t)(run == blockIdx.x ? unit.slot : 2 * run) * QT + r;
            ml[j] = p.part_ml[at];
#pragma unroll
            for (int c = 0; c < C; c++)
                x[j][c] = *reinterpret_cast<const floatx4 *>(p.part_o + at * p.hd + (64 * c + dim < p.hd ? 64 * c + dim : 0));
            if (e + j > unit.last_run) ml[j] = make_float2(-INFINITY, 0.0f);
        }
        float top = M;
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
            if (ml[j].y > 0.0f) top = fmaxf(top, ml[j].x);
        // shares of the sum so far, so that no value is multiplied by more than 1
        const float old = M == -INFINITY ? L : L * exp2_hw(M - top);  // nothing yet, or NaN
        float f[AHEAD];
        L = old;
        M = top;
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            f[j] = ml[j].y > 0.0f ? ml[j].y * exp2_hw(ml[j].x - M) : ml[j].y;
            L += f[j];
        }
        const float inv = L > 0.0f ? 1.0f / L : L;
#pragma unroll
        for (int c = 0; c < C; c++) o[c] *= old * inv;
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            if (ml[j].y == 0.0f) continue;
#pragma unroll
            for (int c = 0; c < C; c++) o[c] += f[j] * inv * x[j][c];
        }
    }
#pragma unroll
    for (int c = 0; c < C; c++)
        if (64 * c + dim < p.hd)
            *reinterpret_cast<floatx4u *>(p.out + ((size_t)(unit.row + (r >> p.log_share)) * p.heads + unit.head +
                                                   (r & ((1 << p.log_share) - 1))) * p.hd + 64 * c + dim) = o[c];
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// Wavefronts a workgroup, runs, workgroups and the working memory's parts.
struct Plan {
    int waves, runs, blocks, d, log_share;  // d: the heads' width, padded
    bool direct;
    int64_t grid;
    size_t tiles, shifts, row_shifts, odd, tables, part_o, part_ml, cut;
    size_t bytes() const { return tiles + shifts + row_shifts + odd + 256 + 3 * tables + part_o + part_ml + cut; }
};

Plan plan(const PackedShape &a, size_t kv_ld) {
    Plan r;
    r.d = a.hd <= 32 ? 32 : a.hd <= 64 ? 64 : 128;
    // tiles of 256 queries where all of a long table's are full (10,000 rows 619 -> 598 us), else of 128 (five tables of up to 6,007 rows
    // in order 513, with 256 534). Heads over 64 wide: 256 at one workgroup a compute unit or, where tables are short, 128 at two,
    // with one buffer each for keys and values (100 of up to 300 rows, in order, 155 -> 139 us, 32 of up to 300 66 -> 54; 8,000
    // rows, 4 heads, 357 and 373).
    r.waves = (r.d == 128 ? a.nq / 2048 >= a.tables : !a.causal && a.nq / 4096 >= a.tables) ? 8 : 4;
    const int qt = 32 * r.waves;
    // heads that share their keys share tiles too, by powers of two up to a wavefront's columns
    r.log_share = 0;
    while (r.log_share < 5 && (a.heads / a.kv_heads) % (2 << r.log_share) == 0) r.log_share++;
    r.runs = r.waves == 8 ? 256 : r.d == 32 ? 768 : 512;  // what the card holds at once
    r.grid = (a.nq / (qt >> r.log_share) + (int64_t)std::min(a.tables, a.nq)) * (a.heads >> r.log_share) + r.runs + 32;
    r.direct = r.d <= 64 && r.waves == 4 && kv_ld < (size_t)1 << 22;  // a block's rows within 2^30 bytes
    // of tables that have tiles, the last one of each in part: where rows are also read where they stand, those of so many queries that
    // more than READERS tiles of queries read them
    const int readers = (a.heads / a.kv_heads) >> r.log_share;
    const int64_t least = r.direct ? (int64_t)(READERS / readers) * (qt >> r.log_share) + 1 : 1;
    const int64_t blocks = a.nkv / KB + std::min((int64_t)std::min(a.tables, a.nkv), r.direct ? a.nq / least : a.nkv);
    r.blocks = (int)blocks;
    const size_t halves = (size_t)blocks * a.kv_heads, places = 2 * (size_t)r.runs * qt;
    r.tiles = up256(halves * r.d * 512);
    r.shifts = up256(halves * 2 * sizeof(int));
    r.row_shifts = up256(halves * 2 * KB);
    r.odd = up256(halves * r.d * sizeof(uint64_t));
    r.tables = up256(((size_t)a.tables + 1) * sizeof(uint32_t));
    r.part_o = up256(places * a.hd * sizeof(float));
    r.part_ml = up256(places * sizeof(float2));
    r.cut = up256((size_t)r.runs * sizeof(CutUnit));
    return r;
}

template <int D, int WAVES>
void launch(hipStream_t s, const Packed &p, const Plan &r) {
    hipLaunchKernelGGL(k_packed_tiles<D>, dim3(std::max(r.blocks, 1), p.kv_heads, 2), dim3(256), 0, s, p);
    TAH_LAUNCHED();
    hipLaunchKernelGGL((k_packed<D, WAVES>), dim3((unsigned)r.grid), dim3(64 * WAVES), 0, s, p);
    TAH_LAUNCHED();
    hipLaunchKernelGGL((k_packed_join<(D + 63) / 64, 32 * WAVES>), dim3(r.runs, 2 * WAVES), dim3(256), 0, s, p);
    TAH_LAUNCHED();
}

}  // namespace

size_t packed_work_bytes(const PackedShape &a, size_t kv_ld) {
    const Plan r = plan(a, kv_ld);
    // a launch takes fewer than 2^32 threads; the tiles' has 256 a block of rows
    if ((uint64_t)r.grid * (64 * r.waves) >> 32 || r.blocks > 0x7FFFFF || a.nq > 0x7FFFFF00)
        throw ArgError{"attend_packed: more rows than a call takes: fewer tables a call"};
    return r.bytes();
}

void packed_attention(hipStream_t s, const PackedShape &a, const float *q, const float *k, const float *v, const int32_t *q_offsets,
                      const int32_t *kv_offsets, size_t q_ld, size_t kv_ld, float *out, void *work) {
    const Plan r = plan(a, kv_ld);
    uint8_t *at = static_cast<uint8_t *>(work);
    auto carve = [&](size_t bytes) {
        uint8_t *here = at;
        at += bytes;
        return here;
    };
    Packed p{q, k, v, q_offsets, kv_offsets, a.tables, a.nq, a.nkv, a.heads, a.kv_heads, a.hd, a.causal ? 1 : 0, q_ld, kv_ld, out};
    p.blocks = r.blocks;
    p.tiles = carve(r.tiles);
    p.shifts = reinterpret_cast<int *>(carve(r.shifts));
    p.row_shifts = reinterpret_cast<int8_t *>(carve(r.row_shifts));
    p.odd = reinterpret_cast<uint64_t *>(carve(r.odd));
    p.plan = reinterpret_cast<PackedPlan *>(carve(256));
    p.first = reinterpret_cast<uint32_t *>(carve(r.tables));
    p.tile_sums = reinterpret_cast<uint32_t *>(carve(r.tables));
    p.block_sums = reinterpret_cast<uint32_t *>(carve(r.tables));
    p.waves = r.waves;
    p.runs = r.runs;
    p.log_share = r.log_share;
    p.direct = r.direct;
    p.part_o = reinterpret_cast<float *>(carve(r.part_o));
    p.part_ml = reinterpret_cast<float2 *>(carve(r.part_ml));
    p.cut = reinterpret_cast<CutUnit *>(carve(r.cut));
    if (r.d == 128)
        r.waves == 8 ? launch<128, 8>(s, p, r) : launch<128, 4>(s, p, r);
    else if (r.d == 64)
        r.waves == 8 ? launch<64, 8>(s, p, r) : launch<64, 4>(s, p, r);
    else
        r.waves == 8 ? launch<32, 8>(s, p, r) : launch<32, 4>(s, p, r);
}

}  // namespace tah
