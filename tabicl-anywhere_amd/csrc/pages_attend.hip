// Attention of queries of many tables over their pages (tah_pages_attend): few queries a table, every key read once.
//
// A unit of work is (table, up to 16 CT columns, key/value head), a column being a query and one of the heads that share the
// key/value head; its keys go in blocks of 64. All units' blocks, one after the other, are cut into equal runs, one a wavefront,
// so tables of any lengths fill the card alike; a run that is not a whole unit leaves a state (maximum, sum, weighted values)
// that k_pages_join puts together with the unit's others.
#include "device_math.hpp"
#include "pages.hpp"

namespace tah {

namespace {

constexpr int WAVES = 4;
constexpr int MOST_WGS = (1 << 24) - 1;  // of 256 threads in a dimension of a launch, which takes fewer than 2^32 threads
// What beginning and ending a unit costs, in blocks: a unit counts as so many more than it has, so that wavefronts with several
// units get fewer of them. 24 tables of up to 6,001 rows 69, 62.5 and 62.4 us for 1, 2 and 4, 64 of up to 20,000 139.5, 140.8, 141.8.
constexpr int BEGIN = 2;

// What runs of blocks leave behind for the join: per slot [columns][hd] outputs and [columns] (maximum, sum); a wavefront has at
// most two units that are not whole, its first and its last: slots 2 w and 2 w + 1. Per query and head the unit's first block and
// the one behind its last, the blocks a wavefront, and the column (blocks a wavefront 0: the output is there).
struct Parts {
    float *o;
    float2 *ml;
    uint4 *units;
    uint32_t *plan;  // blocks a wavefront, blocks in all
};

// A table's queries (from `first`), rows, and blocks: in the chunk of 64 tables that a wavefront holds, one a lane
struct TableWork {
    int first, n, len;
    uint32_t nb, cost;
};

__device__ __forceinline__ TableWork table_work(const PageSet &p, const int32_t *lengths, const int32_t *offsets, int nq, int group,
                                                int columns, int keys, int t) {
    const int i = min(t, p.tables - 1), from = offsets[i], to = offsets[i + 1], told = lengths[i];
    const int a = min(max(from, 0), nq), b = min(max(to, a), nq);
    const long most = min((long)p.ld << p.log_rows, (long)0x7fffffff - 64);
    TableWork w;
    w.first = a;
    w.n = t < p.tables ? b - a : 0;
    w.len = (int)min((long)max(told, 0), most);
    w.nb = (w.len + keys - 1) / keys + BEGIN;
    w.cost = (uint32_t)((w.n * group + columns - 1) / columns) * p.heads * w.nb;
    return w;
}

// 16 (N 2) or 8 (N 1) stored numbers of a lane
template <int FMT, int N>
struct Raw {
    static constexpr int WORDS = 2 * N * page_width(FMT);
    uint32_t w[WORDS];
};

template <int FMT, int N>
__device__ __forceinline__ Raw<FMT, N> load_raw(const uint8_t *at) {
    Raw<FMT, N> r;
    if constexpr (Raw<FMT, N>::WORDS == 2) {
        const uint2 x = *reinterpret_cast<const uint2 *>(at);
        r.w[0] = x.x;
        r.w[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < Raw<FMT, N>::WORDS / 4; i++) {
            const uint4 x = reinterpret_cast<const uint4 *>(at)[i];
            r.w[4 * i] = x.x;
            r.w[4 * i + 1] = x.y;
            r.w[4 * i + 2] = x.z;
            r.w[4 * i + 3] = x.w;
        }
    }
    return r;
}

// bytes of a word, signed, as halves: 0x6400 | (b + 128) is 1024 + 128 + b in fp16, exact
__device__ __forceinline__ halfx2 half_bytes(uint32_t flipped, uint32_t sel) {
    return __builtin_bit_cast(halfx2, __builtin_amdgcn_perm(flipped, 0x64646464u, sel)) - halfx2{(_Float16)1152.0f, (_Float16)1152.0f};
}

// numbers 8 s .. 8 s + 7 as halves: exact in hi (i8); i16 as 256 (hi + lo), hi the high byte, lo the low one over 256: five
// instructions for two, where rounding to a half and the rest took eight; f32 times f in hi + lo
template <int FMT, int N>
__device__ __forceinline__ void to_halves(const Raw<FMT, N> &r, int s, float f, halfx8 &hi, halfx8 &lo) {
    if constexpr (FMT == TAH_KV_I8) {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t w = r.w[2 * s + i] ^ 0x80808080u;
            o[2 * i] = __builtin_bit_cast(uint32_t, half_bytes(w, 0x00050004u));
            o[2 * i + 1] = __builtin_bit_cast(uint32_t, half_bytes(w, 0x00070006u));
        }
        hi = __builtin_bit_cast(halfx8, o);
    } else if constexpr (FMT == TAH_KV_I16) {
        u32x4 a, b;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = r.w[4 * s + i] ^ 0x80008000u;
            a[i] = __builtin_bit_cast(uint32_t, half_bytes(w, 0x00070005u));
            const halfx2 low = __builtin_bit_cast(halfx2, __builtin_amdgcn_perm(w, 0x64646464u, 0x00060004u));
            const _Float16 part = (_Float16)0x1p-8f, back = (_Float16)-4.0f;
            b[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(low, halfx2{part, part}, halfx2{back, back}));
        }
        hi = __builtin_bit_cast(halfx8, a);
        lo = __builtin_bit_cast(halfx8, b);
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __uint_as_float(r.w[8 * s + i]);
        split8(v, f, hi, lo);
    }
}

__device__ __forceinline__ floatx4 mfma(halfx8 a, halfx8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// grid: any number of workgroups; WAVES wavefronts each.
//
// Products are 16 x 16 x 32 with the queries as columns: S = K Q^T for sets of 16 keys, then O^T += V^T P^T. Of a block's 32 KS
// keys a lane (lg = lane / 16) has N = 8 KS: keys N lg .. N lg + N - 1. Set (s, p)'s row r is key N (r / 4) + 8 s + 4 p + r % 4, so
// that the scores of sets (s, 0) and (s, 1) are the operand of the values' product s in place, N consecutive numbers of a
// coordinate are what a lane reads of the values, and a page of 16 rows or more holds all that a lane reads at once. Coordinates go
// likewise: step (c, ks) takes 64 c + 16 lg + 8 ks .. + 7.
//
// Numbers: ints go in as they are (i8 exact in one half, i16 in two bytes), the key's step multiplies its scores, the value's its
// weights; f32 goes in as two halves times the block's power of two. Queries and weights are two halves. So a term is two
// products (i8), three (f32) or four (i16: a low byte is 2^-8 of the largest number, so its product with a low half counts), for
// f32's error. Weights are held below 2^15 (their maximum raised by blocks that pass it by more than 2^3). A column's sums of values have a
// unit of their own, 2^(vunit - 12), raised when a block's largest weight times the largest step that the column sees passes it by as much,
// so that rows that it does not see, or gives no weight, take none of its precision. f32: where columns do not see
// the same rows of a block each row has a power of two of its own, as ints have their steps.
//
// Bound by bytes where tables are long: 64 of up to 20,000 rows, 8 heads of 64 in i8, one query each, 132 us of kernel at least (median
// 140) for 702 MB, 5.3 TB/s, what a large copy reaches (vector instructions issue in 53% of the cycles, matrix instructions in 14%). One
// table of 100,000 rows, 26 us, has 6.1 blocks a wavefront, in runs of 7: the start (lengths, plan, queries, the first keys and their
// steps, one after the other) is 8 us of it, all that 1,000 rows take. i16's four products of 16 columns twice and f32's splitting cost
// more than their bytes; columns past two sets read the keys again (nine queries of four heads: 36 columns, 1.4 times the bytes).
// Tried and slower: a block's keys and values read while the one before is worked on (141 -> 153 us, the compiler has no registers
// for both), three wavefronts a SIMD (176, spilling). Two sets of columns that share what is read: registers allow no third.
template <int FMT, int C, int CT, int KS>
__global__ __launch_bounds__(64 * WAVES, 2) void k_pages_attend(PageSet p, const int32_t *__restrict__ lengths,
                                                                const float *__restrict__ q, const int32_t *__restrict__ offsets,
                                                                int nq, int heads, int causal, size_t q_ld,
                                                                float *__restrict__ out, Parts parts, uint64_t most_blocks) {
    constexpr int W = page_width(FMT), COLS = 16 * CT, HD = 64 * C, M = 4 * C, N = 8 * KS, KEYS = 32 * KS;
    constexpr bool INTS = FMT != TAH_KV_F32, LO = FMT != TAH_KV_I8, BYTES = FMT == TAH_KV_I16;
    // more queries than 16 columns of 64 coordinates wait in LDS, each wavefront's own; the join's sums take their place
    constexpr bool WAIT = C * CT > 1;
    constexpr int QS = WAIT ? CT * C * 2 * 2 * 64 : 0;  // 16-byte words of a wavefront's
    __shared__ __align__(16) uint8_t store[WAVES * (QS * 16 > HD * 68 ? QS * 16 : HD * 68)];
    __shared__ float mref[WAVES][COLS], msum[WAVES][COLS];
    // f32, blocks that some columns see in part: the steps of the block's keys and values, each wavefront's own
    __shared__ __align__(16) float steps_here[WAVES][2][INTS ? 4 : KEYS];
    float (*macc)[HD][17] = reinterpret_cast<float (*)[HD][17]>(store);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int qi = lane & 15, lg = lane >> 4, group = heads / p.heads, hd = p.hd, P = p.rows;
    const uint32_t waves = gridDim.x * WAVES, me = blockIdx.x * WAVES + wave;

    // the plan: every wavefront adds up all tables' blocks and finds its own; a chunk of 64 tables, one a lane, is kept
    TableWork mine_of{};
    uint32_t sums = 0;          // blocks of the chunk's tables up to the lane's
    uint32_t chunk_before = 0;  // blocks before the chunk
    int chunk = 0;
    uint64_t all = 0;
    for (int t0 = 0; t0 < p.tables; t0 += 64) {
        mine_of = table_work(p, lengths, offsets, nq, group, COLS, KEYS, t0 + lane);
        sums = wave_scan(mine_of.cost);
        // in two halves of 16 bits, which 64 tables' sums do not overflow, whatever their offsets say
        const uint32_t low = wave_scan(mine_of.cost & 0xffffu), high = wave_scan(mine_of.cost >> 16);
        all += ((uint64_t)__builtin_amdgcn_readlane(high, 63) << 16) + __builtin_amdgcn_readlane(low, 63);
    }
    // offsets that fall may make more of the queries than there are: nothing is done then
    const uint32_t total = all <= most_blocks ? (uint32_t)all : 0;
    const uint32_t per = max(1u, (total + waves - 1) / waves);
    if (me == 0 && lane == 0) {
        parts.plan[0] = per;
        parts.plan[1] = total;
    }
    const uint32_t wg0 = blockIdx.x * WAVES * per, wg1 = min(total, wg0 + WAVES * per);
    if (wg0 >= total) return;
    if (p.tables > 64) {
        mine_of = table_work(p, lengths, offsets, nq, group, COLS, KEYS, lane);
        sums = wave_scan(mine_of.cost);
    }
    // the table of block `at`, which is at or behind the last one's
    int t = 0;
    uint32_t before = 0;  // blocks before table t
    TableWork tw{};
    auto seek = [&](uint32_t at) {
        uint64_t past;
        while (!(past = __ballot(chunk_before + sums > at)) && chunk + 64 < p.tables) {
            chunk_before += __builtin_amdgcn_readlane(sums, 63);
            chunk += 64;
            mine_of = table_work(p, lengths, offsets, nq, group, COLS, KEYS, chunk + lane);
            sums = wave_scan(mine_of.cost);
        }
        const int l = past ? __ffsll((unsigned long long)past) - 1 : 0;
        t = chunk + l;
        tw.first = __builtin_amdgcn_readlane(mine_of.first, l);
        tw.n = __builtin_amdgcn_readlane(mine_of.n, l);
        tw.len = __builtin_amdgcn_readlane(mine_of.len, l);
        tw.nb = __builtin_amdgcn_readlane(mine_of.nb, l);
        tw.cost = __builtin_amdgcn_readlane(mine_of.cost, l);
        before = chunk_before + __builtin_amdgcn_readlane(sums, l) - tw.cost;
    };

    // a workgroup whose blocks are one unit's: its wavefronts take them in turn and join what they have
    seek(wg0);
    const bool together = wg1 - wg0 > 1 && wg1 <= before + ((wg0 - before) / tw.nb + 1) * tw.nb;
    uint32_t at = together ? wg0 : wg0 + wave * per;
    const uint32_t end = together ? wg1 : min(total, at + per), mine = at;
    while (at < end) {
        seek(at);
        const uint32_t unit = (at - before) / tw.nb, b0 = at - before - unit * tw.nb, b1 = min(tw.nb, b0 + (end - at));
        const bool done = b0 == 0 && b1 == tw.nb;
        if (!together && b0 > 0 && b0 + BEGIN >= tw.nb) {  // behind the unit's blocks
            if (lane < COLS) parts.ml[(2 * (size_t)me + (at == mine ? 0 : 1)) * COLS + lane] = make_float2(-INFINITY, 0.0f);
            at += b1 - b0;
            continue;
        }
        const int tile = unit / p.heads, h = unit - tile * p.heads;
        const int step = together ? WAVES : 1;
        int kb = (int)b0 + (together ? wave : 0);
        // pages of the table, one a lane from `ids0` on
        const int32_t *pages = p.table + (size_t)t * p.ld;
        int ids0 = ((long)kb * KEYS) >> p.log_rows;
        int ids = pages[min(ids0 + lane, p.ld - 1)];
        // the columns' queries and limits
        halfx8 qh[WAIT ? 1 : CT][C][2], ql[WAIT ? 1 : CT][C][2];
        halfx8 *waiting = reinterpret_cast<halfx8 *>(store) + (size_t)wave * QS + lane;
        // whole numbers, log2: ref, and the values' unit with what follows from both (0 where nothing has been seen)
        float to_log2[CT], ref[CT], vunit[CT], base[CT], gap[CT], l[CT];
        int limit[CT];
        floatx4 acc[CT][M];
        int lim_most = 0, lim_least = tw.len;
        bool small = false;  // ints: queries so small that keys' steps may be as large as a product with them does not hold
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const int col = tile * COLS + 16 * ct + qi, i = col / group;
            const bool live = i < tw.n;
            limit[ct] = live ? (causal ? max(0, tw.len - (tw.n - 1 - i)) : tw.len) : 0;
            lim_most = max(lim_most, limit[ct]);
            lim_least = min(lim_least, live ? limit[ct] : tw.len);
            const float *src = q + (size_t)(tw.first + min(i, tw.n - 1)) * q_ld + (size_t)(h * group + col - i * group) * hd;
            float qv[C][16], most = 0.0f;
#pragma unroll
            for (int c = 0; c < C; c++) {
                const bool in = 64 * c + 16 * lg < hd;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const floatx4 x = *reinterpret_cast<const floatx4u *>(src + (in ? 64 * c + 16 * lg + 4 * j : 0));
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        qv[c][4 * j + e] = live && in ? x[e] : 0.0f;
                        most = fmaxf(most, __uint_as_float(finite_bits(__float_as_uint(qv[c][4 * j + e]))));
                    }
                }
            }
            most = half_max(row_max(most));
            const int eq = shift_below(most);
            const float f = pow2(eq);
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    const int at = WAIT ? 0 : ct;
                    split8(qv[c] + 8 * ks, f, qh[at][c][ks], ql[at][c][ks]);
                    if constexpr (WAIT) {
                        waiting[64 * (4 * (ct * C + c) + 2 * ks)] = qh[0][c][ks];
                        waiting[64 * (4 * (ct * C + c) + 2 * ks + 1)] = ql[0][c][ks];
                    }
                }
            to_log2[ct] = (BYTES ? 256.0f : 1.0f) * LOG2E * pow2(-eq);
            small = small || (INTS && most > 0.0f && eq > 60);
            ref[ct] = vunit[ct] = -INFINITY;
            base[ct] = gap[ct] = l[ct] = 0.0f;
#pragma unroll
            for (int m = 0; m < M; m++) acc[ct][m] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            // where the join finds the unit
            if (b0 == 0 && lg == 0 && live && (!together || wave == 0)) {
                const uint32_t u0 = before + unit * tw.nb;
                parts.units[(size_t)(tw.first + i) * heads + h * group + col - i * group] =
                    make_uint4(u0, u0 + tw.nb, done ? 0 : per, 16 * ct + qi);
            }
        }
#pragma unroll
        for (int d = 1; d < 16; d *= 2) {
            lim_most = max(lim_most, __shfl_xor(lim_most, d));
            lim_least = min(lim_least, __shfl_xor(lim_least, d));
        }
        small = __any(small);
        lim_most = __builtin_amdgcn_readfirstlane(lim_most);
        lim_least = __builtin_amdgcn_readfirstlane(lim_least);
        const int last = min((int)b1, (lim_most + KEYS - 1) / KEYS);  // blocks behind every column's limit are not looked at

        // where the lane's parts of block kb are
        const uint8_t *bk, *bv;
        int slk, slv, idk, idv;
        auto place = [&](int kb) {
            const int first = kb * KEYS;
            const int i0 = first >> p.log_rows, i1 = (first + KEYS - N) >> p.log_rows;
            if (i0 < ids0 || i1 >= ids0 + 64) {
                ids0 = i0;
                ids = pages[min(i0 + lane, p.ld - 1)];
            }
            const int kk = first + N * (qi >> 2), kv = first + N * lg;  // the first keys of what the lane reads
            idk = __shfl(ids, (kk >> p.log_rows) - ids0);
            idv = __shfl(ids, (kv >> p.log_rows) - ids0);
            // not one of the pool's, or behind the table's last: -1, and page 0 read instead
            if ((unsigned)idk >= (unsigned)p.pages || kk >> p.log_rows >= p.ld) idk = -1;
            if ((unsigned)idv >= (unsigned)p.pages || kv >> p.log_rows >= p.ld) idv = -1;
            bk = p.pool + (size_t)max(idk, 0) * p.page_bytes + (size_t)h * p.head_bytes;
            bv = p.pool + (size_t)max(idv, 0) * p.page_bytes + (size_t)h * p.head_bytes;
            slk = (kk & (P - 1)) + (qi & 3);
            slv = kv & (P - 1);
        };
        Raw<FMT, 2> kr[2 * KS][C];
        Raw<FMT, KS> vr[M];
        floatx4 stk[INTS ? N / 4 : 1], stv[INTS ? N / 4 : 1];
        auto load_keys = [&] {
#pragma unroll
            for (int sp = 0; sp < 2 * KS; sp++)
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const bool in = 64 * c + 16 * lg < hd;
                    kr[sp][c] = load_raw<FMT, 2>(bk + ((size_t)(slk + 4 * sp) * hd + (in ? 64 * c + 16 * lg : 0)) * W);
                }
        };
        auto load_values = [&] {
#pragma unroll
            for (int m = 0; m < M; m++)
                vr[m] = load_raw<FMT, KS>(bv + ((size_t)P * hd + (size_t)(16 * m < hd ? 16 * m + qi : qi) * P + slv) * W);
            if constexpr (INTS) {
                const float *steps = reinterpret_cast<const float *>(bv + 2 * (size_t)P * hd * W) + slv;
#pragma unroll
                for (int j = 0; j < N / 4; j++) {
                    stk[j] = reinterpret_cast<const floatx4 *>(steps)[j];
                    stv[j] = reinterpret_cast<const floatx4 *>(steps + P)[j];
                }
            }
        };
        while (kb < last) {
            place(kb);
            load_keys();
            if constexpr (C * CT <= 2) load_values();
            const int first = kb * KEYS, kv = first + N * lg;
            const bool whole = first + KEYS <= tw.len && __all(idv >= 0);  // every key there is and on a page
            // of the lane's N keys (values), how many there are
            const int here = whole ? N : (idv >= 0 ? min(max(tw.len - kv, 0), N) : 0);
            const bool all_seen = whole && first + KEYS <= lim_least;
            const bool in_part = lim_least < min(first + KEYS, tw.len);  // some column does not see all that is there
            // coordinates past the head's width; f32: keys that are not there, and the block's keys' power of two
            int ek = 0;
            if (hd & 63) {
#pragma unroll
                for (int sp = 0; sp < 2 * KS; sp++)
#pragma unroll
                    for (int c = 0; c < C; c++)
                        if (64 * c + 16 * lg >= hd)
#pragma unroll
                            for (int i = 0; i < Raw<FMT, 2>::WORDS; i++) kr[sp][c].w[i] = 0;
            }
            if constexpr (!INTS) {
                if (!whole) {
                    const int there = idk >= 0 ? tw.len - first - N * (qi >> 2) - (qi & 3) : 0;  // row of set sp is: 4 sp < there
#pragma unroll
                    for (int sp = 0; sp < 2 * KS; sp++)
                        if (4 * sp >= there)
#pragma unroll
                            for (int c = 0; c < C; c++)
#pragma unroll
                                for (int i = 0; i < Raw<FMT, 2>::WORDS; i++) kr[sp][c].w[i] = 0;
                }
                float rows[2 * KS], most = 0.0f;  // the largest of the lane's numbers of a row
#pragma unroll
                for (int sp = 0; sp < 2 * KS; sp++) {
                    uint32_t bits = 0;
#pragma unroll
                    for (int c = 0; c < C; c++)
#pragma unroll
                        for (int i = 0; i < Raw<FMT, 2>::WORDS; i++) bits = max(bits, finite_bits(kr[sp][c].w[i]));
                    rows[sp] = __uint_as_float(bits);
                    most = fmaxf(most, rows[sp]);
                }
                most = wave_max(most);
                if (!in_part) {
                    ek = shift_below(most);
                } else {  // each by its own
#pragma unroll
                    for (int sp = 0; sp < 2 * KS; sp++) {
                        const int e = shift_below(half_max(row_max(rows[sp])));
#pragma unroll
                        for (int c = 0; c < C; c++)
#pragma unroll
                            for (int i = 0; i < Raw<FMT, 2>::WORDS; i++)
                                kr[sp][c].w[i] = __float_as_uint(__uint_as_float(kr[sp][c].w[i]) * pow2(e));
                        if (lg == 0) steps_here[wave][0][N * (qi >> 2) + 4 * sp + (qi & 3)] = pow2(-e);
                    }
                }
            }
            const float fk = INTS ? 1.0f : pow2(ek);
            floatx4 sc[2 * KS][CT];  // set sp = 2 s + p
            const floatx4 none = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int ks = 0; ks < 2; ks++)
#pragma unroll
                    for (int sp = 0; sp < 2 * KS; sp++) {
                        halfx8 hi, lo;
                        to_halves<FMT, 2>(kr[sp][c], ks, fk, hi, lo);
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) {
                            halfx8 qhi, qlo;
                            if constexpr (WAIT) {
                                qhi = waiting[64 * (4 * (ct * C + c) + 2 * ks)];
                                qlo = waiting[64 * (4 * (ct * C + c) + 2 * ks + 1)];
                            } else {
                                qhi = qh[ct][c][ks];
                                qlo = ql[ct][c][ks];
                            }
                            sc[sp][ct] = mfma(hi, qhi, c + ks ? sc[sp][ct] : none);
                            sc[sp][ct] = mfma(hi, qlo, sc[sp][ct]);
                            if constexpr (LO) sc[sp][ct] = mfma(lo, qhi, sc[sp][ct]);
                            if constexpr (BYTES) sc[sp][ct] = mfma(lo, qlo, sc[sp][ct]);
                        }
                    }
            if constexpr (C * CT > 2) {  // no registers for them before
                __builtin_amdgcn_sched_barrier(0);
                load_values();
            }
            // The values' scale: the power of two of the largest step that a column sees. f32 has one step for the block, which brings
            // every value below 2^14, or in part one for each row.
            float eb[CT], vs = 1.0f;
            uint32_t odd = 0;  // f32: whether a value is not finite
            if constexpr (!INTS) {
                uint32_t rows[N], most = 0;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    rows[i] = 0;
#pragma unroll
                    for (int m = 0; m < M; m++) {
                        if (!whole && i >= here) vr[m].w[i] = 0;
                        odd = max(odd, vr[m].w[i] & 0x7fffffffu);
                        rows[i] = max(rows[i], finite_bits(vr[m].w[i]));
                    }
                    most = max(most, rows[i]);
                }
                if (in_part) {
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const int e = shift_below(row16_reduce(__uint_as_float(rows[i]), fmaxf));
#pragma unroll
                        for (int m = 0; m < M; m++) vr[m].w[i] = __float_as_uint(__uint_as_float(vr[m].w[i]) * pow2(e));
                        steps_here[wave][1][N * lg + i] = pow2(-e);  // of sixteen lanes the same
                    }
                } else {
                    const int e = shift_below(wave_max(__uint_as_float(most)));
                    vs = pow2(e);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) eb[ct] = (float)-e;
                }
            }
            if (INTS && !whole)
#pragma unroll
                for (int j = 0; j < N; j++)
                    if (j >= here) stv[j >> 2][j & 3] = 0.0f;
            auto value_step = [&](int j) {
                if constexpr (INTS) {
                    const float f = stv[j >> 2][j & 3];
                    return f;
                } else {
                    return steps_here[wave][1][N * lg + j];
                }
            };
            auto largest_of = [&](int seen) {
                float most = 0.0f;
#pragma unroll
                for (int j = 0; j < N; j++) most = j < seen ? fmaxf(most, value_step(j)) : most;
                most = half_max(row_max(most));
                return most > 0.0f ? (float)max(__builtin_amdgcn_frexp_expf(most), -126) : -126.0f;
            };
            if (in_part) {
#pragma unroll
                for (int ct = 0; ct < CT; ct++) eb[ct] = largest_of(limit[ct] - kv);
            } else if (INTS) {
                eb[0] = largest_of(N);
#pragma unroll
                for (int ct = 1; ct < CT; ct++) eb[ct] = eb[0];
            }
            halfx8 ph[CT][KS], pl[CT][KS];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                float x[N];
                auto in_log2 = [&](float unk) { return fminf(fmaxf(to_log2[ct] * unk, 0x1p-126f), 0x1p126f); };
                float f = INTS ? to_log2[ct] : in_log2(pow2(-ek));
#pragma unroll
                for (int j = 0; j < N; j++) x[j] = sc[j >> 2][ct][j & 3];
                if (INTS ? small : in_part) {  // the factors first
                    f = 1.0f;
#pragma unroll
                    for (int j = 0; j < N; j++)
                        x[j] *= INTS ? stk[j >> 2][j & 3] * to_log2[ct] : in_log2(steps_here[wave][0][INTS ? 0 : N * lg + j]);
                } else if constexpr (INTS) {
#pragma unroll
                    for (int j = 0; j < N; j++) x[j] *= stk[j >> 2][j & 3];
                }
                if (!all_seen) {
                    const int seen = min(here, min(max(limit[ct] - kv, 0), N));
#pragma unroll
                    for (int j = 0; j < N; j++)
                        if (j >= seen) x[j] = -INFINITY;
                }
                float mb = x[0];
#pragma unroll
                for (int j = 1; j < N; j++) mb = fmaxf(mb, x[j]);
                mb = half_max(row_max(mb)) * f;
                const float top = mb + eb[ct];  // of weights times steps
                const bool grow = mb > ref[ct] + 3.0f, grow_values = top > vunit[ct] + 3.0f;
                if (__any(grow || grow_values)) {
                    const float nref = grow ? floorf(mb) : ref[ct], nvunit = grow_values ? floorf(top) : vunit[ct];
                    l[ct] *= grow ? pow2((int)fmaxf(ref[ct] - nref, -200.0f)) : 1.0f;
                    const float beta = grow_values ? pow2((int)fmaxf(vunit[ct] - nvunit, -200.0f)) : 1.0f;
#pragma unroll
                    for (int m = 0; m < M; m++) acc[ct][m] *= beta;
                    ref[ct] = nref;
                    vunit[ct] = nvunit;
                    base[ct] = nref == -INFINITY ? 0.0f : 12.0f - nref;
                    gap[ct] = nref == -INFINITY ? 0.0f : nref - nvunit;
                }
                // what the block's weights are taken larger by (below 2^-60 they are zeros as halves; their sum is taken of them)
                const float less = fmaxf(gap[ct] + eb[ct], -60.0f), off = base[ct] + less, step = pow2(-(int)eb[ct]);
                float ps = 0.0f;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    u32x4 hw, lw;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int j = 8 * s + 2 * i;
                        float p0 = exp2_hw(fmaf(x[j], f, off)), p1 = exp2_hw(fmaf(x[j + 1], f, off));
                        ps += p0 + p1;
                        if (INTS || in_part) {  // at most 1 where it is seen
                            p0 *= __builtin_amdgcn_fmed3f(value_step(j) * step, 0.0f, 1.0f);
                            p1 *= __builtin_amdgcn_fmed3f(value_step(j + 1) * step, 0.0f, 1.0f);
                        }
                        uint32_t a, b;
                        split2(p0, p1, a, b);
                        hw[i] = a;
                        lw[i] = b;
                    }
                    ph[ct][s] = __builtin_bit_cast(halfx8, hw);
                    pl[ct][s] = __builtin_bit_cast(halfx8, lw);
                }
                l[ct] = fmaf(ps, pow2(-(int)less), l[ct]);
            }
            // values that are not finite: zeros in the products, and what sees one is no number
            if constexpr (!INTS) {
                if (__any(odd >= 0x7f800000u)) {
                    const _Float16 one = (_Float16)1.0f, zero = (_Float16)0.0f;
#pragma unroll
                    for (int m = 0; m < M; m++)
#pragma unroll
                        for (int s = 0; s < KS; s++) {
                            halfx8 bad;
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                const uint32_t w = vr[m].w[8 * s + e];
                                const bool b = (w & 0x7fffffffu) >= 0x7f800000u;
                                bad[e] = b ? one : zero;
                                vr[m].w[8 * s + e] = b ? 0u : w;
                            }
#pragma unroll
                            for (int ct = 0; ct < CT; ct++) {
                                const int seen = min(here, min(max(limit[ct] - kv, 0), N));
                                halfx8 sees;
#pragma unroll
                                for (int e = 0; e < 8; e++) sees[e] = 8 * s + e < seen ? one : zero;
                                const floatx4 n = mfma(bad, sees, none);
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    if (n[i] > 0.0f) acc[ct][m][i] = NAN;
                            }
                        }
                }
            }
#pragma unroll
            for (int m = 0; m < M; m++) {
                if (16 * m >= hd) break;
                __builtin_amdgcn_sched_barrier(0);  // a set's halves at a time: all at once they do not fit the registers
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    halfx8 hi, lo;
                    to_halves<FMT, KS>(vr[m], s, vs, hi, lo);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        acc[ct][m] = mfma(hi, ph[ct][s], acc[ct][m]);
                        acc[ct][m] = mfma(hi, pl[ct][s], acc[ct][m]);
                        if constexpr (LO) acc[ct][m] = mfma(lo, ph[ct][s], acc[ct][m]);
                        if constexpr (BYTES) acc[ct][m] = mfma(lo, pl[ct][s], acc[ct][m]);
                    }
                }
            }
            kb += step;
        }
        at += b1 - b0;
        // the sums over the weights' sum
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const float lw = half_sum(row_sum(l[ct]));
            const float inv = lw > 0.0f ? 1.0f / lw : lw;  // 0 and NaN stay
            const float uv = (BYTES ? 256.0f : 1.0f) * pow2(-(int)gap[ct]);
            if (!together) {
                const size_t own = 2 * (size_t)me + (at - (b1 - b0) == mine ? 0 : 1);
                const int col = 16 * ct + qi, c = tile * COLS + col, i = c / group;
                if (done && i >= tw.n) continue;
                float *dst = done ? out + (size_t)(tw.first + i) * heads * hd + (size_t)(h * group + c - i * group) * hd
                                  : parts.o + (own * COLS + col) * hd;
#pragma unroll
                for (int m = 0; m < M; m++)
                    if (16 * m < hd) {
                        const floatx4 o = acc[ct][m] * inv * uv;
                        *reinterpret_cast<floatx4u *>(dst + 16 * m + 4 * lg) = o;
                    }
                if (!done && lg == 0) parts.ml[own * COLS + col] = make_float2(ref[ct], lw);
                continue;
            }
            if (lg == 0) {
                mref[wave][16 * ct + qi] = ref[ct];
                msum[wave][16 * ct + qi] = lw;
            }
            if (WAIT || ct) __syncthreads();
#pragma unroll
            for (int m = 0; m < M; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) macc[wave][16 * m + 4 * lg + i][qi] = acc[ct][m][i] * inv * uv;
            __syncthreads();
            // 64 WAVES / 16 threads a column
            constexpr int TH = 4 * WAVES;
            const int c16 = tid / TH, col = 16 * ct + c16, c = tile * COLS + col, i = c / group;
            float m = -INFINITY, L = 0.0f, f[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; w++)
                if (msum[w][col] > 0.0f) m = fmaxf(m, mref[w][col]);
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float sw = msum[w][col];
                f[w] = sw > 0.0f ? sw * exp2_hw(mref[w][col] - m) : sw;
                L += f[w];
            }
            const float Li = L > 0.0f ? 1.0f / L : L;
            const size_t own = 2 * (size_t)(blockIdx.x * WAVES);
            for (int dim = tid % TH; dim < hd; dim += TH) {
                float o = 0.0f;
#pragma unroll
                for (int w = 0; w < WAVES; w++)
                    if (msum[w][col] != 0.0f) o += f[w] * Li * macc[w][dim][c16];
                if (!done)
                    parts.o[(own * COLS + col) * hd + dim] = o;
                else if (i < tw.n)
                    out[(size_t)(tw.first + i) * heads * hd + (size_t)(h * group + c - i * group) * hd + dim] = o;
            }
            if (!done && tid % TH == 0) parts.ml[own * COLS + col] = make_float2(m, L);
        }
        if (together) break;
    }
}

// grid (queries x heads, over 4 / PER; in rows of `row` where they are more than MOST_WGS); 256 threads: the states that runs of blocks
// left of a query and head, together: PER wavefronts for each query and head, every PER-th state each. Four where there are few (a
// state after the other takes longest: the call of one query of 8 heads over 100,000 rows 33 us, with one 42; 7 tables of up to 9,000
// 23.6 and 27.5), one where there are many (their number does: 24 tables, up to 9 queries each, of 16 heads 62.4 us, with four 65.6).
// The launch is most of it.
template <int CT, int PER>
__global__ __launch_bounds__(256) void k_pages_join(int tables, int hd, const int32_t *__restrict__ offsets, int items,
                                                    int heads, float *__restrict__ out, Parts parts, uint32_t row) {
    constexpr int COLS = 16 * CT, AHEAD = 8;
    __shared__ float wm[4], wl[4], wo[4][128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t nth = PER == 4 ? blockIdx.x : (blockIdx.y * row + blockIdx.x) * 4 + wave;
    if (nth >= (uint32_t)items) return;
    const int item = (int)nth, part = PER == 4 ? wave : 0;
    const uint4 unit = parts.units[item];
    const uint32_t per = parts.plan[0], total = parts.plan[1], u0 = unit.x, u1 = unit.y, col = unit.w;
    // of no table (what its place holds is another call's); there already
    if (item / heads >= offsets[tables] || unit.z != per || u1 > total || u0 >= u1 || col >= COLS) return;
    const uint32_t w0 = u0 / per, w1 = (u1 - 1) / per, g0 = w0 / WAVES, g1 = w1 / WAVES;
    // the states: the first workgroup's, a wavefront each or one for all, one of each workgroup between, the last one's
    auto together = [&](uint32_t g) {
        const uint32_t a = g * WAVES * per, b = min(total, a + WAVES * per);
        return b - a > 1 && a >= u0 && b <= u1;
    };
    const uint32_t n0 = together(g0) ? 1 : min(w1, g0 * WAVES + WAVES - 1) - w0 + 1;
    const uint32_t n1 = g1 > g0 ? g1 - g0 - 1 : 0, n2 = g1 > g0 ? (together(g1) ? 1 : w1 - g1 * WAVES + 1) : 0;
    const uint32_t count = n0 + n1 + n2;
    auto slot = [&](uint32_t e) {
        const uint32_t w = e < n0 ? w0 + e : (e < n0 + n1 ? (g0 + 1 + e - n0) * WAVES : g1 * WAVES + e - n0 - n1);
        return 2 * (size_t)w + (w == w0 && u0 > w0 * per ? 1 : 0);
    };
    float M = -INFINITY, L = 0.0f, o0 = 0.0f, o1 = 0.0f;
    const int d0 = min(lane, hd - 1), d1 = min(64 + lane, hd - 1);
    for (uint32_t e = part; e < count; e += PER * AHEAD) {
        float2 ml[AHEAD];
        float x0[AHEAD], x1[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            // past the last: the last again, without weight
            const size_t at = slot(min(e + PER * i, count - 1)) * COLS + col;
            ml[i] = parts.ml[at];
            x0[i] = parts.o[at * hd + d0];
            x1[i] = hd > 64 ? parts.o[at * hd + d1] : 0.0f;
            if (e + PER * i >= count) ml[i] = make_float2(-INFINITY, 0.0f);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (ml[i].y > 0.0f) top = fmaxf(top, ml[i].x);
        // shares of the sum so far, so that no value is multiplied by more than 1
        const float old = M == -INFINITY ? L : L * exp2_hw(M - top);  // nothing yet, or NaN
        float f[AHEAD];
        L = old;
        M = top;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            f[i] = ml[i].y > 0.0f ? ml[i].y * exp2_hw(ml[i].x - M) : ml[i].y;
            L += f[i];
        }
        const float inv = L > 0.0f ? 1.0f / L : L;
        o0 *= old * inv;
        o1 *= old * inv;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (ml[i].y == 0.0f) continue;
            o0 += f[i] * inv * x0[i];
            o1 += f[i] * inv * x1[i];
        }
    }
    if constexpr (PER == 4) {
        wo[wave][lane] = o0;
        wo[wave][64 + lane] = o1;
        if (lane == 0) {
            wm[wave] = M;
            wl[wave] = L;
        }
        __syncthreads();
        if (wave > 0) return;
        const float top = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
        L = o0 = o1 = 0.0f;
        float f[4];
#pragma unroll
        for (int w = 0; w < 4; w++) {
            f[w] = wm[w] == -INFINITY ? wl[w] : wl[w] * exp2_hw(wm[w] - top);
            L += f[w];
        }
        const float inv = L > 0.0f ? 1.0f / L : L;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            if (wl[w] == 0.0f) continue;
            o0 += f[w] * inv * wo[w][lane];
            o1 += f[w] * inv * wo[w][64 + lane];
        }
    }
    float *dst = out + (size_t)item * hd;
    if (lane < hd) dst[lane] = o0;
    if (64 + lane < hd) dst[64 + lane] = o1;
}

// Keys of a block: 64, or 32 where a wavefront's registers do not hold more (C parts of 64 coordinates, CT sets of 16 columns).
constexpr int block_keys(int fmt, int C, int CT) {
    const int bytes = page_width(fmt) * C;
    return bytes > 2 || (bytes == 2 && C * CT == 4) ? 32 : 64;
}

// Sets of 16 columns that share what a wavefront reads (f32 heads over 64 wide: no registers for two); workgroups, two a compute
// unit, fewer where there may not be a block for each of their wavefronts.
struct Shape {
    int sets, wgs;
    size_t o_floats, ml_count, units;
    uint64_t blocks;  // at most
};

Shape shape(int fmt, const PageSet &p, int nq, int heads) {
    Shape s;
    const int64_t group = heads / p.heads, columns = (int64_t)nq * group;
    s.sets = columns > 16 * (int64_t)p.tables && (fmt != TAH_KV_F32 || p.hd <= 64) ? 2 : 1;
    const int keys = block_keys(fmt, p.hd > 64 ? 2 : 1, s.sets);
    const uint64_t rows = std::min((uint64_t)p.ld << p.log_rows, (uint64_t)0x7fffffff - 64);
    const uint64_t units = ((uint64_t)std::min(p.tables, nq) + columns / (16 * s.sets)) * p.heads;
    const uint64_t nb = (rows + keys - 1) / keys + BEGIN;
    s.blocks = units > (uint64_t(1) << 32) ? ~uint64_t(0) : units * nb;
    s.wgs = (int)std::min<uint64_t>(512, (s.blocks + WAVES - 1) / WAVES);
    const size_t slots = 2 * (size_t)s.wgs * WAVES;
    s.o_floats = slots * 16 * s.sets * p.hd;
    s.ml_count = slots * 16 * s.sets;
    s.units = (size_t)nq * heads;
    return s;
}

template <int FMT, int C, int CT>
void launch(hipStream_t s, const PageSet &p, const int32_t *lengths, const float *q, const int32_t *offsets, int nq, int heads,
            bool causal, size_t q_ld, float *out, const Parts &parts, const Shape &sh) {
    hipLaunchKernelGGL((k_pages_attend<FMT, C, CT, block_keys(FMT, C, CT) / 32>), dim3(sh.wgs), dim3(64 * WAVES), 0, s, p, lengths, q,
                       offsets, nq, heads, causal ? 1 : 0, q_ld, out, parts, sh.blocks);
    TAH_LAUNCHED();
    const int items = nq * heads;
    if (items <= 1024) {
        hipLaunchKernelGGL((k_pages_join<CT, 4>), dim3(items), dim3(256), 0, s, p.tables, p.hd, offsets, items, heads, out, parts, 0u);
    } else {
        const int wgs = (items + 3) / 4, rows = (wgs + MOST_WGS - 1) / MOST_WGS, row = (wgs + rows - 1) / rows;
        hipLaunchKernelGGL((k_pages_join<CT, 1>), dim3(row, rows), dim3(256), 0, s, p.tables, p.hd, offsets, items, heads, out, parts,
                           (uint32_t)row);
    }
    TAH_LAUNCHED();
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

}  // namespace

size_t pages_attend_work_bytes(int fmt, const PageSet &p, int nq, int heads) {
    const Shape s = shape(fmt, p, nq, heads);
    // the kernels number all units' blocks in 32 bits
    if (s.blocks >= (uint64_t(1) << 31)) throw ArgError{"pages_attend: more rows than a call takes: fewer tables a call"};
    return up256(s.o_floats * sizeof(float)) + up256(s.ml_count * sizeof(float2)) + up256(s.units * sizeof(uint4)) + 256;
}

void pages_attend(hipStream_t s, int fmt, const PageSet &p, const int32_t *lengths, const float *q, const int32_t *offsets, int nq,
                  int heads, bool causal, size_t q_ld, float *out, void *work) {
    const Shape sh = shape(fmt, p, nq, heads);
    uint8_t *at = static_cast<uint8_t *>(work);
    Parts parts;
    parts.o = reinterpret_cast<float *>(at);
    parts.ml = reinterpret_cast<float2 *>(at += up256(sh.o_floats * sizeof(float)));
    parts.units = reinterpret_cast<uint4 *>(at += up256(sh.ml_count * sizeof(float2)));
    parts.plan = reinterpret_cast<uint32_t *>(at + up256(sh.units * sizeof(uint4)));
    auto go = [&](auto kernel) { kernel(s, p, lengths, q, offsets, nq, heads, causal, q_ld, out, parts, sh); };
    const bool wide = p.hd > 64, two = sh.sets == 2;
    if (fmt == TAH_KV_F32)
        wide ? go(launch<TAH_KV_F32, 2, 1>) : (two ? go(launch<TAH_KV_F32, 1, 2>) : go(launch<TAH_KV_F32, 1, 1>));
    else if (fmt == TAH_KV_I16)
        wide ? (two ? go(launch<TAH_KV_I16, 2, 2>) : go(launch<TAH_KV_I16, 2, 1>))
             : (two ? go(launch<TAH_KV_I16, 1, 2>) : go(launch<TAH_KV_I16, 1, 1>));
    else
        wide ? (two ? go(launch<TAH_KV_I8, 2, 2>) : go(launch<TAH_KV_I8, 2, 1>))
             : (two ? go(launch<TAH_KV_I8, 1, 2>) : go(launch<TAH_KV_I8, 1, 1>));
}

}  // namespace tah
