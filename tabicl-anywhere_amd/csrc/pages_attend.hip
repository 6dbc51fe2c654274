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

constexpr int WAVES = 8;

// What a run of blocks leaves behind for the join, per slot: [columns][hd] outputs and [columns] (maximum, sum). A wavefront has
// at most two units that are not whole, its first and its last: slots 2 w and 2 w + 1.
struct Parts {
    float *o;
    float2 *ml;
    uint32_t *plan;  // blocks a wavefront; each table's first block; the blocks in all
};

// queries of table t (from `first`), its rows, and its blocks
struct TableWork {
    int first, n, len, tiles, nb;
    uint32_t cost;
};

__device__ __forceinline__ TableWork table_work(const PageSet &p, const int32_t *lengths, const int32_t *offsets, int nq, int group,
                                                int columns, int t) {
    TableWork w;
    const int a = min(max(offsets[t], 0), nq), b = min(max(offsets[t + 1], a), nq);
    w.first = a;
    w.n = b - a;
    const long most = min((long)p.ld << p.log_rows, (long)0x7fffffff - 64);
    w.len = (int)min((long)max(lengths[t], 0), most);
    w.tiles = (w.n * group + columns - 1) / columns;
    w.nb = max(1, (w.len + 63) >> 6);
    w.cost = (uint32_t)w.tiles * p.heads * w.nb;
    return w;
}

// sixteen stored numbers of a lane as halves: eight for either half of 16, exact in hi (i8) or hi + lo
template <int FMT>
struct Raw;
template <>
struct Raw<TAH_KV_I8> {
    u32x4 w[1];
};
template <>
struct Raw<TAH_KV_I16> {
    u32x4 w[2];
};
template <>
struct Raw<TAH_KV_F32> {
    u32x4 w[4];
};

template <int FMT>
__device__ __forceinline__ Raw<FMT> load_raw(const uint8_t *at) {
    Raw<FMT> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 16); i++) r.w[i] = reinterpret_cast<const u32x4 *>(at)[i];
    return r;
}

// bytes of a word, signed, as halves: 0x6400 | (b + 128) is 1024 + 128 + b in fp16, exact
__device__ __forceinline__ halfx2 half_bytes(uint32_t flipped, uint32_t sel) {
    return __builtin_bit_cast(halfx2, __builtin_amdgcn_perm(flipped, 0x64646464u, sel)) - halfx2{(_Float16)1152.0f, (_Float16)1152.0f};
}

template <int FMT>
__device__ __forceinline__ void to_halves(const Raw<FMT> &r, int s, float f, halfx8 &hi, halfx8 &lo) {
    if constexpr (FMT == TAH_KV_I8) {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t w = r.w[0][2 * s + i] ^ 0x80808080u;
            o[2 * i] = __builtin_bit_cast(uint32_t, half_bytes(w, 0x00050004u));
            o[2 * i + 1] = __builtin_bit_cast(uint32_t, half_bytes(w, 0x00070006u));
        }
        hi = __builtin_bit_cast(halfx8, o);
    } else if constexpr (FMT == TAH_KV_I16) {
        u32x4 a, b;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = r.w[s][i];
            uint32_t x, y;
            split2((float)(int16_t)(w & 0xffffu), (float)(int16_t)(w >> 16), x, y);
            a[i] = x;
            b[i] = y;
        }
        hi = __builtin_bit_cast(halfx8, a);
        lo = __builtin_bit_cast(halfx8, b);
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t w = r.w[2 * s + (i >> 2)][i & 3];
            v[i] = __uint_as_float(w);
        }
        split8(v, f, hi, lo);
    }
}

__device__ __forceinline__ floatx4 mfma(halfx8 a, halfx8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// grid: any number of workgroups of 8 wavefronts.
//
// Products are 16 x 16 x 32 with the queries as columns: S = K Q^T for sets of 16 keys, then O^T += V^T P^T. A lane (lg = lane /
// 16) has keys 16 lg .. 16 lg + 15 of a block: set (s, p)'s row r is key 16 (r / 4) + 8 s + 4 p + r % 4, so that the scores of
// sets (s, 0) and (s, 1) are the operand of the values' product s in place, sixteen consecutive numbers of a coordinate are what
// a lane reads of the values, and a page of 16 rows or more holds all that a lane reads at once. Coordinates go likewise: step
// (c, ks) takes 64 c + 16 lg + 8 ks .. + 7.
//
// Numbers: ints go in as they are (i8 exact in one half, i16 in two), the key's step multiplies its scores, the value's its
// weights; f32 goes in as two halves times the block's power of two. Queries and weights are two halves. So a term is two
// products (i8) or three, for f32's error. Weights are held below 2^15 (their maximum raised by blocks that pass it by more than
// 2^3), times the value's step over a power of two that no step so far passes.
template <int FMT, int C, int CT>
__global__ __launch_bounds__(64 * WAVES) void k_pages_attend(PageSet p, const int32_t *__restrict__ lengths,
                                                             const float *__restrict__ q, const int32_t *__restrict__ offsets,
                                                             int nq, int heads, int causal, size_t q_ld,
                                                             float *__restrict__ out, Parts parts, uint64_t most_blocks) {
    constexpr int W = page_width(FMT), COLS = 16 * CT, HD = 64 * C, M = 4 * C;
    constexpr bool INTS = FMT != TAH_KV_F32, LO = FMT != TAH_KV_I8;
    __shared__ float mref[WAVES][COLS], msum[WAVES][COLS], macc[WAVES][HD][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int qi = lane & 15, lg = lane >> 4, group = heads / p.heads, hd = p.hd, P = p.rows;
    const uint32_t waves = gridDim.x * WAVES, me = blockIdx.x * WAVES + wave;

    // the plan: every wavefront adds up all tables' blocks and finds its own
    uint64_t all = 0;
    for (int t0 = 0; t0 < p.tables; t0 += 64) {
        const int t = t0 + lane;
        const uint64_t c = t < p.tables ? table_work(p, lengths, offsets, nq, group, COLS, t).cost : 0;
        const uint64_t sum = wave_scan(c);
        if (me == 0 && t < p.tables) parts.plan[1 + t] = (uint32_t)(all + sum - c);
        all += __shfl(sum, 63);
    }
    // offsets that fall may make more of the queries than there are: nothing is done then
    const uint32_t total = all <= most_blocks ? __builtin_amdgcn_readfirstlane((uint32_t)all) : 0;
    const uint32_t per = max(1u, (total + waves - 1) / waves);
    if (me == 0 && lane == 0) {
        parts.plan[0] = per;
        parts.plan[1 + p.tables] = total;
    }
    const uint32_t wg0 = blockIdx.x * WAVES * per, wg1 = min(total, wg0 + WAVES * per);
    if (wg0 >= total) return;

    // the table of block `at`, at or behind the one held
    int t = -1;
    uint32_t before = 0;  // blocks before table t
    TableWork tw{};
    auto seek = [&](uint32_t at) {
        if (t >= 0 && at < before + tw.cost) return;
        uint32_t sums = t < 0 ? 0 : before + tw.cost;
        for (int t0 = t + 1; t0 < p.tables; t0 += 64) {
            const int i = t0 + lane;
            const uint32_t c = i < p.tables ? table_work(p, lengths, offsets, nq, group, COLS, i).cost : 0;
            const uint32_t sum = wave_scan(c);
            const uint64_t past = __ballot(sums + sum > at);
            if (past) {
                const int l = __ffsll((unsigned long long)past) - 1;
                t = __builtin_amdgcn_readfirstlane(t0 + l);
                before = sums + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(c, l);
                tw = table_work(p, lengths, offsets, nq, group, COLS, t);
                return;
            }
            sums += __builtin_amdgcn_readlane(sum, 63);
        }
    };

    // one unit: its columns' queries and limits, and the state that its blocks add to
    int tile = 0, h = 0;
    halfx8 qh[CT][C][2], ql[CT][C][2];
    float to_log2[CT], ref[CT], l[CT];
    int limit[CT], ev;
    floatx4 acc[CT][M];
    int lim_most = 0, lim_least = 0;
    auto begin = [&](uint32_t unit) {
        tile = unit / p.heads;
        h = unit - tile * p.heads;
        ev = INTS ? -1000 : 1000;
        lim_most = 0;
        lim_least = tw.len;
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
                    const floatx4 x = in ? (floatx4) * reinterpret_cast<const floatx4u *>(src + 64 * c + 16 * lg + 4 * j)
                                         : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        qv[c][4 * j + e] = live ? x[e] : 0.0f;
                        most = fmaxf(most, __uint_as_float(finite_bits(__float_as_uint(qv[c][4 * j + e]))));
                    }
                }
            }
            most = half_max(row_max(most));
            const int eq = min(shift_for_max(most), 126);
            const float f = pow2(eq);
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int ks = 0; ks < 2; ks++) split8(qv[c] + 8 * ks, f, qh[ct][c][ks], ql[ct][c][ks]);
            to_log2[ct] = LOG2E * pow2(-eq);
            ref[ct] = -INFINITY;
            l[ct] = 0.0f;
#pragma unroll
            for (int m = 0; m < M; m++) acc[ct][m] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int d = 1; d < 16; d *= 2) {
            lim_most = max(lim_most, __shfl_xor(lim_most, d));
            lim_least = min(lim_least, __shfl_xor(lim_least, d));
        }
        lim_most = __builtin_amdgcn_readfirstlane(lim_most);
        lim_least = __builtin_amdgcn_readfirstlane(lim_least);
    };

    // pages of the table, one a lane from `ids0` on
    int ids = -1, ids0 = 0;
    auto pages_from = [&](int i0) {
        ids0 = i0;
        ids = page_of(p, t, (long)(i0 + lane) << p.log_rows);
    };
    auto block = [&](int kb) {
        const int first = kb * 64;
        const int i0 = first >> p.log_rows, i1 = (first + 48) >> p.log_rows;
        if (i0 < ids0 || i1 >= ids0 + 64) pages_from(i0);
        const int kk = first + 16 * (qi >> 2), kv = first + 16 * lg;  // the first keys of what the lane reads
        const int idk = __shfl(ids, (kk >> p.log_rows) - ids0), idv = __shfl(ids, (kv >> p.log_rows) - ids0);
        const uint8_t *bk = p.pool + (size_t)max(idk, 0) * p.page_bytes + (size_t)h * p.head_bytes;
        const uint8_t *bv = p.pool + (size_t)max(idv, 0) * p.page_bytes + (size_t)h * p.head_bytes;
        const int slk = (kk & (P - 1)) + (qi & 3), slv = kv & (P - 1);
        const bool whole = first + 64 <= tw.len && __all(idv >= 0);  // every key there is and on a page
        // of the lane's sixteen keys (values), how many there are
        const int here = whole ? 16 : (idv >= 0 ? min(max(tw.len - kv, 0), 16) : 0);
        const bool all_seen = whole && first + 64 <= lim_least;
        Raw<FMT> kr[4][C], vr[M];
#pragma unroll
        for (int sp = 0; sp < 4; sp++)
#pragma unroll
            for (int c = 0; c < C; c++) {
                const bool in = 64 * c + 16 * lg < hd;
                kr[sp][c] = load_raw<FMT>(bk + ((size_t)(slk + 4 * sp) * hd + (in ? 64 * c + 16 * lg : 0)) * W);
                if (!in)
#pragma unroll
                    for (int i = 0; i < (int)(sizeof(Raw<FMT>) / 16); i++) kr[sp][c].w[i] = u32x4{0, 0, 0, 0};
            }
        floatx4 stk[INTS ? 4 : 1], stv[INTS ? 4 : 1];
        if constexpr (INTS) {
            const float *steps = reinterpret_cast<const float *>(bv + 2 * (size_t)P * hd * W) + slv;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                stk[j] = reinterpret_cast<const floatx4 *>(steps)[j];
                stv[j] = reinterpret_cast<const floatx4 *>(steps + P)[j];
            }
        }
#pragma unroll
        for (int m = 0; m < M; m++) {
            const int dim = 16 * m + qi;
            vr[m] = load_raw<FMT>(bv + ((size_t)P * hd + (size_t)(16 * m < hd ? dim : qi) * P + slv) * W);
        }
        // f32: the block's keys' power of two, those that are not there left out
        int ek = 0;
        if constexpr (!INTS) {
            if (!whole) {
                const int there = idk >= 0 ? tw.len - kk - (qi & 3) : 0;  // row of set sp is there: 4 sp < there
#pragma unroll
                for (int sp = 0; sp < 4; sp++)
                    if (4 * sp >= there)
#pragma unroll
                        for (int c = 0; c < C; c++)
#pragma unroll
                            for (int i = 0; i < 4; i++) kr[sp][c].w[i] = u32x4{0, 0, 0, 0};
            }
            uint32_t most = 0;
#pragma unroll
            for (int sp = 0; sp < 4; sp++)
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) most = max(most, finite_bits(kr[sp][c].w[i][e]));
            ek = min(shift_for_max(wave_max(__uint_as_float(most))), 126);
        }
        const float fk = INTS ? 1.0f : pow2(ek), unk = INTS ? 1.0f : pow2(-ek);
        floatx4 sc[4][CT];  // set sp = 2 s + p
        const floatx4 none = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int sp = 0; sp < 4; sp++)
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    halfx8 hi, lo;
                    to_halves<FMT>(kr[sp][c], ks, fk, hi, lo);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        sc[sp][ct] = mfma(hi, qh[ct][c][ks], c + ks ? sc[sp][ct] : none);
                        sc[sp][ct] = mfma(hi, ql[ct][c][ks], sc[sp][ct]);
                        if constexpr (LO) sc[sp][ct] = mfma(lo, qh[ct][c][ks], sc[sp][ct]);
                    }
                }
        // the values' scale: ints by a power of two that no step passes, f32 by one that brings every value below 2^14
        float vs = 1.0f;
        uint32_t odd = 0;  // f32: whether a value is not finite
        if constexpr (INTS) {
            float most = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                if (!whole && j >= here) stv[j >> 2][j & 3] = 0.0f;
                most = fmaxf(most, stv[j >> 2][j & 3]);
            }
            most = half_max(row_max(most));
            const int e = most > 0.0f ? __builtin_amdgcn_frexp_expf(most) : -1000;
            if (e > ev) {
                const float f = ev > -1000 ? pow2(ev - e) : 0.0f;
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int m = 0; m < M; m++) acc[ct][m] *= f;
                ev = e;
            }
            vs = pow2(-max(ev, -126));
        } else {
            uint32_t most = 0;
#pragma unroll
            for (int m = 0; m < M; m++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (!whole && 4 * i + e >= here) vr[m].w[i][e] = 0;
                        odd = max(odd, vr[m].w[i][e] & 0x7fffffffu);
                        most = max(most, finite_bits(vr[m].w[i][e]));
                    }
            const int e = min(shift_for_max(wave_max(__uint_as_float(most))), 126);
            if (e < ev) {
                const float f = ev < 1000 ? pow2(e - ev) : 0.0f;
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int m = 0; m < M; m++) acc[ct][m] *= f;
                ev = e;
            }
            vs = pow2(ev);
        }
        halfx8 ph[CT][2], pl[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            float x[16];
            const float f = INTS ? to_log2[ct] : fminf(fmaxf(to_log2[ct] * unk, 0x1p-126f), 0x1p126f);
#pragma unroll
            for (int j = 0; j < 16; j++) {
                x[j] = sc[j >> 2][ct][j & 3];
                if constexpr (INTS) x[j] *= stk[j >> 2][j & 3];
            }
            if (!all_seen) {
                const int seen = min(here, min(max(limit[ct] - kv, 0), 16));
#pragma unroll
                for (int j = 0; j < 16; j++)
                    if (j >= seen) x[j] = -INFINITY;
            }
            float mb = x[0];
#pragma unroll
            for (int j = 1; j < 16; j++) mb = fmaxf(mb, x[j]);
            mb = half_max(row_max(mb)) * f;
            const bool grow = mb > ref[ct] + 3.0f;
            if (__any(grow)) {
                const float nref = grow ? mb : ref[ct];
                const float alpha = grow ? exp2_hw(ref[ct] - nref) : 1.0f;
                l[ct] *= alpha;
#pragma unroll
                for (int m = 0; m < M; m++) acc[ct][m] *= alpha;
                ref[ct] = nref;
            }
            const float off = ref[ct] == -INFINITY ? 0.0f : 12.0f - ref[ct];
#pragma unroll
            for (int s = 0; s < 2; s++) {
                u32x4 hw, lw;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int j = 8 * s + 2 * i;
                    float p0 = exp2_hw(fmaf(x[j], f, off)), p1 = exp2_hw(fmaf(x[j + 1], f, off));
                    l[ct] += p0 + p1;
                    if constexpr (INTS) {
                        p0 *= stv[j >> 2][j & 3] * vs;
                        p1 *= stv[j >> 2][(j + 1) & 3] * vs;
                    }
                    uint32_t a, b;
                    split2(p0, p1, a, b);
                    hw[i] = a;
                    lw[i] = b;
                }
                ph[ct][s] = __builtin_bit_cast(halfx8, hw);
                pl[ct][s] = __builtin_bit_cast(halfx8, lw);
            }
        }
        // values that are not finite: zeros in the products, and what sees one is no number
        if constexpr (!INTS) {
            if (__any(odd >= 0x7f800000u)) {
                const _Float16 one = (_Float16)1.0f, zero = (_Float16)0.0f;
#pragma unroll
                for (int m = 0; m < M; m++)
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        halfx8 bad;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const uint32_t w = vr[m].w[2 * s + (e >> 2)][e & 3];
                            const bool b = (w & 0x7fffffffu) >= 0x7f800000u;
                            bad[e] = b ? one : zero;
                            vr[m].w[2 * s + (e >> 2)][e & 3] = b ? 0u : w;
                        }
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) {
                            const int seen = min(here, min(max(limit[ct] - kv, 0), 16));
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
#pragma unroll
            for (int s = 0; s < 2; s++) {
                halfx8 hi, lo;
                to_halves<FMT>(vr[m], s, vs, hi, lo);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    acc[ct][m] = mfma(hi, ph[ct][s], acc[ct][m]);
                    acc[ct][m] = mfma(hi, pl[ct][s], acc[ct][m]);
                    if constexpr (LO) acc[ct][m] = mfma(lo, ph[ct][s], acc[ct][m]);
                }
            }
        }
    };
    // blocks b0 <= kb < b1 of the unit, every `step`th; those behind every column's limit are not looked at
    auto blocks = [&](int b0, int b1, int step) {
        ids0 = -64;
        b1 = min(b1, (lim_most + 63) >> 6);
        for (int kb = b0; kb < b1; kb += step) block(kb);
    };
    // acc over l is in units of this
    auto unit_value = [&] { return INTS ? (ev > -1000 ? pow2(ev) : 0.0f) : pow2(-min(ev, 149)); };

    seek(wg0);
    const uint32_t unit0 = (wg0 - before) / tw.nb, u0 = before + unit0 * tw.nb;
    if (wg1 <= u0 + tw.nb && wg1 - wg0 > 1) {
        // the workgroup's blocks are one unit's: its wavefronts take them in turn and join what they have
        begin(unit0);
        blocks((int)(wg0 - u0) + wave, (int)(wg1 - u0), WAVES);
        const bool done = wg0 == u0 && wg1 == u0 + tw.nb;
        const float unit = unit_value();
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const float lw = half_sum(row_sum(l[ct]));
            const float inv = lw > 0.0f ? 1.0f / lw : lw;  // 0 and NaN stay
            if (lg == 0) {
                mref[wave][16 * ct + qi] = ref[ct];
                msum[wave][16 * ct + qi] = lw;
            }
            if (ct) __syncthreads();
#pragma unroll
            for (int m = 0; m < M; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) macc[wave][16 * m + 4 * lg + i][qi] = acc[ct][m][i] * inv * unit;
            __syncthreads();
            // thread t: column t / 32, coordinates t % 32 + 32 ..
            const int c16 = tid >> 5, col = 16 * ct + c16;
            float m = -INFINITY, L = 0.0f, f[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; w++)
                if (msum[w][col] > 0.0f) m = fmaxf(m, mref[w][col]);
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float s = msum[w][col];
                f[w] = s > 0.0f ? s * exp2_hw(mref[w][col] - m) : s;
                L += f[w];
            }
            const float Li = L > 0.0f ? 1.0f / L : L;
            const int at = tile * COLS + col, i = at / group;
            const size_t slot = 2 * (size_t)(blockIdx.x * WAVES);
            for (int dim = tid & 31; dim < hd; dim += 32) {
                float o = 0.0f;
#pragma unroll
                for (int w = 0; w < WAVES; w++)
                    if (msum[w][col] != 0.0f) o += f[w] * macc[w][dim][c16];
                o *= Li;
                if (done) {
                    if (i < tw.n) out[(size_t)(tw.first + i) * heads * hd + (size_t)(h * group + at - i * group) * hd + dim] = o;
                } else {
                    parts.o[(slot * COLS + col) * hd + dim] = o;
                }
            }
            if (!done && (tid & 31) < WAVES)
                parts.ml[(slot + 2 * (tid & 31)) * COLS + col] = (tid & 31) ? make_float2(-INFINITY, 0.0f) : make_float2(m, L);
        }
        return;
    }
    // every wavefront its own blocks
    uint32_t at = wg0 + wave * per;
    const uint32_t end = min(total, at + per);
    const uint32_t mine = at;
    while (at < end) {
        seek(at);
        const uint32_t unit = (at - before) / tw.nb, b0 = at - before - unit * tw.nb;
        const uint32_t b1 = min((uint32_t)tw.nb, b0 + (end - at));
        begin(unit);
        blocks((int)b0, (int)b1, 1);
        const bool done = b0 == 0 && b1 == (uint32_t)tw.nb;
        const float uv = unit_value();
        const size_t slot = 2 * (size_t)me + (at == mine ? 0 : 1);
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const float lw = half_sum(row_sum(l[ct]));
            const float inv = lw > 0.0f ? 1.0f / lw : lw;
            const int col = 16 * ct + qi, c = tile * COLS + col, i = c / group;
            if (done && i >= tw.n) continue;
            float *dst = done ? out + (size_t)(tw.first + i) * heads * hd + (size_t)(h * group + c - i * group) * hd
                              : parts.o + (slot * COLS + col) * hd;
#pragma unroll
            for (int m = 0; m < M; m++)
                if (16 * m < hd) {
                    floatx4 o = acc[ct][m] * inv * uv;
                    *reinterpret_cast<floatx4u *>(dst + 16 * m + 4 * lg) = o;
                }
            if (!done && lg == 0) parts.ml[slot * COLS + col] = make_float2(ref[ct], lw);
        }
        at += b1 - b0;
    }
}

// grid (queries x heads); 256 threads: the states that wavefronts left of one query and head, together. A unit that one run held
// whole has its output already.
template <int CT>
__global__ __launch_bounds__(256) void k_pages_join(PageSet p, const int32_t *__restrict__ lengths, const int32_t *__restrict__ offsets,
                                                    int nq, int heads, uint32_t waves, float *__restrict__ out, Parts parts) {
    constexpr int COLS = 16 * CT;
    __shared__ float wm[4], wl[4], wo[4][128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = heads / p.heads, hd = p.hd;
    const int r = blockIdx.x / heads, head = blockIdx.x - r * heads;
    // the table of the query: so many tables' queries end at or before it
    int t = 0;
    for (int t0 = 0; t0 < p.tables - 1; t0 += 64) t += __popcll(__ballot(t0 + lane < p.tables - 1 && offsets[t0 + lane + 1] <= r));
    const TableWork tw = table_work(p, lengths, offsets, nq, group, COLS, t);
    if (r < tw.first || r >= tw.first + tw.n) return;
    const uint32_t per = parts.plan[0], total = parts.plan[1 + p.tables];
    if (total == 0) return;
    const int h = head / group, c = (r - tw.first) * group + head - h * group, tile = c / COLS, col = c - tile * COLS;
    const uint32_t u0 = parts.plan[1 + t] + ((uint32_t)tile * p.heads + h) * tw.nb, u1 = u0 + tw.nb;
    const uint32_t w0 = u0 / per, w1 = (u1 - 1) / per;
    if (w0 == w1) return;
    if (u0 % per == 0 && w0 % WAVES == 0 && u1 <= (w0 + WAVES) * per) {
        // one workgroup may have held it whole, with its wavefronts in turn
        const uint32_t wg0 = w0 * per, wg1 = min(total, wg0 + WAVES * per);
        if (wg1 == u1) return;
    }
    float M = -INFINITY, L = 0.0f, o[2] = {0.0f, 0.0f};
    for (uint32_t b = w0 + 64 * wave; b <= w1; b += 256) {
        const uint32_t w = b + lane;
        const size_t slot = 2 * (size_t)w + (w == w0 && u0 > w0 * per ? 1 : 0);
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (w <= w1) ml = parts.ml[slot * COLS + col];
        const float m = wave_max(ml.y > 0.0f ? ml.x : -INFINITY);
        const float top = fmaxf(M, m);
        const float f = ml.y > 0.0f ? ml.y * exp2_hw(ml.x - top) : ml.y;
        const float old = M == -INFINITY ? 0.0f : exp2_hw(M - top);
        L *= old;
        o[0] *= old;
        o[1] *= old;
        M = top;
        uint64_t live = __ballot(ml.y != 0.0f);
        while (live) {
            const int j = __ffsll((unsigned long long)live) - 1;
            live &= live - 1;
            const float fj = __shfl(f, j);
            const size_t sj = 2 * (size_t)(b + j) + (b + j == w0 && u0 > w0 * per ? 1 : 0);
            const float *src = parts.o + (sj * COLS + col) * hd;
            L += fj;
            if (lane < hd) o[0] += fj * src[lane];
            if (64 + lane < hd) o[1] += fj * src[64 + lane];
        }
    }
    wo[wave][lane] = o[0];
    wo[wave][64 + lane] = o[1];
    if (lane == 0) {
        wm[wave] = M;
        wl[wave] = L;
    }
    __syncthreads();
    if (wave > 0) return;
    const float top = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    L = o[0] = o[1] = 0.0f;
    for (int w = 0; w < 4; w++) {
        if (wl[w] == 0.0f) continue;
        const float f = wm[w] == -INFINITY ? 1.0f : exp2_hw(wm[w] - top);
        L += wl[w] * f;
        o[0] += wo[w][lane] * f;
        o[1] += wo[w][64 + lane] * f;
    }
    const float inv = L > 0.0f ? 1.0f / L : L;
    float *dst = out + (size_t)r * heads * hd + (size_t)head * hd;
    if (lane < hd) dst[lane] = o[0] * inv;
    if (64 + lane < hd) dst[64 + lane] = o[1] * inv;
}

// Sets of 16 columns that share what a wavefront reads, and the workgroups: one a compute unit, fewer where there may not be a
// block for each of their wavefronts.
struct Shape {
    int sets, wgs;
    size_t o_floats, ml_count;
    uint64_t blocks;  // at most
};

Shape shape(const PageSet &p, int nq, int heads) {
    Shape s;
    const int64_t group = heads / p.heads, columns = (int64_t)nq * group;
    s.sets = columns > 16 * (int64_t)p.tables ? 2 : 1;
    const uint64_t rows = std::min((uint64_t)p.ld << p.log_rows, (uint64_t)0x7fffffff - 64);
    const uint64_t units = ((uint64_t)std::min(p.tables, nq) + columns / (16 * s.sets)) * p.heads;
    const uint64_t nb = std::max<uint64_t>(1, (rows + 63) / 64);
    s.blocks = units > (uint64_t(1) << 32) ? ~uint64_t(0) : units * nb;
    s.wgs = (int)std::min<uint64_t>(256, (s.blocks + WAVES - 1) / WAVES);
    const size_t slots = 2 * (size_t)s.wgs * WAVES;
    s.o_floats = slots * 16 * s.sets * p.hd;
    s.ml_count = slots * 16 * s.sets;
    return s;
}

template <int FMT, int C, int CT>
void launch(hipStream_t s, const PageSet &p, const int32_t *lengths, const float *q, const int32_t *offsets, int nq, int heads,
            bool causal, size_t q_ld, float *out, const Parts &parts, const Shape &sh) {
    hipLaunchKernelGGL((k_pages_attend<FMT, C, CT>), dim3(sh.wgs), dim3(64 * WAVES), 0, s, p, lengths, q, offsets, nq,
                       heads, causal ? 1 : 0, q_ld, out, parts, sh.blocks);
    TAH_LAUNCHED();
    hipLaunchKernelGGL(k_pages_join<CT>, dim3((unsigned)nq * heads), dim3(256), 0, s, p, lengths, offsets, nq, heads,
                       (uint32_t)sh.wgs * WAVES, out, parts);
    TAH_LAUNCHED();
}

template <int FMT, int C>
void launch_sets(hipStream_t s, const PageSet &p, const int32_t *lengths, const float *q, const int32_t *offsets, int nq,
                 int heads, bool causal, size_t q_ld, float *out, const Parts &parts, const Shape &sh) {
    if (sh.sets == 1)
        launch<FMT, C, 1>(s, p, lengths, q, offsets, nq, heads, causal, q_ld, out, parts, sh);
    else
        launch<FMT, C, 2>(s, p, lengths, q, offsets, nq, heads, causal, q_ld, out, parts, sh);
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

}  // namespace

size_t pages_attend_work_bytes(const PageSet &p, int nq, int heads) {
    const Shape s = shape(p, nq, heads);
    // the kernels number all units' blocks in 32 bits
    if (s.blocks >= (uint64_t(1) << 31)) throw ArgError{"pages_attend: more rows than a call takes: fewer tables a call"};
    return up256(s.o_floats * sizeof(float)) + up256(s.ml_count * sizeof(float2)) + up256(((size_t)p.tables + 2) * sizeof(uint32_t));
}

void pages_attend(hipStream_t s, int fmt, const PageSet &p, const int32_t *lengths, const float *q, const int32_t *offsets, int nq,
                  int heads, bool causal, size_t q_ld, float *out, void *work) {
    const Shape sh = shape(p, nq, heads);
    uint8_t *at = static_cast<uint8_t *>(work);
    Parts parts;
    parts.o = reinterpret_cast<float *>(at);
    parts.ml = reinterpret_cast<float2 *>(at += up256(sh.o_floats * sizeof(float)));
    parts.plan = reinterpret_cast<uint32_t *>(at + up256(sh.ml_count * sizeof(float2)));
    auto with = [&](auto f) {
        constexpr int FMT = decltype(f)::value;
        if (p.hd <= 64)
            launch_sets<FMT, 1>(s, p, lengths, q, offsets, nq, heads, causal, q_ld, out, parts, sh);
        else
            launch_sets<FMT, 2>(s, p, lengths, q, offsets, nq, heads, causal, q_ld, out, parts, sh);
    };
    if (fmt == TAH_KV_F32)
        with(std::integral_constant<int, TAH_KV_F32>{});
    else if (fmt == TAH_KV_I16)
        with(std::integral_constant<int, TAH_KV_I16>{});
    else
        with(std::integral_constant<int, TAH_KV_I8>{});
}

}  // namespace tah
