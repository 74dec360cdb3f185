// lmr_rows.hip — batched load / add / store of whole rows: the records of a batch are rows of a
// table (row_len elements each) instead of single elements.
//
//   lmr_rows_load    out[t, :] = rnd(scale * table[i[t], :])            (an embedding lookup; an
//                    8-bit cache read back: element = code * scale of its group)
//   lmr_rows_add     table[r, :] = rnd(table[r, :] + scale * sum of vals[t, :] over i[t] = r)
//                    (the lookup's gradient; every collision counted, in a fixed order)
//   lmr_rows_store   table[i[t], :] = rnd(vals[t, :]), the last record of a row wins; 8-bit tables
//                    take codes and one f32 scale per group, both of the same record
//
// Arithmetic is f32; each result is rounded once, to the nearest even, when it is written: a row is read
// and written in its own type, so a sum over a whole batch must not round in between.
//
// All of it is bound by memory where a batch is large (a copy of 1 GiB runs at 5.0 TB/s on the card that
// the times below are from) and by launches where it is small.
#include "lmr_internal.hpp"
#include "lmr_rows.hpp"
#include <algorithm>
#include <tuple>

namespace lmr {
namespace {

template <int IW>
__device__ __forceinline__ int64_t row_index(const RowBatch& b, uint64_t t) {
    if constexpr (IW == 4) return reinterpret_cast<const int32_t*>(b.idx)[t];
    else return reinterpret_cast<const int64_t*>(b.idx)[t];
}

// whether index i names a row; one that is neither a row nor a pad is reported (by `lead` threads)
__device__ __forceinline__ bool is_row(const RowBatch& b, int64_t i, uint64_t rows, uint32_t* err, bool lead) {
    if (b.has_pad && i == b.pad) return false;
    if (uint64_t(i) < rows) return true;
    if (lead) atomicOr(err, LMR_ERRBIT_OOB);
    return false;
}

// the record's row, or -1: a pad, or out of bounds (reported by `lead` threads)
template <int IW>
__device__ __forceinline__ int64_t row_of(const RowBatch& b, uint64_t t, uint64_t rows, uint32_t* err, bool lead) {
    const int64_t i = row_index<IW>(b, t);
    return is_row(b, i, rows, err, lead) ? i : -1;
}

// A thread moves U chunks of 8 elements. The batch's chunks are numbered row after row and dealt to
// blocks in runs of 256 U, so that any row length fills the lanes; the row of a chunk is a division by
// the row's chunks (one in 64 bits per block, one in 32 per chunk, both multiplications). The result is
// written past the caches' reuse order: it is as large as the table's rows or larger, and read once
// (65536 bf16 rows of 4096: 142 us against 159 through the caches, and 158, 144, 142, 146 us with U = 1,
// 2, 4, 8). Now 134 us, 5.3 TB/s (medians here and below); 262144 e4m3 rows of 1024 to bf16 142 us, 5.7 TB/s;
// 16 rows 2.6 us. Groups that are no multiple of 8 (65536 e4m3 rows of 1000, groups of 100) 37 us, 5.4 TB/s.
// GA: groups of a multiple of 8 elements, so that a chunk has one scale.
template <typename T, typename O, int IW, int U, bool GA>
__global__ __launch_bounds__(256) void k_rows_load(RowTable tab, RowBatch b, O* out, uint32_t* err, Divisor cpr, Divisor cpg) {
    const uint64_t base = uint64_t(blockIdx.x) * (256 * U);
    const uint64_t row0 = quotient64(base, cpr);
    const uint32_t rem = uint32_t(base - row0 * cpr.d) + threadIdx.x, n = uint32_t(b.n) - uint32_t(row0);
    using I = std::conditional_t<IW == 4, int32_t, int64_t>;
    const I* idx = reinterpret_cast<const I*>(b.idx) + row0;
    out += row0 * b.stride;
    uint32_t t[U], c[U], col[U];                         // record, chunk of it, where that begins
    I r[U];
    bool live[U];
    // (each step for all U before the next, and no load under a condition that another load decides:
    // the loads of a step are in flight together)
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t off = rem + u * 256;
        t[u] = quotient32(off, cpr);
        c[u] = off - t[u] * cpr.d;
        col[u] = span_of(c[u], tab.row_len).at;
        r[u] = idx[min(t[u], n - 1)];
    }
#pragma unroll
    for (int u = 0; u < U; u++) live[u] = t[u] < n && is_row(b, r[u], tab.rows, err, c[u] == 0);
    Chunk<T> x[U];
    float sc[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint64_t row = uint32_t(r[u]);             // (a table has fewer rows than 2^32)
        if constexpr (is_code<T>::v && GA)
            sc[u] = *(live[u] ? tab.scales + row * tab.groups + quotient32(c[u], cpg) : reinterpret_cast<const float*>(b.idx));
        x[u] = fetch(reinterpret_cast<const T*>(tab.data) + row * tab.row_len, col[u], tab.row_len, live[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (t[u] >= n) continue;
        float v[kChunk];
        unpack(x[u], v);
        if constexpr (is_code<T>::v && !GA) {
            if (live[u]) {
                const uint32_t g = col[u] / tab.group;
                const float* sc = tab.scales + uint64_t(uint32_t(r[u])) * tab.groups + g;
                uint32_t left = (g + 1) * tab.group - col[u];                 // elements of this group from here
                float s = *sc;
#pragma unroll
                for (int i = 0; i < kChunk; i++) {
                    if (left == 0) {
                        left = tab.group;
                        if (col[u] + i < tab.row_len) s = *++sc;
                    }
                    left--;
                    v[i] *= s;
                }
            }
        }
        // (the code's product first: scale times a group's scale may leave f32's range where the result does not)
        if constexpr (is_code<T>::v && GA) {
            const float s = live[u] ? sc[u] : 0.f;
#pragma unroll
            for (int i = 0; i < kChunk; i++) v[i] *= s;
        }
        const float m = live[u] ? b.scale : 0.f;         // (times a chunk of zeros)
#pragma unroll
        for (int i = 0; i < kChunk; i++) v[i] *= m;
        O* p = out + uint64_t(t[u]) * b.stride;
        if (tab.row_len >= kChunk) stream_chunk(p + col[u], pack<O>(v));
        else put(p, 0, tab.row_len, pack<O>(v));
    }
}

template <bool WHOLE = false, typename T>
__device__ __forceinline__ void add_to_row(T* row, const Span& sp, Chunk<T> old, const float (&acc)[kChunk], float scale) {
    float v[kChunk];
    unpack(old, v);
#pragma unroll
    for (int i = 0; i < kChunk; i++) v[i] = fmaf(scale, acc[i], v[i]);
    if constexpr (WHOLE) store_chunk(row + sp.at, pack<T>(v));
    else put_own(row, sp, pack<T>(v));
}

// ---------------------------------------------------------------- add, few records
// One launch: a block per record and 512 columns. Each wave finds the record's row in the whole list (MOST
// indices at most); a record with an earlier one of its row leaves. The first sums the row's records in
// order, its four waves a quarter each where there are more than four. The blocks' number and their work
// both grow with the batch (add_plan says how far): 512 records of 1024 4.9 us, 8.6 sorted; 1024 of 1024
// 8.9 and 9.7; 512 of 4096 10.2 and 9.9; 600 of 2048 10.1 and 9.3, 1024 15.4 and 10.2.
template <typename T, typename V, int IW, int MOST>
__global__ __launch_bounds__(256) void k_rows_add_few(RowTable tab, RowBatch b, const V* vals, uint32_t* err) {
    __shared__ uint16_t list[MOST];
    __shared__ float sum[3][64][kChunk + 1];
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t r = row_of<IW>(b, t, tab.rows, err, threadIdx.x == 0 && blockIdx.y == 0);
    if (r < 0) return;
    const Span sp = span_of(blockIdx.y * 64 + lane, tab.row_len);
    const bool on = sp.lo < sp.hi;
    T* row = reinterpret_cast<T*>(tab.data) + uint64_t(r) * tab.row_len;
    const Chunk<T> old = fetch(row, sp.at, tab.row_len, on && w == 0);
    uint32_t total = 0;
    bool hit[MOST / 64], earlier = false;
#pragma unroll
    for (int i = 0; i < MOST / 64; i++) {
        const uint32_t u = i * 64 + lane;
        hit[i] = u < b.n && row_index<IW>(b, u) == r;
        earlier |= hit[i] && u < t;
    }
    if (__ballot(earlier)) return;                                 // (alike in every wave)
#pragma unroll
    for (int i = 0; i < MOST / 64; i++) {
        const uint64_t m = __ballot(hit[i]);
        if (hit[i] && w == 0) list[total + __popcll(m & ((1ull << lane) - 1))] = uint16_t(i * 64 + lane);
        total += __popcll(m);
    }
    __syncthreads();
    const uint32_t share = total > 4 ? (total + 3) / 4 : total;
    const uint32_t j0 = min(total, w * share), j1 = min(total, j0 + share);
    float acc[kChunk] = {};
    constexpr int U = 4;
    for (uint32_t j = j0; j < j1; j += U) {
        Chunk<V> c[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t rec = list[min(j + u, total - 1)];
            c[u] = fetch(vals + uint64_t(rec) * b.stride, sp.at, tab.row_len, on && j + u < j1);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float v[kChunk];
            unpack(c[u], v);
#pragma unroll
            for (int i = 0; i < kChunk; i++) acc[i] += v[i];
        }
    }
    if (total > 4) {
        if (w > 0) {
#pragma unroll
            for (int i = 0; i < kChunk; i++) sum[w - 1][lane][i] = acc[i];
        }
        __syncthreads();
        if (w == 0) {
#pragma unroll
            for (int o = 0; o < 3; o++)
#pragma unroll
                for (int i = 0; i < kChunk; i++) acc[i] += sum[o][lane][i];
        }
    }
    if (w == 0 && on) add_to_row(row, sp, old, acc, b.scale);
}

// ---------------------------------------------------------------- add, many records
// The records sorted by row (and by place inside a row), then summed run by run.
//
// Sort of many: least significant digit first, digits of up to 10 bits. A pass is two launches: each block
// counts the digits of its tile, then places its tile behind what earlier tiles and lower digits
// take. Records keep their order among equal digits: a wave ranks its 64 records by ballots, waves
// and tiles follow one another in order. Bound by the latency of its launches (a pass over 131072 records
// 14 us), so tiles are small while they are few (whole batches of 16 columns in tiles of 1024, 2048, 4096, 8192:
// 262144 records 43.9, 46.5, 51.9, 63.6 us, 600000 71.0, 69.0, 69.4, 83.5, 2 million 239, 219, 211, 218,
// 8 million 815, 736, 695, 696). With more than 64 tiles a launch of its own adds up their counts: 65536
// records of 64 columns 34.6 us with it, 33.9 without, 300000 51 us with it, 74 in tiles large enough to do without.
constexpr int kSortThreads = 512;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kSortBits = 10;
constexpr uint32_t kNoRow = 0xffffffffu;

struct SortPass {
    const uint2* in;      // (row, record); null: the batch's indices
    uint2* out;
    uint32_t* hist;       // [tiles][1 << bits], then the digits' totals
    uint32_t n, shift, bits, tiles;
    bool summed;          // hist holds prefixes over the tiles (k_rows_prefix)
    uint32_t* joins;      // the count to clear for k_rows_sum, in the first launch
};

template <int IW>
__device__ __forceinline__ uint2 sort_record(const SortPass& p, const RowBatch& b, const RowTable& tab, uint32_t* err, uint32_t j) {
    if (p.in) return p.in[j];
    const int64_t r = row_of<IW>(b, j, tab.rows, err, true);
    return {r < 0 ? uint32_t(tab.rows) : uint32_t(r), j};          // skipped records sort behind every row
}

template <int IW, int IPT>
__global__ __launch_bounds__(kSortThreads) void k_rows_count(SortPass p, RowBatch b, RowTable tab, uint32_t* err) {
    __shared__ uint32_t cnt[1 << kSortBits];
    const uint32_t nd = 1u << p.bits;
    if (!p.in && blockIdx.x == 0 && threadIdx.x == 0) *p.joins = 0;
    for (uint32_t d = threadIdx.x; d < nd; d += kSortThreads) cnt[d] = 0;
    __syncthreads();
    const uint32_t j0 = blockIdx.x * (kSortThreads * IPT) + threadIdx.x;
#pragma unroll
    for (int k = 0; k < IPT; k++) {
        const uint32_t j = j0 + k * kSortThreads;
        if (j < p.n) atomicAdd(&cnt[(sort_record<IW>(p, b, tab, err, j).x >> p.shift) & (nd - 1)], 1u);
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < nd; d += kSortThreads) p.hist[uint64_t(blockIdx.x) * nd + d] = cnt[d];
}

// many tiles: each digit's counts become the counts of the tiles before, the totals go behind them. A block
// has 64 digits, its 16 waves a sixteenth of the tiles each: their sums first, then the counts again
__global__ __launch_bounds__(1024) void k_rows_prefix(SortPass p) {
    __shared__ uint32_t part[16][64];
    const uint32_t nd = 1u << p.bits, lane = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
    const uint32_t share = (p.tiles + 15) / 16, t0 = min(p.tiles, w * share), t1 = min(p.tiles, t0 + share);
    constexpr int U = 16;                                          // reads in flight
    uint32_t sum = 0;
    if (d < nd)
        for (uint32_t t = t0; t < t1; t += U) {
            uint32_t c[U];
#pragma unroll
            for (int i = 0; i < U; i++) c[i] = p.hist[uint64_t(min(t + i, t1 - 1)) * nd + d];
#pragma unroll
            for (int i = 0; i < U; i++) sum += t + i < t1 ? c[i] : 0;
        }
    part[w][lane] = sum;
    __syncthreads();
    sum = 0;
    for (uint32_t i = 0; i < w; i++) sum += part[i][lane];
    if (d >= nd) return;
    for (uint32_t t = t0; t < t1; t += U) {
        uint32_t c[U];
#pragma unroll
        for (int i = 0; i < U; i++) c[i] = p.hist[uint64_t(min(t + i, t1 - 1)) * nd + d];
#pragma unroll
        for (int i = 0; i < U; i++) {
            if (t + i >= t1) continue;
            p.hist[uint64_t(t + i) * nd + d] = sum;
            sum += c[i];
        }
    }
    if (w == 15) p.hist[uint64_t(p.tiles) * nd + d] = sum;
}

// the lanes of the wave whose digit is this lane's: a ballot per bit, kept where it agrees
__device__ __forceinline__ uint64_t same_digit(uint32_t d, bool live) {
    const uint64_t all = __ballot(live);
    uint32_t lo = uint32_t(all), hi = uint32_t(all >> 32);
#pragma unroll
    for (int i = 0; i < kSortBits; i++) {
        const uint32_t one = uint32_t(int32_t(d << (31 - i)) >> 31);          // all ones or none
        const uint64_t m = __ballot(one != 0);
        lo &= ~(uint32_t(m) ^ one);
        hi &= ~(uint32_t(m >> 32) ^ one);
    }
    return uint64_t(hi) << 32 | lo;
}
__device__ __forceinline__ uint32_t lanes_below(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi(uint32_t(m >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(m), 0));
}

template <int IW, int IPT>
__global__ __launch_bounds__(kSortThreads) void k_rows_place(SortPass p, RowBatch b, RowTable tab, uint32_t* err) {
    __shared__ uint32_t cnt[kSortWaves][1 << kSortBits];
    __shared__ uint32_t base[1 << kSortBits];
    __shared__ uint32_t wsum[kSortWaves];
    const uint32_t nd = 1u << p.bits, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (uint32_t d = lane; d < nd; d += 64) cnt[w][d] = 0;
    // what lies before this tile's records of a digit: thread x has digits 2x and 2x + 1
    uint32_t before[2] = {0, 0}, total[2] = {0, 0};
    if (2 * threadIdx.x < nd) {
        const uint2* h = reinterpret_cast<const uint2*>(p.hist) + threadIdx.x;
        if (p.summed) {
            const uint2 c = h[uint64_t(blockIdx.x) * (nd / 2)], e = h[uint64_t(p.tiles) * (nd / 2)];
            before[0] = c.x, before[1] = c.y, total[0] = e.x, total[1] = e.y;
        } else {
            for (uint32_t t = 0; t < p.tiles; t += 16) {           // (16 reads in flight, the last ones again)
                uint2 c[16];
#pragma unroll
                for (int i = 0; i < 16; i++) c[i] = h[min(t + i, p.tiles - 1) * (nd / 2)];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    if (t + i >= p.tiles) continue;
                    if (t + i < blockIdx.x) before[0] += c[i].x, before[1] += c[i].y;
                    total[0] += c[i].x, total[1] += c[i].y;
                }
            }
        }
    }
    uint32_t run = total[0] + total[1];                            // exclusive scan over the threads
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const uint32_t o = __shfl_up(run, s, 64);
        if (int(lane) >= s) run += o;
    }
    if (lane == 63) wsum[w] = run;
    __syncthreads();
    uint32_t lower = run - total[0] - total[1];
    for (uint32_t i = 0; i < w; i++) lower += wsum[i];
    if (2 * threadIdx.x < nd) {
        base[2 * threadIdx.x] = lower + before[0];
        base[2 * threadIdx.x + 1] = lower + total[0] + before[1];
    }
    // a wave's records are neighbours: IPT rounds of 64
    const uint32_t j0 = blockIdx.x * (kSortThreads * IPT) + w * (64 * IPT) + lane;
    uint2 rec[IPT];
    uint32_t rank[IPT];
#pragma unroll
    for (int k = 0; k < IPT; k++)
        rec[k] = j0 + k * 64 < p.n ? sort_record<IW>(p, b, tab, err, j0 + k * 64) : uint2{kNoRow, 0};
#pragma unroll
    for (int k = 0; k < IPT; k++) {
        const bool live = j0 + k * 64 < p.n;
        const uint32_t d = (rec[k].x >> p.shift) & (nd - 1);
        const uint64_t same = same_digit(d, live);
        const uint32_t below = lanes_below(same);
        const uint32_t had = live ? cnt[w][d] : 0;
        rank[k] = had + below;
        __builtin_amdgcn_wave_barrier();                           // every lane has read before one writes
        if (live && below == 0) cnt[w][d] = had + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < nd; d += kSortThreads) {    // waves in order behind the tile's base
        uint32_t at = base[d];
#pragma unroll
        for (int i = 0; i < kSortWaves; i++) {
            const uint32_t c = cnt[i][d];
            cnt[i][d] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < IPT; k++) {
        const uint32_t to = cnt[w][(rec[k].x >> p.shift) & (nd - 1)] + rank[k];
        if (j0 + k * 64 < p.n && to < p.n) p.out[to] = rec[k];     // (indices changed under way: still in bounds)
    }
}

// Up to kRankMost records: one launch, in which each block counts, for the records of its own, how many of
// the whole list come before them: rows below theirs, and equal rows of earlier records. The list stands in
// LDS; a thread compares four of its rows at a time with R records' (a record's count from `shares` threads).
// Bound by n^2 comparisons of two instructions, 64 at a time, spread over all compute units: a block has a
// 256th of the records, at least 16. Sums of 64 columns: 1500 records 10.4 us, 13.4 with a sort by digits in
// one block, 5003 13.3 and 19.9, 8192 17.1 and 15.1 with k_rows_merge (5003 in blocks of 32: 14.4; 8192 in
// blocks of 16 19.3, of 64 22.7, with one record a thread 18.5).
constexpr uint32_t kRankMost = 6144;

// (TILE: the records of the block's tile of the list, not the whole list)
template <int IW, uint32_t TILE>
__global__ __launch_bounds__(1024) void k_rows_rank(SortPass p, uint32_t part, RowBatch b, RowTable tab, uint32_t* err) {
    constexpr int R = 2, U = 4;                                    // a thread's records, its reads in flight
    __shared__ uint4 rows_at[TILE / 4];
    __shared__ uint32_t rank[64];
    const uint32_t base = blockIdx.x * part / TILE * TILE, count = min(TILE, p.n - base), padded = (count + 3) & ~3u;
    const uint32_t first = blockIdx.x * part - base, wide = part / R;
    const uint32_t mine = threadIdx.x % wide * R, share = threadIdx.x / wide, shares = 1024 / wide;
    uint32_t* const row_at = reinterpret_cast<uint32_t*>(rows_at);
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.joins = 0;
    if (threadIdx.x < part) rank[threadIdx.x] = 0;
    for (uint32_t j0 = threadIdx.x; j0 < padded; j0 += 1024 * U) {
        uint32_t row[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t j = j0 + u * 1024;
            const int64_t r = j < count ? row_of<IW>(b, base + j, tab.rows, err, j - first < part) : 0;
            row[u] = j >= count ? kNoRow : r < 0 ? uint32_t(tab.rows) : uint32_t(r);     // (kNoRow is below none)
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (j0 + u * 1024 < padded) row_at[j0 + u * 1024] = row[u];
    }
    __syncthreads();
    uint32_t row[R], before[R];
#pragma unroll
    for (int k = 0; k < R; k++) {
        const uint32_t i = first + mine + k;
        row[k] = i < count ? row_at[i] : 0;
        before[k] = 0;
    }
#pragma unroll 4
    for (uint32_t c = share < shares ? share : padded; c < padded / 4; c += shares) {
        const uint4 r = rows_at[c];
#pragma unroll
        for (int k = 0; k < R; k++) {
            const uint32_t limit = row[k] + (c * 4 < first + mine + k);                // equal rows count too
            before[k] += (r.x < limit) + (r.y < limit) + (r.z < limit) + (r.w < limit);
        }
    }
#pragma unroll
    for (int k = 0; k < R; k++) {
        const uint32_t i = first + mine + k;
        if (share == 0 && i < count && i % 4)                        // but for the record itself and its four's later ones
            for (uint32_t j = i; j <= (i | 3); j++) before[k] -= row_at[j] == row[k];
        atomicAdd(&rank[mine + k], before[k]);
    }
    __syncthreads();
    if (share != 0) return;
#pragma unroll
    for (int k = 0; k < R; k++) {
        const uint32_t i = first + mine + k;
        if (i >= count) continue;
        const uint32_t to = base + rank[mine + k];
        if constexpr (TILE == kRankMost) {
            p.out[to] = {row[k], i};
        } else {
            uint32_t* const rows = reinterpret_cast<uint32_t*>(p.out);                 // for k_rows_merge
            rows[to] = row[k];
            rows[p.n + to] = base + i;
        }
    }
}

// Up to kMergeMost records: tiles of kMergeTile sorted as above, then each record's place is its own in its
// tile and, by binary search in LDS, what the other tiles have below it (equal rows of earlier tiles too).
// Two launches, bound by their latency. Sums of 64 columns: 8192 records 15.1 us, 20.1 by digits, 16384 16.0
// and 22.2, 32768 21.9 and 27.6 (in tiles of 512 14.4, 16.1, 23.4, of 2048 16.7, 17.6, 26.6).
constexpr uint32_t kMergeMost = 32768;
constexpr uint32_t kMergeTile = 1024;

__global__ __launch_bounds__(1024) void k_rows_merge(SortPass p, uint32_t part) {
    __shared__ uint4 rows_at[kMergeMost / 4];
    __shared__ uint32_t rank[kMergeMost / 256];
    const uint32_t* const rows = reinterpret_cast<const uint32_t*>(p.in);              // n rows, then their records
    const uint32_t* const row_at = reinterpret_cast<const uint32_t*>(rows_at);
    const uint32_t first = blockIdx.x * part;
    if (threadIdx.x < part) rank[threadIdx.x] = 0;
    constexpr int U = 4;                                           // reads in flight
    for (uint32_t c0 = threadIdx.x; c0 * 4 < p.n; c0 += 1024 * U) {
        uint4 r[U];
#pragma unroll
        for (int u = 0; u < U; u++) r[u] = reinterpret_cast<const uint4*>(rows)[min(c0 + u * 1024, (p.n - 1) / 4)];
#pragma unroll
        for (int u = 0; u < U; u++)
            if ((c0 + u * 1024) * 4 < p.n) rows_at[c0 + u * 1024] = r[u];
    }
    __syncthreads();
    const uint32_t tiles = (p.n + kMergeTile - 1) / kMergeTile;
    for (uint32_t x = threadIdx.x; x < part * tiles; x += 1024) {
        const uint32_t mine = x % part, tile = x / part, i = first + mine, base = tile * kMergeTile;
        if (i >= p.n) continue;
        uint32_t below = i - base;
        if (tile != i / kMergeTile) {
            const uint32_t limit = row_at[i] + (base < i), count = min(kMergeTile, p.n - base);
            below = 0;
#pragma unroll
            for (uint32_t step = kMergeTile; step; step /= 2)
                if (below + step <= count && row_at[base + below + step - 1] < limit) below += step;
        }
        atomicAdd(&rank[mine], below);
    }
    __syncthreads();
    const uint32_t i = first + threadIdx.x;
    if (threadIdx.x < part && i < p.n) p.out[rank[threadIdx.x]] = {row_at[i], rows[p.n + i]};
}

// Sum: a group of LPR lanes (8 elements each) takes a tile of K neighbours of the sorted records. A row
// whose records begin in the tile and end there or in the next one is summed by this group alone and
// added to the table at once. Only longer runs are cut: their parts go to `last` (the tile in which
// they begin) and `first` (every later one), and k_rows_join adds them up. Every value is read once and
// every named row read and written once: 131072 bf16 records of 4096 into f32 take 446 us here (4.9 TB/s
// of the 2.2 GB that must move) of 496 in all.
struct SumArgs {
    const uint2* rec;     // sorted (row, record)
    float* first;         // [tiles][pitch]
    float* last;
    uint32_t* joins;      // [0]: rows to join, [1 ..]: the tiles in which they begin, in any order
    uint32_t n, k, tiles, pitch;
    uint32_t lanes;       // of a row's part in k_rows_join
    Divisor chunks;       // column chunks of k_rows_sum
};

// (WHOLE: rows of a multiple of 8 elements, whose chunks do not overlap. U: records whose values are in
// flight together)
template <typename T, typename V, int LPR, bool WHOLE, int U>
__global__ __launch_bounds__(256) void k_rows_sum(RowTable tab, RowBatch b, const V* vals, SumArgs a) {
    constexpr bool kLong = WHOLE || LPR > 8;                       // (shorter rows take the fewest lanes)
    uint32_t gid = (blockIdx.x * 256u + threadIdx.x) / LPR;
    if constexpr (LPR == 64) gid = __builtin_amdgcn_readfirstlane(gid);
    const uint32_t tile = uint32_t(quotient64(gid, a.chunks));
    if (tile >= a.tiles) return;
    const uint32_t chunk = (gid - tile * a.chunks.d) * LPR + threadIdx.x % LPR;
    const Span sp = WHOLE ? Span{chunk * kChunk, 0, kChunk} : span_of(chunk, tab.row_len);
    const bool on = WHOLE ? sp.at < tab.row_len : sp.lo < sp.hi;
    float* const first = a.first + uint64_t(tile) * a.pitch + chunk * kChunk;
    float* const last = a.last + uint64_t(tile) * a.pitch + chunk * kChunk;
    const uint32_t rows = uint32_t(tab.rows), k0 = tile * a.k, k1 = min(a.n, k0 + a.k);
    // record k0 + j, j <= 2K <= 64: where the group is a wave, its lanes hold the tile's records and the
    // next one's, read at once
    uint2 held = {kNoRow, 0};
    uint32_t behind = kNoRow;
    if constexpr (LPR == 64) {
        if (k0 + (threadIdx.x & 63) < a.n) held = a.rec[k0 + (threadIdx.x & 63)];
        if (k0 + 64 < a.n) behind = a.rec[k0 + 64].x;
    }
    auto row_at = [&](uint32_t j) -> uint32_t {
        if constexpr (LPR == 64) return j < 64 ? uint32_t(__builtin_amdgcn_readlane(int(held.x), int(j))) : behind;
        else return k0 + j < a.n ? a.rec[k0 + j].x : kNoRow;
    };
    auto record_at = [&](uint32_t j) -> uint32_t {
        if constexpr (LPR == 64) return uint32_t(__builtin_amdgcn_readlane(int(held.y), int(j)));
        else return k0 + j < a.n ? a.rec[k0 + j].y : 0;
    };
    const uint32_t before = k0 > 0 ? a.rec[k0 - 1].x : kNoRow, long_before = k0 > a.k ? a.rec[k0 - a.k - 1].x : kNoRow;
    const uint32_t lead = row_at(0), last_row = row_at(k1 - k0 - 1), next = row_at(k1 - k0), next2 = row_at(2 * a.k);
    bool began = before == lead;                                   // the run at hand began before this tile
    uint32_t skip = kNoRow, tail = kNoRow, jend = k1 - k0;
    // the first run is the tile before's, which goes on into this one to its end
    if (began && next != lead && long_before != lead) {
        skip = lead;
        began = false;
    }
    // the last run begins here and ends in the next tile: followed to its end
    if (last_row == next && before != next && next2 != next) {
        tail = next;
        jend = min(a.n, k1 + a.k) - k0;
    }
    float acc[kChunk] = {};
    bool open = false;                                             // the last record's run goes on
    for (uint32_t j = 0; j < jend; j += U) {                       // (K is a multiple of U)
        uint2 e[U + 1];
#pragma unroll
        for (int u = 0; u < U; u++) e[u] = {row_at(j + u), record_at(j + u)};
        e[U].x = row_at(j + U);
        if (j >= a.k && e[0].x != tail) break;
        Chunk<V> c[U];
        Chunk<T> old[U];
        bool ends[U], part[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            // (a record past the batch: the caller changed the indices while they were sorted)
            const bool mine = j < a.k ? e[u].x != skip : e[u].x == tail;
            const bool live = mine && e[u].x < rows && e[u].y < a.n;
            c[u] = fetch<kLong>(vals + uint64_t(e[u].y) * b.stride, sp.at, tab.row_len, on && live);
            ends[u] = live && e[u].x != e[u + 1].x;
            part[u] = began;
            if (ends[u]) began = false;
            old[u] = fetch<kLong>(reinterpret_cast<const T*>(tab.data) + uint64_t(e[u].x) * tab.row_len, sp.at, tab.row_len,
                                  on && ends[u] && !part[u]);
            if (live) open = !ends[u];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float v[kChunk];
            unpack(c[u], v);
#pragma unroll
            for (int i = 0; i < kChunk; i++) acc[i] += v[i];
            if (!ends[u]) continue;
            if (on) {
                if (part[u]) store_chunk(first, pack<float>(acc));
                else add_to_row<WHOLE>(reinterpret_cast<T*>(tab.data) + uint64_t(e[u].x) * tab.row_len, sp, old[u], acc, b.scale);
            }
#pragma unroll
            for (int i = 0; i < kChunk; i++) acc[i] = 0.f;
        }
    }
    if (open && !began && chunk == 0) a.joins[1 + atomicAdd(a.joins, 1u)] = tile;
    if (open && on) store_chunk(began ? first : last, pack<float>(acc));
}

// Rows that reach past the tile after the one in which they begin: a wave takes such a row and the columns
// that `lanes` lanes hold, its lane groups a share of the parts each. Where there are many parts (one row
// may have every record) the block does it together. Few lanes, so that the parts of one row are read by
// as many compute units as its columns allow (8192 records of 512 columns, all of one row: 64, 45, 35 us
// with 64, 32, 16 lanes; 131072 of 4096 as tokens come: 502, 502, 506). A long run of few columns is left to
// few of them all the same: 131072 records of 64 columns, all of one row, take 80 us in all, 42 of even rows;
// 2^20 of 128 255 and 138. The list's order is no one's:
// every row is in it once, and its parts are added in an order that their number fixes.
constexpr uint32_t kWaveParts = 64;
constexpr uint32_t kJoinWaves = 8;

__device__ __forceinline__ void add_parts(const SumArgs& a, uint32_t tile, uint32_t j0, uint32_t j1, uint32_t chunk, float (&acc)[kChunk]) {
    constexpr int U = 8;
    for (uint32_t j = j0; j < j1; j += U) {                        // (U parts in flight, the last one again)
        Chunk<float> c[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t i = min(j + u, j1 - 1);
            c[u] = load_chunk((i == 0 ? a.last + uint64_t(tile) * a.pitch : a.first + uint64_t(tile + i) * a.pitch) + chunk * kChunk);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (j + u >= j1) continue;
            float v[kChunk];
            unpack(c[u], v);
#pragma unroll
            for (int i = 0; i < kChunk; i++) acc[i] += v[i];
        }
    }
}

template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void k_rows_join(RowTable tab, float scale, SumArgs a, Divisor wide) {
    __shared__ float sum[kJoinWaves][64][kChunk + 1];
    __shared__ uint32_t many[kJoinWaves];
    const uint32_t lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), items = *a.joins * wide.d, gap = gridDim.x;
    const uint32_t per = 64 / a.lanes, group = lane / a.lanes;     // shares of a wave, this lane's
    for (uint32_t base = blockIdx.x; base < items; base += gap * kJoinWaves) {
        const uint32_t item = base + gap * w;                      // neighbours go to different blocks
        uint32_t parts = 0;
        if (item < items) {
            const uint32_t which = uint32_t(quotient64(item, wide)), tile = a.joins[1 + which];
            const uint32_t row = a.rec[uint64_t(tile + 1) * a.k].x;
            // the last tile that begins inside the run: tiles [lo, ..] begin with `row`, narrowed 64 ways a step
            uint32_t lo = tile + 1, hi = a.tiles;
            while (hi - lo > 1) {
                const uint32_t step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step;
                const uint64_t in = __ballot(at < hi && a.rec[uint64_t(at) * a.k].x == row);
                const uint32_t next = lo + __popcll(in) * step;    // (sorted: the true lanes come first)
                hi = min(hi, next + step);
                lo = next;
            }
            parts = row < uint32_t(tab.rows) ? lo - tile + 1 : 0;  // (see k_rows_sum: changed indices)
            const uint32_t chunk = (item - which * wide.d) * a.lanes + lane % a.lanes;
            const Span sp = span_of(chunk, tab.row_len);
            if (parts > 0 && parts <= kWaveParts) {
                T* p = reinterpret_cast<T*>(tab.data) + uint64_t(row) * tab.row_len;
                const bool on = sp.lo < sp.hi;
                const Chunk<T> old = fetch(p, sp.at, tab.row_len, on && group == 0);
                const uint32_t share = (parts + per - 1) / per;
                float acc[kChunk] = {};
                if (on) add_parts(a, tile, min(parts, group * share), min(parts, (group + 1) * share), chunk, acc);
                for (uint32_t o = 1; o < per; o++)
#pragma unroll
                    for (int i = 0; i < kChunk; i++) {
                        const float v = __shfl(acc[i], int(o * a.lanes + lane % a.lanes), 64);
                        if (group == 0) acc[i] += v;
                    }
                if (on && group == 0) add_to_row(p, sp, old, acc, scale);
            }
        }
        if (lane == 0) many[w] = parts > kWaveParts ? parts : 0;
        __syncthreads();
        for (uint32_t i = 0; i < kJoinWaves; i++) {
            const uint32_t n = many[i];                            // (alike in the whole block)
            if (n == 0) continue;
            const uint32_t which = uint32_t(quotient64(base + gap * i, wide)), tile = a.joins[1 + which];
            const uint32_t mine = w * per + group, share = (n + kJoinWaves * per - 1) / (kJoinWaves * per);
            const uint32_t chunk = (base + gap * i - which * wide.d) * a.lanes + lane % a.lanes;
            const Span sp = span_of(chunk, tab.row_len);
            const bool on = sp.lo < sp.hi;
            float acc[kChunk] = {};
            if (on) add_parts(a, tile, min(n, mine * share), min(n, (mine + 1) * share), chunk, acc);
#pragma unroll
            for (int k = 0; k < kChunk; k++) sum[w][lane][k] = acc[k];
            __syncthreads();
            if (w == 0 && group == 0 && on) {
                for (uint32_t o = 1; o < kJoinWaves * per; o++)
#pragma unroll
                    for (int k = 0; k < kChunk; k++) acc[k] += sum[o / per][o % per * a.lanes + lane][k];
                T* p = reinterpret_cast<T*>(tab.data) + uint64_t(a.rec[uint64_t(tile + 1) * a.k].x) * tab.row_len;
                add_to_row(p, sp, fetch(p, sp.at, tab.row_len, true), acc, scale);
            }
            __syncthreads();
        }
        __syncthreads();                                           // (every wave has read `many`)
    }
}

// ---------------------------------------------------------------- store
// Of several records of one row the last is stored. Few records: each looks for its row in the rest of
// the list (64 rows of 1024 codes: 2.9 us against 4.7 with claims, 1024: 4.3 against 5.8, 2048: 6.6
// against 6.3). Many: a first launch raises the row's claim to the record's number + 1; the record that
// finds its own number there stores, and clears the claim.
enum { kDistinct, kScanned, kClaimed };

template <int IW>
__global__ __launch_bounds__(256) void k_rows_claim(RowTable tab, RowBatch b, uint32_t* err) {
    const uint64_t t = uint64_t(blockIdx.x) * 256 + threadIdx.x;
    if (t >= b.n) return;
    const int64_t r = row_of<IW>(b, t, tab.rows, err, true);
    if (r >= 0) atomicMax(&tab.claims[r], uint32_t(t) + 1);
}

// a code word of four elements
template <typename T>
__device__ __forceinline__ uint32_t to_codes(const float* x, const GroupScale& q) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = q.inv == 0.f ? 0.f : x[i] * q.inv;  // |y| <= Q (1 + 2^-22): rounds to a code
    if constexpr (std::is_same_v<T, code_i8>) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) w |= (uint32_t(__float2int_rn(y[i])) & 0xffu) << (8 * i);
        return w;
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true));
    }
}
__device__ __forceinline__ uint32_t max_bits(const float (&v)[kChunk]) {
    uint32_t m = 0;                                                // largest |x| as bits: infinities and NaN on top
#pragma unroll
    for (int i = 0; i < kChunk; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}
__device__ __forceinline__ uint32_t max_over(uint32_t m, uint32_t lanes) {
    for (uint32_t d = lanes / 2; d; d /= 2) m = max(m, uint32_t(__shfl_xor(int(m), int(d), 64)));
    return m;
}
template <typename T>
__device__ __forceinline__ Chunk<T> pack_codes(const float (&v)[kChunk], const GroupScale& q) {
    return {{to_codes<T>(v, q), to_codes<T>(v + 4, q)}};
}

// L lanes per record: 8 to 64 (as many as hold a short row, so that a wave takes several), or the whole
// block. Groups of up to 512 elements: as many lanes as hold one (a power of two) find its largest |x|
// by shuffles and keep its values in registers. Longer groups are read twice, the second time from cache.
// 16384 bf16 rows of 2048 to i8: 24 us, 4.2 TB/s; 65536 rows of 64 to e4m3 10 us (26 with a wave for each). With
// the claims' launch, 65536 bf16 rows: of 1024 in groups of 128 to e4m3 41 us, 5.0 TB/s; of 1000 in groups of 100
// 48 us, 4.1; of 1152 in groups of 576 62 us, 3.7 (to i8 67, 3.4); of 4096 to bf16 217 us, 5.0 TB/s, of 64 11 us.
template <typename T, typename V, int IW, int L>
__global__ __launch_bounds__(256) void k_rows_store(RowTable tab, RowBatch b, const V* vals, uint32_t* err, int how, uint32_t lpg) {
    constexpr int kWaves = L > 64 ? L / 64 : 1;                    // waves that share a record
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6, mine_of = threadIdx.x % L;
    uint32_t t = blockIdx.x * (256 / L) + threadIdx.x / L;
    if constexpr (L >= 64) t = __builtin_amdgcn_readfirstlane(t);
    if (t >= b.n) return;
    const int64_t r = row_of<IW>(b, t, tab.rows, err, mine_of == 0);
    bool mine = r >= 0;
    if (how == kScanned) {
        bool later = false;
        for (uint32_t u = t + 1 + (L > 64 ? lane : mine_of); u < b.n; u += L > 64 ? 64 : L) later |= row_index<IW>(b, u) == r;
        const uint64_t found = __ballot(later);
        mine = mine && !(L >= 64 ? found : found >> (lane & ~uint32_t(L - 1)) & ((1ull << (L & 63)) - 1));
    } else if (how == kClaimed) {
        mine = mine && tab.claims[r] == t + 1;
        if constexpr (kWaves > 1) __syncthreads();                 // every wave has read the claim
        if (mine && mine_of == 0) tab.claims[r] = 0;
    }
    if (!mine) return;
    T* row = reinterpret_cast<T*>(tab.data) + uint64_t(r) * tab.row_len;
    const V* x = vals + uint64_t(t) * b.stride;
    if constexpr (!is_code<T>::v) {
        constexpr int U = 4;                                       // chunks in flight
        const uint32_t chunks = (tab.row_len + kChunk - 1) / kChunk;
        for (uint32_t c = mine_of; c < chunks; c += U * L) {
            Chunk<V> v[U];
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = fetch(x, span_of(c + u * L, tab.row_len).at, tab.row_len, c + u * L < chunks);
#pragma unroll
            for (int u = 0; u < U; u++) {
                float f[kChunk];
                unpack(v[u], f);
                if (c + u * L < chunks) put(row, span_of(c + u * L, tab.row_len).at, tab.row_len, pack<T>(f));
            }
        }
    } else if (lpg) {
        const uint32_t in = mine_of & (lpg - 1), at = span_of(in, tab.group).at;
        for (uint32_t g0 = 0; g0 < tab.groups; g0 += L / lpg) {
            const uint32_t g = g0 + mine_of / lpg;
            const bool on = g < tab.groups && in * kChunk < tab.group;
            float v[kChunk];
            unpack(fetch(x + g * tab.group, at, tab.group, on), v);
            const GroupScale q = group_scale<T>(max_over(max_bits(v), lpg));
            if (!on) continue;
            put(row + g * tab.group, at, tab.group, pack_codes<T>(v, q));
            if (in == 0) tab.scales[uint64_t(r) * tab.groups + g] = q.scale;
        }
    } else if constexpr (L >= 64) {
        __shared__ uint32_t top[2][4];
        for (uint32_t g = 0; g < tab.groups; g++) {
            const V* xg = x + uint64_t(g) * tab.group;
            T* rg = row + uint64_t(g) * tab.group;
            uint32_t m = 0;
            constexpr int U = 4;                                   // chunks in flight
            const uint32_t chunks = (tab.group + kChunk - 1) / kChunk;
            for (uint32_t c = mine_of; c < chunks; c += U * L) {
                Chunk<V> v[U];
#pragma unroll
                for (int u = 0; u < U; u++) v[u] = fetch(xg, span_of(c + u * L, tab.group).at, tab.group, c + u * L < chunks);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float f[kChunk];
                    unpack(v[u], f);
                    m = max(m, max_bits(f));
                }
            }
            m = max_over(m, 64);
            if constexpr (kWaves > 1) {                            // (two sets: a wave may be one group ahead)
                if (lane == 0) top[g & 1][w] = m;
                __syncthreads();
                m = max(max(top[g & 1][0], top[g & 1][1]), max(top[g & 1][2], top[g & 1][3]));
            }
            const GroupScale q = group_scale<T>(m);
            for (uint32_t c = mine_of; c < chunks; c += U * L) {
                Chunk<V> v[U];
#pragma unroll
                for (int u = 0; u < U; u++) v[u] = fetch(xg, span_of(c + u * L, tab.group).at, tab.group, c + u * L < chunks);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float f[kChunk];
                    unpack(v[u], f);
                    if (c + u * L < chunks) put(rg, span_of(c + u * L, tab.group).at, tab.group, pack_codes<T>(f, q));
                }
            }
            if (mine_of == 0) tab.scales[uint64_t(r) * tab.groups + g] = q.scale;
        }
    }
}

// A launch and its own status: what hipGetLastError holds may be an earlier call's, for whoever asks there.
template <typename... P, typename... A>
hipError_t launch(void (*kernel)(P...), dim3 grid, unsigned threads, hipStream_t s, const A&... given) {
    std::tuple<P...> args(static_cast<P>(given)...);
    return std::apply([&](auto&... a) {
        void* at[] = {&a...};
        return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), at, 0, s);
    }, args);
}

bool is_float_type(uint32_t type) { return type <= LMR_ROW_BF16; }
template <typename F>
hipError_t by_value_type(uint32_t type, F&& f) {
    switch (type) {
    case LMR_ROW_F32: return f(float{});
    case LMR_ROW_F16: return f(_Float16{});
    default: return f(__bf16{});
    }
}
template <typename F>
hipError_t by_row_type(uint32_t type, F&& f) {
    switch (type) {
    case LMR_ROW_I8: return f(code_i8{});
    case LMR_ROW_E4M3: return f(code_e4m3{});
    default: return by_value_type(type, f);
    }
}
template <typename F>
hipError_t by_index(uint32_t size, F&& f) {
    return size == 4 ? f(std::integral_constant<int, 4>{}) : f(std::integral_constant<int, 8>{});
}

hipError_t launch_load(const RowTable& tab, const RowBatch& b, void* out, uint32_t out_type, uint32_t* err, hipStream_t s) {
    const Divisor cpr = divisor((tab.row_len + kChunk - 1) / kChunk);
    const bool ga = tab.group % kChunk == 0;             // (other types: the whole row is the group, and unused)
    const Divisor cpg = divisor(ga ? tab.group / kChunk : 1);
    return by_row_type(tab.type, [&](auto t) { return by_value_type(out_type, [&](auto o) { return by_index(b.index_size, [&](auto iw) {
        using T = decltype(t);
        using O = decltype(o);
        constexpr int IW = decltype(iw)::value;
        O* p = reinterpret_cast<O*>(out);
        const uint64_t chunks = b.n * cpr.d;
        // four chunks a thread keep four reads in flight; a batch that would leave compute units
        // without a block gives each thread one
        const bool four = chunks >= 2048ull * 256;
        const dim3 grid(unsigned(four ? (chunks + 1023) / 1024 : (chunks + 255) / 256));
        if constexpr (is_code<T>::v) {
            if (!ga) return launch(four ? k_rows_load<T, O, IW, 4, false> : k_rows_load<T, O, IW, 1, false>, grid, 256, s, tab, b, p, err, cpr, cpg);
        }
        return launch(four ? k_rows_load<T, O, IW, 4, true> : k_rows_load<T, O, IW, 1, true>, grid, 256, s, tab, b, p, err, cpr, cpg);
    }); }); });
}
enum RowSort { kRanked, kMerged, kDigits };
// How a batch of adds runs, and its workspace: two lists of (row, record), the digit counts, and the
// parts of rows that reach past a group's records.
struct AddPlan {
    uint32_t few;                            // k_rows_add_few for at most so many records, 0: sorted
    RowSort sort;
    uint32_t bits, passes, ipt, tiles;       // sort: bits of a digit, passes, records a thread takes, tiles
    uint32_t lanes, chunks, k, groups;       // sum: lanes of a group, its column chunks, records, groups
    uint32_t pitch;
    uint64_t rec[2], hist, joins, first, last, bytes;
};
AddPlan add_plan(uint64_t rows, uint32_t row_len, uint64_t n) {
    AddPlan p = {};
    const uint64_t blocks = n * ((row_len + 511) / 512);
    p.few = n <= 512 && blocks <= 4096 ? 512 : n <= 1024 && blocks <= 2048 ? 1024 : 0;
    if (p.few) return p;
    const uint32_t key_bits = 32 - __builtin_clz(uint32_t(rows) | 1);     // keys 0 .. rows
    p.sort = n <= kRankMost ? kRanked : n <= kMergeMost ? kMerged : kDigits;
    p.passes = (key_bits + kSortBits - 1) / kSortBits;
    p.bits = (key_bits + p.passes - 1) / p.passes;
    // (tiles of 1024, 2048 and 4096 records: see above kSortThreads)
    p.ipt = n <= (1 << 18) ? 2 : n <= (1 << 20) ? 4 : 8;
    p.tiles = uint32_t((n + p.ipt * kSortThreads - 1) / (p.ipt * kSortThreads));
    const uint32_t cols = (row_len + kChunk - 1) / kChunk;
    p.lanes = cols > 32 ? 64 : cols > 16 ? 32 : cols > 8 ? 16 : 8;
    p.chunks = (cols + p.lanes - 1) / p.lanes;
    // 32 records a group, fewer where that would leave less than about 8 waves per compute unit (131072
    // records of 4096, all launches: 647, 557, 516, 504 us with 4, 8, 16, 32; 5003 of 1001: 28.9, 32.0, 38.9
    // with 4, 8, 16)
    const uint64_t waves = n * p.chunks * p.lanes / 64;
    p.k = waves >= 32 * 2048 ? 32 : waves >= 16 * 2048 ? 16 : waves >= 8 * 2048 ? 8 : 4;
    p.groups = uint32_t((n + p.k - 1) / p.k);
    p.pitch = cols * kChunk;
    uint64_t at = 0;
    auto take = [&at](uint64_t bytes) { const uint64_t o = at; at += (bytes + 255) & ~uint64_t(255); return o; };
    p.rec[0] = take(n * sizeof(uint2));
    p.rec[1] = take(p.sort == kMerged || (p.sort == kDigits && p.passes > 1) ? n * sizeof(uint2) : 0);
    p.hist = take(p.sort != kDigits ? 0 : (uint64_t(p.tiles) + 1) << p.bits << 2);
    p.joins = take((uint64_t(p.groups) + 1) * 4);
    p.first = take(uint64_t(p.groups) * p.pitch * 4);
    p.last = take(uint64_t(p.groups) * p.pitch * 4);
    p.bytes = at;
    return p;
}

template <int IW>
hipError_t sort_records(const AddPlan& p, const RowTable& tab, const RowBatch& b, uint8_t* work, uint32_t* err, hipStream_t s,
                        const uint2** sorted) {
    const uint2* in = nullptr;
    const uint32_t n = uint32_t(b.n);
    uint32_t* const joins = reinterpret_cast<uint32_t*>(work + p.joins);
    if (p.sort != kDigits) {
        uint2* const a = reinterpret_cast<uint2*>(work + p.rec[0]);
        *sorted = a;
        if (p.sort == kRanked) {
            const uint32_t part = std::max<uint32_t>(16, (n + 511) / 512 * 2);         // 256 blocks
            return launch(k_rows_rank<IW, kRankMost>, dim3((n + part - 1) / part), 1024, s,
                          SortPass{nullptr, a, nullptr, n, 0, 0, 1, false, joins}, part, b, tab, err);
        }
        uint2* const t = reinterpret_cast<uint2*>(work + p.rec[1]);
        const uint32_t part = (n + 255) / 256;
        const hipError_t e = launch(k_rows_rank<IW, kMergeTile>, dim3((n + 63) / 64), 1024, s,
                                    SortPass{nullptr, t, nullptr, n, 0, 0, 1, false, joins}, 64u, b, tab, err);
        if (e != hipSuccess) return e;
        return launch(k_rows_merge, dim3((n + part - 1) / part), 1024, s, SortPass{t, a, nullptr, n, 0, 0, 1, false, joins}, part);
    }
    for (uint32_t i = 0; i < p.passes; i++) {
        uint2* out = reinterpret_cast<uint2*>(work + p.rec[i & 1]);
        SortPass q = {in, out, reinterpret_cast<uint32_t*>(work + p.hist), uint32_t(b.n), i * p.bits, p.bits, p.tiles, p.tiles > 64,
                      reinterpret_cast<uint32_t*>(work + p.joins)};
        auto go = [&](auto ipt) {
            constexpr int IPT = decltype(ipt)::value;
            hipError_t e = launch(k_rows_count<IW, IPT>, dim3(p.tiles), kSortThreads, s, q, b, tab, err);
            if (e == hipSuccess && q.summed) e = launch(k_rows_prefix, dim3(((1u << p.bits) + 63) / 64), 1024, s, q);
            return e != hipSuccess ? e : launch(k_rows_place<IW, IPT>, dim3(p.tiles), kSortThreads, s, q, b, tab, err);
        };
        const hipError_t e = p.ipt == 2 ? go(std::integral_constant<int, 2>{}) : p.ipt == 4 ? go(std::integral_constant<int, 4>{})
                                        : go(std::integral_constant<int, 8>{});
        if (e != hipSuccess) return e;
        in = out;
    }
    *sorted = in;
    return hipSuccess;
}

hipError_t launch_add(const RowTable& tab, const RowBatch& b, const void* vals, uint32_t val_type, void* work, uint32_t* err,
                      hipStream_t s) {
    const AddPlan p = add_plan(tab.rows, tab.row_len, b.n);
    if (p.few)
        return by_value_type(tab.type, [&](auto t) { return by_value_type(val_type, [&](auto v) { return by_index(b.index_size, [&](auto iw) {
            using V = decltype(v);
            const dim3 grid(unsigned(b.n), (tab.row_len + 511) / 512);
            const V* x = reinterpret_cast<const V*>(vals);
            return launch(p.few == 512 ? k_rows_add_few<decltype(t), V, decltype(iw)::value, 512>
                                       : k_rows_add_few<decltype(t), V, decltype(iw)::value, 1024>, grid, 256, s, tab, b, x, err);
        }); }); });
    uint8_t* w = reinterpret_cast<uint8_t*>(work);
    const uint2* sorted = nullptr;
    hipError_t e = by_index(b.index_size, [&](auto iw) { return sort_records<decltype(iw)::value>(p, tab, b, w, err, s, &sorted); });
    if (e != hipSuccess) return e;
    const SumArgs a = {sorted, reinterpret_cast<float*>(w + p.first), reinterpret_cast<float*>(w + p.last), reinterpret_cast<uint32_t*>(w + p.joins),
                       uint32_t(b.n), p.k, p.groups, p.pitch, std::min(p.lanes, tab.row_len > 1024 ? 32u : 16u), divisor(p.chunks)};
    const Divisor wide = divisor((tab.row_len + a.lanes * kChunk - 1) / (a.lanes * kChunk));
    const unsigned join_blocks = unsigned(std::min<uint64_t>(uint64_t(p.groups) * wide.d, 512));
    const unsigned blocks = unsigned((uint64_t(p.groups) * p.chunks * p.lanes + 255) / 256);
    return by_value_type(tab.type, [&](auto t) { return by_value_type(val_type, [&](auto v) {
        using T = decltype(t);
        using V = decltype(v);
        const V* x = reinterpret_cast<const V*>(vals);
        auto sum = [&](auto lanes, auto whole, auto u) {
            return launch(k_rows_sum<T, V, decltype(lanes)::value, decltype(whole)::value, decltype(u)::value>, dim3(blocks), 256, s, tab, b, x, a);
        };
        auto by_lanes = [&](auto whole, auto u) {
            switch (p.lanes) {
            case 8: return sum(std::integral_constant<int, 8>{}, whole, u);
            case 16: return sum(std::integral_constant<int, 16>{}, whole, u);
            case 32: return sum(std::integral_constant<int, 32>{}, whole, u);
            default: return sum(std::integral_constant<int, 64>{}, whole, u);
            }
        };
        // (131072 bf16 records of 4096: 514 us with 4 in flight, 504 with 8; ends of rows that are not whole cost
        // registers: 5003 of 1001 took 1.5 us longer with 8)
        const hipError_t e = tab.row_len % kChunk ? by_lanes(std::false_type{}, std::integral_constant<int, 4>{})
                             : p.k == 4           ? by_lanes(std::true_type{}, std::integral_constant<int, 4>{})
                                                  : by_lanes(std::true_type{}, std::integral_constant<int, 8>{});
        return e != hipSuccess ? e : launch(k_rows_join<T>, dim3(join_blocks), 64 * kJoinWaves, s, tab, b.scale, a, wide);
    }); });
}
hipError_t launch_store(const RowTable& tab, const RowBatch& b, const void* vals, uint32_t val_type, uint32_t* err, hipStream_t s) {
    const int how = b.n == 1 ? kDistinct : b.n <= LMR_ROW_SCAN ? kScanned : tab.claims ? kClaimed : kDistinct;
    uint32_t lpg = 0;                                              // lanes that hold a group, 0: longer groups
    if (tab.group <= 64 * kChunk)
        for (lpg = 1; lpg * kChunk < tab.group;) lpg *= 2;
    // a block shares a record where records alone do not fill the card and a row has work for it (64
    // rows of 4096: 3.5 us against 7.0 with a wave; 2048 rows of 1024: 6.6 against 6.3)
    const uint32_t need = lpg ? std::min(64u, lpg * tab.groups) : 64u, held = is_float_type(tab.type) ? (tab.row_len + 7) / 8 : need;
    const uint32_t lanes = b.n < 2048 && tab.row_len > 512 ? 256 : held > 32 ? 64 : held > 16 ? 32 : held > 8 ? 16 : 8;
    return by_row_type(tab.type, [&](auto t) { return by_value_type(val_type, [&](auto v) { return by_index(b.index_size, [&](auto iw) {
        using T = decltype(t);
        using V = decltype(v);
        constexpr int IW = decltype(iw)::value;
        const V* x = reinterpret_cast<const V*>(vals);
        if (how == kClaimed) {
            const hipError_t e = launch(k_rows_claim<IW>, dim3(unsigned((b.n + 255) / 256)), 256, s, tab, b, err);
            if (e != hipSuccess) return e;
        }
        auto go = [&](auto l) {
            constexpr int L = decltype(l)::value;
            return launch(k_rows_store<T, V, IW, L>, dim3(unsigned((b.n + 256 / L - 1) / (256 / L))), 256, s, tab, b, x, err, how, lpg);
        };
        switch (lanes) {
        case 8: return go(std::integral_constant<int, 8>{});
        case 16: return go(std::integral_constant<int, 16>{});
        case 32: return go(std::integral_constant<int, 32>{});
        case 64: return go(std::integral_constant<int, 64>{});
        default: return go(std::integral_constant<int, 256>{});
        }
    }); }); });
}

uint32_t type_bytes(uint32_t type) {
    switch (type) {
    case LMR_ROW_F32: return 4;
    case LMR_ROW_F16: case LMR_ROW_BF16: return 2;
    default: return 1;
    }
}
bool aligned(const void* p, uint32_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

lmr_status_t check_table(const lmr_rows_t* t) {
    if (!t || t->type >= LMR_NUM_ROW_TYPES) return LMR_E_INVALID;
    if (t->row_len == 0 || t->row_len > LMR_ROW_MAX_LEN || t->rows > LMR_ROWS_MAX) return LMR_E_INVALID;
    if (t->rows && (!t->data || !aligned(t->data, type_bytes(t->type)))) return LMR_E_INVALID;
    if (t->claims && !aligned(t->claims, 4)) return LMR_E_INVALID;
    if (t->type == LMR_ROW_I8 || t->type == LMR_ROW_E4M3) {
        if (t->group == 0 || t->row_len % t->group != 0) return LMR_E_INVALID;
        if (t->rows && (!t->scales || !aligned(t->scales, 4))) return LMR_E_INVALID;
    }
    return LMR_OK;
}

// the records and the n x row_len values beside them (load: the output; stride 0: one row for every record)
lmr_status_t check_batch(const lmr_ctx* ctx, const lmr_rows_t* t, const void* idx, uint32_t index_size, uint64_t n,
                         const void* vals, uint32_t val_type, uint64_t stride, bool may_repeat) {
    if (!ctx) return LMR_E_INVALID;
    const lmr_status_t st = check_table(t);
    if (st != LMR_OK) return st;
    if ((index_size != 4 && index_size != 8) || val_type > LMR_ROW_BF16 || n > LMR_ROW_MAX_BATCH) return LMR_E_INVALID;
    if (n * t->row_len > LMR_ROW_MAX_VALUES) return LMR_E_INVALID;
    if (n > 0 && (!idx || !vals || !aligned(idx, index_size) || !aligned(vals, type_bytes(val_type)))) return LMR_E_INVALID;
    if (n > 1 && stride < t->row_len && !(may_repeat && stride == 0)) return LMR_E_INVALID;
    if (stride > LMR_ROW_MAX_STRIDE) return LMR_E_INVALID;
    return LMR_OK;
}

RowTable table_of(const lmr_rows_t* t) {
    RowTable r;
    r.data = t->data;
    r.scales = t->scales;
    r.claims = t->claims;
    r.rows = t->rows;
    r.row_len = uint32_t(t->row_len);
    r.type = t->type;
    const bool code = t->type == LMR_ROW_I8 || t->type == LMR_ROW_E4M3;
    r.group = code ? t->group : uint32_t(t->row_len);
    r.groups = uint32_t(t->row_len) / r.group;
    return r;
}
RowBatch batch_of(const void* idx, uint32_t index_size, uint64_t n, int has_pad, int64_t pad, float scale, uint64_t stride) {
    RowBatch b;
    b.idx = idx;
    b.index_size = index_size;
    b.has_pad = has_pad != 0;
    b.pad = pad;
    b.n = n;
    b.scale = scale;
    b.stride = stride;
    return b;
}

// the context's device for the launches of one call, the caller's afterwards
struct OnDevice {
    int was = 0;
    bool ok, moved = false;
    explicit OnDevice(int device) {
        ok = hipGetDevice(&was) == hipSuccess;
        if (ok && was != device) ok = moved = hipSetDevice(device) == hipSuccess;
        if (!ok) (void)hipGetLastError();
    }
    ~OnDevice() { if (moved) (void)hipSetDevice(was); }
};
// (a failure is told by the status and not left in the runtime; an earlier call's error stays)
lmr_status_t hip_status(hipError_t e) {
    if (e != hipSuccess) (void)hipGetLastError();
    return e == hipSuccess ? LMR_OK : LMR_E_HIP;
}

}  // namespace
}  // namespace lmr

using namespace lmr;

extern "C" {

lmr_status_t lmr_rows_load(lmr_ctx_t* ctx, const lmr_rows_t* table, const void* d_idx, uint32_t index_size, uint64_t n,
                           int has_pad, int64_t pad, float scale, void* d_out, uint32_t out_type, uint64_t out_stride,
                           lmr_stream_t stream) {
    const lmr_status_t st = check_batch(ctx, table, d_idx, index_size, n, d_out, out_type, out_stride, false);
    if (st != LMR_OK || n == 0) return st;
    OnDevice dev(ctx->device);
    if (!dev.ok) return LMR_E_HIP;
    return hip_status(launch_load(table_of(table), batch_of(d_idx, index_size, n, has_pad, pad, scale, out_stride), d_out,
                                  out_type, ctx->d_err, reinterpret_cast<hipStream_t>(stream)));
}

uint64_t lmr_rows_add_workspace(const lmr_rows_t* table, uint64_t n) {
    if (check_table(table) != LMR_OK || n > LMR_ROW_MAX_BATCH) return 0;
    return add_plan(table->rows, uint32_t(table->row_len), n).bytes;
}

lmr_status_t lmr_rows_add(lmr_ctx_t* ctx, const lmr_rows_t* table, const void* d_idx, uint32_t index_size, uint64_t n,
                          int has_pad, int64_t pad, float scale, const void* d_vals, uint32_t val_type, uint64_t val_stride,
                          void* d_work, uint64_t work_bytes, lmr_stream_t stream) {
    const lmr_status_t st = check_batch(ctx, table, d_idx, index_size, n, d_vals, val_type, val_stride, true);
    if (st != LMR_OK) return st;
    if (table->type > LMR_ROW_BF16) return LMR_E_UNSUPPORTED;
    if (n == 0) return LMR_OK;
    if (work_bytes < lmr_rows_add_workspace(table, n) || (work_bytes && (!d_work || !aligned(d_work, 16))))
        return LMR_E_WORKSPACE;
    OnDevice dev(ctx->device);
    if (!dev.ok) return LMR_E_HIP;
    return hip_status(launch_add(table_of(table), batch_of(d_idx, index_size, n, has_pad, pad, scale, val_stride), d_vals,
                                 val_type, d_work, ctx->d_err, reinterpret_cast<hipStream_t>(stream)));
}

lmr_status_t lmr_rows_store(lmr_ctx_t* ctx, const lmr_rows_t* table, const void* d_idx, uint32_t index_size, uint64_t n,
                            int has_pad, int64_t pad, const void* d_vals, uint32_t val_type, uint64_t val_stride,
                            lmr_stream_t stream) {
    const lmr_status_t st = check_batch(ctx, table, d_idx, index_size, n, d_vals, val_type, val_stride, true);
    if (st != LMR_OK || n == 0) return st;
    OnDevice dev(ctx->device);
    if (!dev.ok) return LMR_E_HIP;
    return hip_status(launch_store(table_of(table), batch_of(d_idx, index_size, n, has_pad, pad, 1.f, val_stride), d_vals,
                                   val_type, ctx->d_err, reinterpret_cast<hipStream_t>(stream)));
}

}  // extern "C"
