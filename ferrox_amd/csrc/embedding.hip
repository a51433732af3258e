// Embedding lookup with scaling and its dense weight gradient:
//   out[n] = scale * W[id_n];   dW[v] = scale * sum over n with id_n = v of g[n]  (every row of dW is written)
// An id outside 0 .. V - 1 (padding) gives a row of zeros and no gradient.
//
// The lookup is a gather of rows, bound by memory.  The gradient sorts the (id, n) pairs by id, stably, and then adds the rows of g
// along the sorted order: every token's row is read once, no atomics, and the order of every sum depends on the ids alone.
//   sort     up to 32768 tokens: one launch in which every block owns 256 consecutive ids, reads all tokens, keeps those of its ids
//            in LDS and places them by one stable counting pass; how many tokens lie below its ids is counted on the way and is where
//            its part of the order begins.  More tokens (or so many ids that the blocks would read too much): radix passes of 8 bits
//            over tiles of 4096 tokens (counts per tile, one scan over digits and tiles, stable scatter).
//   add      a piece of P consecutive sorted positions is summed by the threads of one (or a part of one) block, which run along
//            the row; an id whose tokens all lie in one piece is written at once, an id that crosses a piece's border leaves one
//            partial row per piece.  The same launch writes the zero rows of the ids that do not occur.
//   join     an id that crosses borders has its partial rows added in order.
// Frequent ids (a few percent of all tokens for one id are ordinary) are so spread over many blocks.
#include <mutex>

#include "vecio.hpp"

namespace {
using namespace vio;

// ---- lookup --------------------------------------------------------------------------------------------------------------------
// One thread per vector of the output, U of them a block apart; a row has nv vectors, the last of which may be incomplete.  All loads of
// the ids, then all loads of the table are in flight together: a token outside the table reads row 0 and stores zeros.
template <typename T, int V>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const T* __restrict__ W, const int64_t* __restrict__ ids, T* __restrict__ out, i64 total,
                                                            unsigned nv, i64 vocab, int D, T scale) {
    constexpr int U = 4;
    const i64 first = (i64)blockIdx.x * (256 * U);
    const i64 row0 = first / nv;  // block-uniform
    const unsigned off = (unsigned)(first - row0 * nv), last = (unsigned)(min(total - first, (i64)(256 * U)) - 1);
    unsigned dr[U], col[U];
    i64 id[U];
    T v[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned q = off + min(u * 256 + threadIdx.x, last);  // past the end: the last vector again, not stored
        dr[u] = q / nv;
        col[u] = (q - dr[u] * nv) * V;
        id[u] = ids[row0 + dr[u]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (id[u] < 0 || id[u] >= vocab) id[u] = -1;
        load_part<V>(W + (id[u] < 0 ? 0 : id[u]) * D, (int)col[u], D, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (u * 256 + threadIdx.x <= last) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[u][e] = id[u] < 0 ? T(0) : v[u][e] * scale;
            store_part<V>(out + (row0 + dr[u]) * D, (int)col[u], D, v[u]);
        }
    }
}

// ---- stable sort of the ids ------------------------------------------------------------------------------------------------------
constexpr int SORT_NT = 1024, SORT_WAVES = SORT_NT / 64, BITS = 8, BINS = 1 << BITS;
constexpr int RANGE_MAX = 32768, TILE = 4096;  // tokens: positions of the one-launch sort fit 16 bits and its LDS

// padding sorts behind every id
__device__ __forceinline__ uint32_t key_of(int64_t id, i64 vocab) { return id >= 0 && id < vocab ? (uint32_t)id : (uint32_t)vocab; }

// Stable ranks of K items per thread by the digit at `shift`.  Item j of a thread is number (wave * K + j) * 64 + lane of the
// block's items.  rank[j]: how many earlier items of the same wave have the same digit.  counts [wave][bin]: the waves' totals.
// Lanes with the same digit find each other by one ballot per bit.
template <int K>
__device__ __forceinline__ void rank_items(const uint32_t (&key)[K], int shift, uint32_t (&rank)[K], volatile uint32_t* counts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    volatile uint32_t* mine = counts + wave * BINS;
    for (int b = lane; b < BINS; b += 64) mine[b] = 0;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const uint32_t d = (key[j] >> shift) & (BINS - 1);
        uint64_t same = ~0ull;
#pragma unroll
        for (int b = 0; b < BITS; ++b) {
            const uint64_t set = __ballot((d >> b) & 1);
            same &= (d >> b) & 1 ? set : ~set;
        }
        const int before = __popcll(same & ((1ull << lane) - 1));
        const uint32_t sofar = mine[d];  // all lanes read before one lane per digit adds: one wave, LDS operations stay in order
        __builtin_amdgcn_wave_barrier();
        if (before == 0) mine[d] = sofar + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
        rank[j] = sofar + before;
    }
}

// counts [wave][bin] -> where the items of (bin, wave) start among the block's items: an exclusive scan in (bin, wave) order.
// wsum: 4 values.  Barriers on both sides.
__device__ __forceinline__ void scan_counts(uint32_t* counts, uint32_t* wsum) {
    __syncthreads();
    const int t = threadIdx.x, lane = t & 63;
    uint32_t sum = 0, incl = 0, before[SORT_WAVES];
    if (t < BINS) {
        uint32_t v[SORT_WAVES];  // all reads in flight before the first write
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) v[w] = counts[w * BINS + t];
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) {
            before[w] = sum;
            sum += v[w];
        }
        incl = sum;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t o = __shfl_up(incl, m, 64);
            if (lane >= m) incl += o;
        }
        if (lane == 63) wsum[t >> 6] = incl;
    }
    __syncthreads();
    if (t < BINS) {
        uint32_t base = incl - sum;
        for (int w = 0; w < (t >> 6); ++w) base += wsum[w];
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) counts[w * BINS + t] = base + before[w];
    }
    __syncthreads();
}

// The kept tokens of the one-launch sort to their places: rounds of R tokens per thread.  m tokens with digits ldig and positions lpos,
// in order; start [BINS] (more than one round): where the next item of a digit goes; one round: its own scan and base say it.
template <int R>
__device__ __forceinline__ void place_items(uint32_t* __restrict__ keys, uint32_t* __restrict__ pos, uint32_t lo, uint32_t base, uint32_t m,
                                            const uint16_t* lpos, const uint8_t* ldig, uint32_t* counts, uint32_t* start, uint32_t* wsum) {
    constexpr uint32_t ROUND = R * SORT_NT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t r = 0; r < m; r += ROUND) {
        uint32_t dig[R], rank[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const uint32_t i = r + (wave * R + j) * 64 + lane;
            dig[j] = i < m ? ldig[i] : BINS - 1;  // past the list: behind every item of the last digit
        }
        rank_items<R>(dig, 0, rank, counts);
        scan_counts(counts, wsum);
        // counts[wave][d] - counts[0][d]: items of the digit in the waves in front
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const uint32_t i = r + (wave * R + j) * 64 + lane;
            if (i < m) {
                const uint32_t first = m > ROUND ? start[dig[j]] - counts[dig[j]] : base;
                const uint32_t to = first + counts[wave * BINS + dig[j]] + rank[j];
                keys[to] = lo + dig[j];
                pos[to] = lpos[i];
            }
        }
        if (m <= ROUND) return;
        __syncthreads();
        if (threadIdx.x < BINS) {  // the round's items of a digit: the distance to the next digit's start
            const uint32_t d = threadIdx.x;
            start[d] += (d + 1 < BINS ? counts[d + 1] : min(m - r, ROUND)) - counts[d];
        }
        __syncthreads();  // before the next round clears the counts
    }
}

// The one-launch sort: block b owns ids 256 b .. 256 b + 255 (the last block also the padding key `vocab`), n <= 1024 K.
// Reading: thread t of wave w holds tokens (w K + j) 64 + lane, all loads in flight at once.  Every block looks at every token, so
// what is done per token is kept to two comparisons and counts per lane; the few tokens of the block's own ids are then placed.
template <int K>
__global__ __launch_bounds__(SORT_NT) void sort_range_kernel(const int64_t* __restrict__ ids, uint32_t* __restrict__ keys, uint32_t* __restrict__ pos,
                                                             int n, i64 vocab) {
    FX_DYNAMIC_SMEM(uint32_t, smem);
    uint32_t* counts = smem;                                   // [SORT_WAVES][BINS]
    uint32_t* start = counts + SORT_WAVES * BINS;              // [BINS]
    uint32_t* wsum = start + BINS;                             // 4
    uint32_t* inside = wsum + 4;                               // [SORT_WAVES]: tokens of this block's ids per wave
    uint32_t* below = inside + SORT_WAVES;                     // [SORT_WAVES]: tokens of smaller ids per wave
    uint16_t* lpos = reinterpret_cast<uint16_t*>(below + SORT_WAVES);  // [K * SORT_NT]: the kept tokens, in order
    uint8_t* ldig = reinterpret_cast<uint8_t*>(lpos + K * SORT_NT);
    constexpr int RL = K < 4 ? K : 4;                          // tokens per thread and round of a long list
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t lo = blockIdx.x * BINS;
    uint32_t key[K];
    {
        int64_t id[K];  // unconditional loads: a branch around each would make them wait for one another
#pragma unroll
        for (int j = 0; j < K; ++j) id[j] = ids[min((wave * K + j) * 64 + lane, n - 1)];
#pragma unroll
        for (int j = 0; j < K; ++j) key[j] = (wave * K + j) * 64 + lane < n ? key_of(id[j], vocab) : 0xffffffffu;
    }
    uint32_t both = 0;  // tokens of this block's ids in the low half, of smaller ids in the high half: at most 64 K = 2048 per wave
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const uint32_t d = key[j] - lo;
        both += d < (uint32_t)BINS ? 1u : 0u;
        both += key[j] < lo ? 0x10000u : 0u;
    }
    both = wave_sum(both);
    if (lane == 0) {
        inside[wave] = both & 0xffffu;
        below[wave] = both >> 16;
    }
    if (threadIdx.x < BINS) start[threadIdx.x] = 0;
    __syncthreads();
    uint32_t at = 0, m = 0, base = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
        if (w < wave) at += inside[w];
        m += inside[w];
        base += below[w];
    }
    if (m == 0) return;  // block-uniform
    const bool many = m > RL * SORT_NT;  // more than one round: the digits are counted beforehand
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const uint32_t d = key[j] - lo;
        const bool mine = d < (uint32_t)BINS;
        const uint64_t who = __ballot(mine);
        if (who) {  // wave-uniform
            if (mine) {
                const uint32_t to = at + (uint32_t)__popcll(who & ((1ull << lane) - 1));
                lpos[to] = (uint16_t)((wave * K + j) * 64 + lane);
                ldig[to] = (uint8_t)d;
                if (many) atomicAdd(&start[d], 1u);  // whole numbers: any order
            }
            at += (uint32_t)__popcll(who);
        }
    }
    __syncthreads();
    if (many) {  // block-uniform
        uint32_t sum = 0, incl = 0;
        if (threadIdx.x < BINS) {
            sum = incl = start[threadIdx.x];
#pragma unroll
            for (int q = 1; q < 64; q <<= 1) {
                const uint32_t o = __shfl_up(incl, q, 64);
                if (lane >= q) incl += o;
            }
            if (lane == 63) wsum[wave] = incl;
        }
        __syncthreads();
        if (threadIdx.x < BINS) {
            uint32_t s = base + incl - sum;
            for (int w = 0; w < wave; ++w) s += wsum[w];
            start[threadIdx.x] = s;
        }
    }
    if (m <= SORT_NT) place_items<1>(keys, pos, lo, base, m, lpos, ldig, counts, start, wsum);
    else place_items<RL>(keys, pos, lo, base, m, lpos, ldig, counts, start, wsum);
}

// One radix pass over many tiles.  The first pass reads the ids themselves (keys_in == null).
constexpr int TILE_K = TILE / SORT_NT;
__device__ __forceinline__ void tile_items(const int64_t* ids, const uint32_t* keys_in, const uint32_t* pos_in, i64 n, i64 vocab, uint32_t (&key)[TILE_K],
                                           uint32_t (&at)[TILE_K]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j < TILE_K; ++j) {  // unconditional loads (the last token again past the end), all in flight
        const i64 i = (i64)blockIdx.x * TILE + (wave * TILE_K + j) * 64 + lane, ic = min(i, n - 1);
        key[j] = keys_in ? keys_in[ic] : key_of(ids[ic], vocab);
        at[j] = keys_in ? pos_in[ic] : (uint32_t)i;
        if (i >= n) key[j] = 0xffffffffu;
    }
}
__global__ __launch_bounds__(SORT_NT) void sort_count_kernel(const int64_t* __restrict__ ids, const uint32_t* __restrict__ keys_in, i64 n, i64 vocab,
                                                             int shift, uint32_t* __restrict__ table, unsigned tiles) {
    __shared__ uint32_t hist[BINS];
    for (int b = threadIdx.x; b < BINS; b += SORT_NT) hist[b] = 0;
    __syncthreads();
    uint32_t key[TILE_K];
#pragma unroll
    for (int j = 0; j < TILE_K; ++j) {
        const i64 i = min((i64)blockIdx.x * TILE + j * SORT_NT + threadIdx.x, n - 1);
        key[j] = keys_in ? keys_in[i] : key_of(ids[i], vocab);
    }
#pragma unroll
    for (int j = 0; j < TILE_K; ++j)
        if ((i64)blockIdx.x * TILE + j * SORT_NT + threadIdx.x < n) atomicAdd(&hist[(key[j] >> shift) & (BINS - 1)], 1u);  // whole numbers: any order
    __syncthreads();
    for (int b = threadIdx.x; b < BINS; b += SORT_NT) table[(i64)b * tiles + blockIdx.x] = hist[b];
}
// exclusive scan of `entries` counts in place, one block
__global__ __launch_bounds__(SORT_NT) void sort_scan_kernel(uint32_t* __restrict__ table, i64 entries) {
    __shared__ uint32_t wsum[SORT_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (i64 at = 0; at < entries; at += SORT_NT * 4) {
        const i64 i = at + (i64)threadIdx.x * 4;
        uint32_t v[4], sum = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            v[u] = i + u < entries ? table[i + u] : 0;
            sum += v[u];
        }
        uint32_t incl = sum;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t o = __shfl_up(incl, m, 64);
            if (lane >= m) incl += o;
        }
        if (lane == 63) wsum[wave] = incl;
        __syncthreads();
        uint32_t base = carry + incl - sum, all = 0;
        for (int w = 0; w < SORT_WAVES; ++w) {
            if (w < wave) base += wsum[w];
            all += wsum[w];
        }
        carry += all;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (i + u < entries) table[i + u] = base;
            base += v[u];
        }
    }
}
__global__ __launch_bounds__(SORT_NT) void sort_scatter_kernel(const int64_t* __restrict__ ids, const uint32_t* __restrict__ keys_in,
                                                               const uint32_t* __restrict__ pos_in, i64 n, i64 vocab, int shift,
                                                               const uint32_t* __restrict__ table, unsigned tiles, uint32_t* __restrict__ keys,
                                                               uint32_t* __restrict__ pos) {
    __shared__ uint32_t counts[SORT_WAVES * BINS];
    __shared__ uint32_t wsum[4];
    __shared__ uint32_t shiftby[BINS];
    uint32_t key[TILE_K], at[TILE_K], rank[TILE_K];
    tile_items(ids, keys_in, pos_in, n, vocab, key, at);
    rank_items<TILE_K>(key, shift, rank, counts);
    scan_counts(counts, wsum);
    // from the place among the tile's items to the place among all: the tile's start of the digit, table against counts[0]
    for (int b = threadIdx.x; b < BINS; b += SORT_NT) shiftby[b] = table[(i64)b * tiles + blockIdx.x] - counts[b];
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j < TILE_K; ++j) {
        const i64 i = (i64)blockIdx.x * TILE + (wave * TILE_K + j) * 64 + lane;
        if (i < n) {
            const uint32_t d = (key[j] >> shift) & (BINS - 1);
            const uint32_t to = counts[wave * BINS + d] + rank[j] + shiftby[d];
            keys[to] = key[j];
            pos[to] = at[j];
        }
    }
}

// ---- adding along the sorted order -------------------------------------------------------------------------------------------------
__device__ __forceinline__ i64 lower_bound(const uint32_t* __restrict__ keys, i64 n, uint32_t v) {  // first position with keys >= v
    i64 lo = 0, hi = n;
    while (lo < hi) {
        const i64 mid = (lo + hi) >> 1;
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

constexpr int ZROWS = 64;  // ids per block of the zero rows

struct Add {
    i64 n, vocab, D;
    int P;                 // sorted positions of a piece
    unsigned pieces, add_blocks;
    int tpp_log;           // threads of a piece: 2^tpp_log, they cover V << tpp_log columns per pass over blockIdx.y
};

// Blocks [0, add_blocks): pieces, 256 >> tpp_log of them each.  The blocks behind: zero rows.
// edge [piece][2][D]: the partial row of the run that starts at or before the piece's first position and crosses a border (slot 0),
// of the run that begins inside and crosses the end (slot 1).
template <typename T, int V>
__global__ __launch_bounds__(256) void embedding_add_kernel(const T* __restrict__ g, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                                                            T* __restrict__ dW, T* __restrict__ edge, T scale, const Add a) {
    if (blockIdx.x >= a.add_blocks) {
        __shared__ uint8_t present[ZROWS];
        const i64 v0 = (i64)(blockIdx.x - a.add_blocks) * ZROWS;
        if (threadIdx.x < ZROWS) {
            const i64 v = v0 + threadIdx.x;
            const i64 p = v < a.vocab ? lower_bound(keys, a.n, (uint32_t)v) : a.n;
            present[threadIdx.x] = v >= a.vocab || (p < a.n && keys[p] == (uint32_t)v);
        }
        __syncthreads();
        T zero[V];
#pragma unroll
        for (int u = 0; u < V; ++u) zero[u] = T(0);
        // all 256 threads run over (row, vector) pairs of this block's column range
        const i64 c0 = (i64)blockIdx.y * (V << a.tpp_log), c1 = min(a.D, c0 + (V << a.tpp_log));
        const int nv = (int)((c1 - c0 + V - 1) / V);
        for (int i = threadIdx.x; i < ZROWS * nv; i += 256) {
            const int r = i / nv;
            if (!present[r]) {
                const int j = (int)c0 + (i - r * nv) * V;
                T* const row = dW + (v0 + r) * a.D;
                if (j + V <= a.D) store_stream<V>(row + j, zero);
                else store_part<V>(row, j, (int)a.D, zero);
            }
        }
        return;
    }
    const int tpp = 1 << a.tpp_log;
    const i64 piece = (i64)blockIdx.x * (256 >> a.tpp_log) + (threadIdx.x >> a.tpp_log);
    const i64 col = (i64)blockIdx.y * (V << a.tpp_log) + (i64)(threadIdx.x & (tpp - 1)) * V;
    if (piece >= a.pieces || col >= a.D) return;
    const i64 p0 = piece * a.P, p1 = min(a.n, p0 + a.P);
    T acc[V];
#pragma unroll
    for (int u = 0; u < V; ++u) acc[u] = T(0);
    bool open = p0 > 0 && keys[p0 - 1] == keys[p0];  // the run in hand began in an earlier piece
    constexpr int U = 8;
    for (i64 p = p0; p < p1; p += U) {
        uint32_t k[U + 1];
        T v[U][V];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const i64 at = min(p + j, p1 - 1);
            k[j] = keys[at];
            load_part<V>(g + (i64)pos[at] * a.D, (int)col, (int)a.D, v[j]);
        }
        const i64 behind = min(p + U, p1);
        k[U] = behind < a.n ? keys[behind] : 0xffffffffu;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (p + j < p1) {
#pragma unroll
                for (int u = 0; u < V; ++u) acc[u] = acc[u] + v[j][u];
                const bool last = p + j + 1 == p1;
                const uint32_t next = last ? k[U] : k[j + 1];
                const bool ends = next != k[j];
                if (ends || last) {
                    if (k[j] < (uint32_t)a.vocab) {
                        if (open || !ends) {
                            store_part<V>(edge + (piece * 2 + (open ? 0 : (k[j] == keys[p0] ? 0 : 1))) * a.D, (int)col, (int)a.D, acc);
                        } else {
#pragma unroll
                            for (int u = 0; u < V; ++u) acc[u] = acc[u] * scale;
                            store_part<V>(dW + (i64)k[j] * a.D, (int)col, (int)a.D, acc);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < V; ++u) acc[u] = T(0);
                    open = false;
                }
            }
        }
    }
}

// Block b: the border between pieces b and b + 1.  The border where a crossing run crosses first adds all of the run's partial rows:
// four groups of threads take every fourth piece, then the four sums are added in order.
template <typename T, int V>
__global__ __launch_bounds__(256) void embedding_join_kernel(const uint32_t* __restrict__ keys, const T* __restrict__ edge, T* __restrict__ dW, T scale,
                                                             const Add a) {
    __shared__ T sm[4][64 * V];
    const i64 b = blockIdx.x, border = (b + 1) * a.P;  // < n
    const i64 first = b * a.P;  // piece b's first position
    const uint32_t k = keys[border], k1 = keys[border - 1], kf = keys[first], kb = keys[first > 0 ? first - 1 : 0];  // in flight together
    const bool whole = kf == k;                                // the run holds all of piece b
    // no run crosses here, or an earlier border has it (block-uniform)
    if ((k >= (uint32_t)a.vocab) | (k1 != k) | (whole & (first > 0) & (kb == k))) return;
    // the run's last piece: the first from b + 1 on that is the last one or ends before the run does; 64 pieces are looked at together
    const int lane = threadIdx.x & 63, group = threadIdx.x >> 6;
    i64 end = b + 1;
    for (;;) {
        const i64 q = min(end + lane, (i64)a.pieces - 1);
        const uint64_t stops = __ballot(q + 1 >= (i64)a.pieces || keys[(q + 1) * a.P] != k);
        if (stops) {
            end = min(end + __ffsll((unsigned long long)stops) - 1, (i64)a.pieces - 1);
            break;
        }
        end += 64;
    }
    const i64 col = ((i64)blockIdx.y * 64 + lane) * V;
    T acc[V];
#pragma unroll
    for (int u = 0; u < V; ++u) acc[u] = T(0);
    if (col < a.D) {
        constexpr int U = 8;
        for (i64 q = b + group; q <= end; q += 4 * U) {
            T v[U][V];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const i64 piece = q + 4 * j;
                if (piece <= end) {
                    load_part<V>(edge + (piece * 2 + (piece == b && !whole ? 1 : 0)) * a.D, (int)col, (int)a.D, v[j]);
                } else {
#pragma unroll
                    for (int u = 0; u < V; ++u) v[j][u] = T(0);
                }
            }
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int u = 0; u < V; ++u) acc[u] = acc[u] + v[j][u];
        }
    }
#pragma unroll
    for (int u = 0; u < V; ++u) sm[group][lane * V + u] = acc[u];
    __syncthreads();
    if (group == 0 && col < a.D) {
#pragma unroll
        for (int u = 0; u < V; ++u) {
            T s = acc[u];
            for (int w = 1; w < 4; ++w) s = s + sm[w][lane * V + u];
            acc[u] = s * scale;
        }
        store_part<V>(dW + (i64)k * a.D, (int)col, (int)a.D, acc);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
template <typename T>
int check(fx_ctx* c, const char* what, i64 n, i64 vocab, i64 D) {
    FX_CHECK_CTX(c);
    FX_REQUIRE(n >= 0 && vocab >= 1 && D >= 1, "%s: bad sizes (%lld tokens, table [%lld, %lld])", what, (long long)n, (long long)vocab, (long long)D);
    FX_REQUIRE(n < (1ll << 31) && vocab < (1ll << 31) && D < (1ll << 31), "%s: dimension exceeds 2^31", what);
    return FX_OK;
}

template <typename T>
int embedding_fwd(fx_ctx* c, const T* W, const int64_t* ids, T* out, i64 n, i64 vocab, i64 D, T scale) {
    if (int rc = check<T>(c, "fx_embedding_fwd", n, vocab, D)) return rc;
    if (n == 0) return FX_OK;
    FX_REQUIRE(W && ids && out, "fx_embedding_fwd: null pointer");
    FX_REQUIRE(!fx::overlap(out, n * D, W, vocab * D) && !fx::overlap((const char*)out, n * D * (i64)sizeof(T), (const char*)ids, n * 8),
               "fx_embedding_fwd: the output overlaps an input");
    constexpr int V = 16 / (int)sizeof(T);
    const i64 nv = fx::ceil_div(D, (i64)V), most = 0xffffffll * 1024 / nv;  // tokens of one launch, which has fewer than 2^32 threads
    for (i64 k = 0; k < n; k += most) {
        const i64 total = std::min(n - k, most) * nv;
        FX_LAUNCH(dim3((unsigned)fx::ceil_div(total, (i64)1024)), dim3(256), 0, c->stream,
                  (W, ids + k, out + k * D, total, (unsigned)nv, vocab, (int)D, scale), embedding_fwd_kernel<T, V>);
        FX_LAUNCH_CHECK();
    }
    return FX_OK;
}

template <int K> int sort_range(fx_ctx* c, const int64_t* ids, uint32_t* keys, uint32_t* pos, i64 n, i64 vocab) {
    constexpr size_t lds = (SORT_WAVES * BINS + BINS + 4 + 2 * SORT_WAVES) * 4 + (size_t)K * SORT_NT * 3;
    static const hipError_t attr = hipFuncSetAttribute((const void*)sort_range_kernel<K>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    FX_HIP_CHECK(attr);
    FX_LAUNCH(dim3((unsigned)(vocab / BINS + 1)), dim3(SORT_NT), lds, c->stream, (ids, keys, pos, (int)n, vocab), sort_range_kernel<K>);
    FX_LAUNCH_CHECK();
    return FX_OK;
}

template <typename T, int V>
int add_and_join(fx_ctx* c, const T* g, const uint32_t* keys, const uint32_t* pos, T* dW, T* edge, T scale, Add a) {
    a.tpp_log = 0;
    while (a.tpp_log < 8 && ((i64)V << a.tpp_log) < a.D) ++a.tpp_log;
    const i64 cols = fx::ceil_div(a.D, (i64)V << a.tpp_log), add_blocks = fx::ceil_div((i64)a.pieces, (i64)(256 >> a.tpp_log));
    const i64 blocks = add_blocks + fx::ceil_div(a.vocab, (i64)ZROWS);
    // a launch has fewer than 2^32 threads: 256 for 64 ids
    FX_REQUIRE(blocks < (1 << 24) && cols <= 65535 && fx::ceil_div(a.D, (i64)64 * V) <= 65535, "fx_embedding_bwd: too many rows or columns");
    a.add_blocks = (unsigned)add_blocks;
    FX_LAUNCH(dim3((unsigned)blocks, (unsigned)cols), dim3(256), 0, c->stream, (g, keys, pos, dW, edge, scale, a), embedding_add_kernel<T, V>);
    FX_LAUNCH_CHECK();
    if (a.pieces > 1) {
        FX_LAUNCH(dim3(a.pieces - 1, (unsigned)fx::ceil_div(a.D, (i64)64 * V)), dim3(256), 0, c->stream, (keys, edge, dW, scale, a), embedding_join_kernel<T, V>);
        FX_LAUNCH_CHECK();
    }
    return FX_OK;
}

template <typename T>
int embedding_bwd(fx_ctx* c, const T* g, const int64_t* ids, T* dW, i64 n, i64 vocab, i64 D, T scale) {
    if (int rc = check<T>(c, "fx_embedding_bwd", n, vocab, D)) return rc;
    FX_REQUIRE(dW && (n == 0 || (g && ids)), "fx_embedding_bwd: null pointer");
    FX_REQUIRE(!fx::overlap(dW, vocab * D, g, n * D) && !fx::overlap((const char*)dW, vocab * D * (i64)sizeof(T), (const char*)ids, n * 8),
               "fx_embedding_bwd: the output overlaps an input");
    std::lock_guard<std::mutex> lk(c->launch_mutex);
    constexpr int V = 16 / (int)sizeof(T);
    Add a;
    a.n = n;
    a.vocab = vocab;
    a.D = D;
    // pieces of 16 positions (about two per block slot at 16384 tokens); longer ones where there would be more than 4096 of them
    a.P = (int)std::max<i64>(16, fx::ceil_div(n, (i64)4096));
    a.pieces = (unsigned)fx::ceil_div(n, (i64)a.P);
    a.add_blocks = 0;
    a.tpp_log = 0;
    int passes = 1;
    while (passes < 4 && (vocab >> (BITS * passes)) != 0) ++passes;  // the largest key is vocab itself
    // The one-launch sort while its blocks are few, what they read together (8 bytes per token each) stays below 128 MB, and a block has
    // no more than a few rounds of tokens to place.  Whole call against the tiled passes (us), rows of 8 floats: 16000 tokens of 30000 ids
    // 24.6 / 42.4, of 260000 44 / 60, 32000 of 130000 40 / 62, 4000 of a million 64 / 73, 100 of four million 107 / 104; rows of 64 floats:
    // 32768 tokens of 1000 ids 46 / 49, of 500 58 / 49, 16384 of 500 35 / 40, 8192 of 200 29 / 25, 4096 of 200 19 / 23.
    const i64 ranges = vocab / BINS + 1;
    const bool small = n <= RANGE_MAX && ranges <= 8192 && n * ranges <= (1ll << 24) && n <= (passes == 1 ? 4096 : 8192 * ranges);
    const i64 tiles = fx::ceil_div(n, (i64)TILE), entries = tiles * BINS;
    // scratch: [keys][pos] once or twice, the table of counts, the partial rows
    const i64 nkeys = fx::ceil_div(n, (i64)64) * 64, lists = small ? 2 : 4;
    const i64 head = (lists * nkeys + (small ? 0 : entries)) * 4, edge_at = fx::ceil_div(head, (i64)256) * 256;
    char* scratch = (char*)c->get_scratch(edge_at + 2 * (i64)a.pieces * D * (i64)sizeof(T) + 256);
    if (!scratch) return FX_ERR_OOM;
    uint32_t* lists_p = (uint32_t*)scratch;
    uint32_t *keys = lists_p, *pos = lists_p + nkeys;
    if (n > 0 && small) {
        int rc;
        if (n <= SORT_NT) rc = sort_range<1>(c, ids, keys, pos, n, vocab);
        else if (n <= 4 * SORT_NT) rc = sort_range<4>(c, ids, keys, pos, n, vocab);
        else if (n <= 16 * SORT_NT) rc = sort_range<16>(c, ids, keys, pos, n, vocab);
        else rc = sort_range<32>(c, ids, keys, pos, n, vocab);
        if (rc) return rc;
    } else if (n > 0) {
        uint32_t* table = lists_p + 4 * nkeys;
        for (int p = 0; p < passes; ++p) {
            // the lists change places so that the last pass ends in the first pair
            const bool to_first = (passes - 1 - p) % 2 == 0;
            uint32_t *to = to_first ? lists_p : lists_p + 2 * nkeys, *from = to_first ? lists_p + 2 * nkeys : lists_p;
            const uint32_t* kin = p == 0 ? nullptr : from;
            FX_LAUNCH(dim3((unsigned)tiles), dim3(SORT_NT), 0, c->stream, (ids, kin, n, vocab, p * BITS, table, (unsigned)tiles), sort_count_kernel);
            FX_LAUNCH_CHECK();
            FX_LAUNCH(dim3(1), dim3(SORT_NT), 0, c->stream, (table, entries), sort_scan_kernel);
            FX_LAUNCH_CHECK();
            FX_LAUNCH(dim3((unsigned)tiles), dim3(SORT_NT), 0, c->stream,
                      (ids, kin, kin ? from + nkeys : nullptr, n, vocab, p * BITS, table, (unsigned)tiles, to, to + nkeys), sort_scatter_kernel);
            FX_LAUNCH_CHECK();
        }
    }
    T* edge = (T*)(scratch + edge_at);
    return add_and_join<T, V>(c, g, keys, pos, dW, edge, scale, a);
}
}  // namespace

#define FX_DEFINE_EMBEDDING(T, S)                                                                                                      \
    extern "C" int fx_embedding_fwd_##S(fx_ctx* c, const T* W, const int64_t* ids, T* out, int64_t n, int64_t vocab, int64_t D, T scale) { \
        return embedding_fwd<T>(c, W, ids, out, n, vocab, D, scale);                                                                  \
    }                                                                                                                                  \
    extern "C" int fx_embedding_bwd_##S(fx_ctx* c, const T* g, const int64_t* ids, T* dW, int64_t n, int64_t vocab, int64_t D, T scale) { \
        return embedding_bwd<T>(c, g, ids, dW, n, vocab, D, scale);                                                                   \
    }
FX_DEFINE_EMBEDDING(float, f32)
FX_DEFINE_EMBEDDING(double, f64)
