// Table lookup out[i] = scale * W[ids[i]] and its gradient dW[v] = scale * sum over ids[i] == v of g[i].
//
// The gradient sorts the token ids (stable radix sort on (id, position) pairs) and sums the rows of g in sorted order:
// the occurrences of one token become one RUN of neighbouring slots.  Slots are cut into tiles of equal length, so the
// work is even however often a token occurs; a run inside one tile is finished there, a run over several tiles leaves one
// fp32 partial row per tile and a second launch joins them.  No floating-point atomics: the order of every sum depends on
// the sizes and the ids alone.
#include "common.h"

namespace {

template <bool I64>
__device__ __forceinline__ int64_t ld_id(const void* __restrict__ ids, int64_t i) {
    return I64 ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}

// ------------------------------------------------------------------------------------------------ forward
// The output is a flat row of n * nv pieces of VEC elements; a thread moves U pieces 256 apart, so stores are contiguous
// whatever the width.  Piece -> row needs a division by nv: the block's first row comes from one 64-bit division (scalar),
// the rest from a multiplication by `magic` = ceil(2^32 / nv), exact while (256 U + nv) * nv < 2^32.
template <class T, int VEC, int U, bool I64>
__global__ __launch_bounds__(256) void k_embedding_fwd(const T* __restrict__ w, int64_t ldw, int64_t V, const void* __restrict__ ids,
                                                       int64_t n, uint32_t nv, uint32_t magic, float scale, T* __restrict__ out,
                                                       int64_t ldo) {
    typedef BgVec<T, VEC> Vec;
    const int64_t total = n * nv, p0 = (int64_t)blockIdx.x * (256 * U);
    const int64_t row0 = p0 / nv;
    const uint32_t rem0 = (uint32_t)(p0 - row0 * nv);
    int64_t row[U], id[U];
    uint32_t col[U];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t o = rem0 + threadIdx.x + 256 * u;
        const uint32_t q = magic ? __umulhi(o, magic) : o;                 // magic 0: nv == 1
        row[u] = row0 + q;
        col[u] = (o - q * nv) * VEC;
        live[u] = p0 + threadIdx.x + 256 * u < total;
        id[u] = live[u] ? ld_id<I64>(ids, row[u]) : -1;
    }
    Vec x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (id[u] >= 0 && id[u] < V) x[u] = *reinterpret_cast<const Vec*>(w + id[u] * ldw + col[u]);
        else
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[u].v[k] = (T)0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (!live[u]) continue;
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[u].v[k] = (T)((float)x[u].v[k] * scale);
        *reinterpret_cast<Vec*>(out + row[u] * ldo + col[u]) = x[u];
    }
}

// ------------------------------------------------------------------------------------------------ stable sort of the ids
// Least significant digit first, one pass = a histogram per tile of keys and a placement.  The key of a missing token is
// V, behind every row.  Both launches carry extra workgroups that zero a share of dW meanwhile: the sort of a batch's
// tokens is bound by latency, not by memory.
constexpr int kDigitBits = 9;
constexpr int kBins = 1 << kDigitBits;
constexpr int kSortThreads = 512;

struct Fill { uint4* p; int64_t n16; };                  // n16 pieces of 16 bytes

__device__ __forceinline__ void d_fill(Fill f, int64_t block, int64_t blocks) {
    for (int64_t i = block * kSortThreads + threadIdx.x; i < f.n16; i += blocks * kSortThreads) f.p[i] = make_uint4(0u, 0u, 0u, 0u);
}

template <int SRC>      // 0: int64 ids, 1: int32 ids, 2: keys of an earlier pass
__device__ __forceinline__ int32_t ld_key(const void* __restrict__ src, int64_t i, int64_t V) {
    if (SRC == 2) return static_cast<const int32_t*>(src)[i];
    const int64_t id = ld_id<SRC == 0>(src, i);
    return (int32_t)(id >= 0 && id < V ? id : V);
}

// hist[bin * n_tiles + tile]
template <int SRC, int ROUNDS>
__global__ __launch_bounds__(kSortThreads) void k_sort_hist(const void* __restrict__ src, int64_t n, int64_t V, int shift, int bins,
                                                            int32_t* __restrict__ hist, int n_tiles, Fill fill) {
    if ((int)blockIdx.x >= n_tiles) { d_fill(fill, blockIdx.x - n_tiles, gridDim.x - n_tiles); return; }
    __shared__ int32_t h[kBins];
    if (threadIdx.x < kBins) h[threadIdx.x] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * (kSortThreads * ROUNDS);
    int32_t key[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t i = base + r * kSortThreads + threadIdx.x;
        key[r] = i < n ? ld_key<SRC>(src, i, V) : -1;
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (key[r] >= 0) atomicAdd(&h[(key[r] >> shift) & (bins - 1)], 1);
    __syncthreads();
    if ((int)threadIdx.x < bins) hist[(int64_t)threadIdx.x * n_tiles + blockIdx.x] = h[threadIdx.x];
}

// in place: hist[bin][tile] -> number of that bin's keys in earlier tiles; total[bin] = all of them.  One wave per bin.
__global__ __launch_bounds__(256) void k_sort_scan(int32_t* __restrict__ hist, int n_tiles, int bins, int32_t* __restrict__ total) {
    const int bin = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (bin >= bins) return;
    int32_t* h = hist + (int64_t)bin * n_tiles;
    int32_t carry = 0;
    for (int t0 = 0; t0 < n_tiles; t0 += 64) {
        const int t = t0 + lane;
        const int32_t v = t < n_tiles ? h[t] : 0;
        int32_t x = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int32_t y = __shfl_up(x, off, 64);
            if (lane >= off) x += y;
        }
        if (t < n_tiles) h[t] = carry + x - v;
        carry += __shfl(x, 63, 64);
    }
    if (lane == 0) total[bin] = carry;
}

// Placement.  A wave owns 64 * ROUNDS consecutive keys; the rank of a key among its wave's equal digits comes from
// ballots over the digit's bits, then the waves' and the tiles' counts are added: stable by construction.
template <int SRC, int ROUNDS, bool SCANNED>
__global__ __launch_bounds__(kSortThreads) void k_sort_place(const void* __restrict__ src, const int32_t* __restrict__ pos_in, int64_t n,
                                                             int64_t V, int shift, int bits, const int32_t* __restrict__ hist,
                                                             const int32_t* __restrict__ total, int n_tiles,
                                                             int32_t* __restrict__ key_out, int32_t* __restrict__ pos_out, Fill fill) {
    if ((int)blockIdx.x >= n_tiles) { d_fill(fill, blockIdx.x - n_tiles, gridDim.x - n_tiles); return; }
    constexpr int kWaves = kSortThreads / 64;
    __shared__ int32_t cnt[kWaves][kBins];
    __shared__ int32_t wsum[kWaves];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, bins = 1 << bits;
    const int64_t first = (int64_t)blockIdx.x * (kSortThreads * ROUNDS) + wave * (64 * ROUNDS) + lane;
    int32_t key[ROUNDS], pos[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t i = first + 64 * r;
        key[r] = i < n ? ld_key<SRC>(src, i, V) : -1;
        pos[r] = i < n ? (SRC == 2 ? pos_in[i] : (int32_t)i) : 0;
    }
    for (int w = 0; w < kWaves; ++w) cnt[w][t] = 0;                      // kSortThreads == kBins
    int32_t before = 0, all = 0;                                         // of bin t: keys in earlier tiles, in all tiles
    if (t < bins) {
        const int32_t* h = hist + (int64_t)t * n_tiles;
        if (SCANNED) { before = h[blockIdx.x]; all = total[t]; }
        else
            for (int k = 0; k < n_tiles; ++k) {
                const int32_t v = h[k];
                all += v;
                before += k < (int)blockIdx.x ? v : 0;
            }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int d = (key[r] >> shift) & (bins - 1);
        uint64_t peers = __ballot(key[r] >= 0);
        for (int b = 0; b < bits; ++b) {
            const uint64_t m = __ballot((d >> b) & 1);
            peers &= ((d >> b) & 1) ? m : ~m;
        }
        const int below = __popcll(peers & ((1ull << lane) - 1));
        const int32_t c = cnt[wave][d];                                  // one wave, one row of cnt: LDS keeps its order
        __builtin_amdgcn_wave_barrier();
        if (key[r] >= 0 && below == 0) cnt[wave][d] = c + __popcll(peers);
        __builtin_amdgcn_wave_barrier();
        rank[r] = c + below;
    }
    // exclusive sum of `all` over the bins
    int32_t x = all;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int32_t y = __shfl_up(x, off, 64);
        if (lane >= off) x += y;
    }
    if (lane == 63) wsum[wave] = x;
    __syncthreads();
    int32_t base = before + x - all;
    for (int w = 0; w < wave; ++w) base += wsum[w];
    for (int w = 0; w < kWaves; ++w) { const int32_t c = cnt[w][t]; cnt[w][t] = base; base += c; }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        if (key[r] < 0) continue;
        const int32_t dst = cnt[wave][(key[r] >> shift) & (bins - 1)] + rank[r];
        key_out[dst] = key[r];
        pos_out[dst] = pos[r];
    }
}

// ------------------------------------------------------------------------------------------------ sums over the runs
// LG lanes carry one tile of C slots over LG * EPT columns; EPT elements per lane, one piece (WIDE) or LG apart.
template <class T, int EPT, bool WIDE>
struct RowPiece {
    alignas(sizeof(T) * EPT) T v[EPT];
    __device__ __forceinline__ void load(const T* __restrict__ row, int c0, int lane, int LG, int64_t D) {
        if (WIDE) {
            const int64_t c = c0 + lane * EPT;
            if (c < D) *reinterpret_cast<BgVec<T, EPT>*>(v) = *reinterpret_cast<const BgVec<T, EPT>*>(row + c);
        } else {
#pragma unroll
            for (int k = 0; k < EPT; ++k) { const int64_t c = c0 + lane + k * LG; if (c < D) v[k] = row[c]; }
        }
    }
};
template <class T, int EPT, bool WIDE, bool ROUND>      // ROUND: to T with the scale; else fp32 as it is
__device__ __forceinline__ void st_row(void* __restrict__ dst, const float (&acc)[EPT], float scale, int c0, int lane, int LG, int64_t D) {
    if (ROUND) {
        T* row = static_cast<T*>(dst);
        if (WIDE) {
            const int64_t c = c0 + lane * EPT;
            BgVec<T, EPT> o;
#pragma unroll
            for (int k = 0; k < EPT; ++k) o.v[k] = (T)(acc[k] * scale);
            if (c < D) *reinterpret_cast<BgVec<T, EPT>*>(row + c) = o;
        } else {
#pragma unroll
            for (int k = 0; k < EPT; ++k) { const int64_t c = c0 + lane + k * LG; if (c < D) row[c] = (T)(acc[k] * scale); }
        }
    } else {
        float* row = static_cast<float*>(dst);
#pragma unroll
        for (int k = 0; k < EPT; ++k) { const int64_t c = c0 + (WIDE ? lane * EPT + k : lane + k * LG); if (c < D) row[c] = acc[k]; }
    }
}

// part[(2 * tile + which) * D + c]: which 0 = the run that began in an earlier tile, 1 = one that goes on into the next
template <class T, int EPT, bool WIDE>
__global__ __launch_bounds__(256) void k_embedding_runs(const int32_t* __restrict__ key, const int32_t* __restrict__ pos, int64_t n,
                                                        int32_t V, const T* __restrict__ g, int64_t ldg, int64_t D, float scale,
                                                        T* __restrict__ dw, float* __restrict__ part, int C, int LG, int64_t n_tiles) {
    constexpr int U = 4;
    const int lane = threadIdx.x & (LG - 1);
    const int64_t tile = (int64_t)blockIdx.x * (256 / LG) + threadIdx.x / LG;
    if (tile >= n_tiles) return;
    const int c0 = blockIdx.y * (LG * EPT);
    const int64_t k0 = tile * C, k1 = k0 + C < n ? k0 + C : n;
    int32_t cur = key[k0];
    bool earlier = k0 > 0 && key[k0 - 1] == cur;
    const int32_t after = k1 < n ? key[k1] : -1;
    float acc[EPT];
#pragma unroll
    for (int e = 0; e < EPT; ++e) acc[e] = 0.f;
    for (int64_t k = k0; k < k1; k += U) {
        int32_t kk[U];
        RowPiece<T, EPT, WIDE> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            kk[u] = k + u < k1 ? key[k + u] : -1;
            if (kk[u] >= 0 && kk[u] < V) x[u].load(g + (int64_t)pos[k + u] * ldg, c0, lane, LG, D);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kk[u] < 0) continue;
            if (kk[u] != cur) {
                if (cur < V) {
                    if (earlier) st_row<T, EPT, WIDE, false>(part + 2 * tile * D, acc, 1.f, c0, lane, LG, D);
                    else st_row<T, EPT, WIDE, true>(dw + (int64_t)cur * D, acc, scale, c0, lane, LG, D);
                }
                cur = kk[u];
                earlier = false;
#pragma unroll
                for (int e = 0; e < EPT; ++e) acc[e] = 0.f;
            }
            if (cur < V)
#pragma unroll
                for (int e = 0; e < EPT; ++e) acc[e] += (float)x[u].v[e];
        }
    }
    if (cur < V) {
        if (earlier) st_row<T, EPT, WIDE, false>(part + 2 * tile * D, acc, 1.f, c0, lane, LG, D);
        else if (after == cur) st_row<T, EPT, WIDE, false>(part + (2 * tile + 1) * D, acc, 1.f, c0, lane, LG, D);
        else st_row<T, EPT, WIDE, true>(dw + (int64_t)cur * D, acc, scale, c0, lane, LG, D);
    }
}

// The run that begins in tile blockIdx.x and goes on: its own partial and the following tiles' are added, kJoin threads
// deep (strided over the tiles) and then down those kJoin in order.
constexpr int kJoin = 8, kJoinCols = 32;
template <class T>
__global__ __launch_bounds__(kJoin* kJoinCols) void k_embedding_join(const int32_t* __restrict__ key, int64_t n, int32_t V,
                                                                     const float* __restrict__ part, int C, int64_t n_tiles, int64_t D,
                                                                     float scale, T* __restrict__ dw) {
    const int64_t tile = blockIdx.x, k0 = tile * C, k1 = k0 + C;
    if (k1 >= n) return;
    const int32_t cur = key[k1 - 1];
    if (cur >= V || key[k1] != cur) return;
    if (k0 > 0 && key[k0] == cur && key[k0 - 1] == cur) return;          // it began earlier: that tile joins it
    int64_t lo = k1, hi = n - 1;                                         // last slot of the run
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        if (key[mid] == cur) lo = mid; else hi = mid - 1;
    }
    const int64_t last = lo / C;
    __shared__ float sum[kJoin][kJoinCols];
    const int tx = threadIdx.x % kJoinCols, ty = threadIdx.x / kJoinCols;
    const int64_t c = (int64_t)blockIdx.y * kJoinCols + tx;
    float s = ty == 0 && c < D ? part[(2 * tile + 1) * D + c] : 0.f;
    if (c < D)
        for (int64_t t = tile + 1 + ty; t <= last; t += kJoin) s += part[2 * t * D + c];
    sum[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < D) {
        for (int y = 1; y < kJoin; ++y) s += sum[y][tx];
        dw[(int64_t)cur * D + c] = (T)(s * scale);
    }
}

struct BwdPlan {                       // pieces of the workspace (bytes) and the shape of the launches: functions of n, V, D only
    int passes, bits, rounds, n_tiles;
    int64_t key_a, key_b, pos_a, pos_b, hist, total, part, bytes;
    int C, LG;
    int64_t run_tiles;
};

BwdPlan bwd_plan(int64_t n, int64_t V, int64_t D) {
    BwdPlan p;
    int b = 1;
    while (V >> b) ++b;                                   // keys go up to V
    p.passes = (b + kDigitBits - 1) / kDigitBits;
    p.bits = (b + p.passes - 1) / p.passes;
    p.rounds = n <= 65536 ? 2 : 8;
    p.n_tiles = (int)((n + kSortThreads * p.rounds - 1) / (kSortThreads * p.rounds));
    const int64_t nv = (D + 3) / 4;
    p.LG = nv > 32 ? 64 : nv > 16 ? 32 : nv > 8 ? 16 : 8;
    p.C = 128;
    while (p.C > 16 && n * nv / ((int64_t)p.C * 64) < 4096) p.C /= 2;
    p.run_tiles = (n + p.C - 1) / p.C;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    p.key_a = take(4 * n); p.key_b = take(4 * n); p.pos_a = take(4 * n); p.pos_b = take(4 * n);
    p.hist = take((int64_t)4 * kBins * p.n_tiles);
    p.total = take(4 * kBins);
    p.part = take(8 * p.run_tiles * D);
    p.bytes = at;
    return p;
}

constexpr int64_t kMaxWidth = 1 << 15;      // (1024 + nv) * nv < 2^32 for `magic`
constexpr int64_t kMaxPieces = (int64_t)1 << 33;       // work-items of a launch stay below 2^32

template <class T, int VEC, bool I64>
int launch_fwd(const T* w, int64_t ldw, int64_t V, const void* ids, int64_t n, int64_t D, float scale, T* out, int64_t ldo,
                hipStream_t s) {
    const uint32_t nv = (uint32_t)(D / VEC);
    const uint32_t magic = nv == 1 ? 0u : (uint32_t)(((1ull << 32) + nv - 1) / nv);
    if (n > kMaxPieces / nv) return BG_ERR_SHAPE;
    const int64_t total = n * nv;
    if (total <= 1 << 16)
        k_embedding_fwd<T, VEC, 1, I64><<<bg_grid_for(total, 256, 1 << 30), 256, 0, s>>>(w, ldw, V, ids, n, nv, magic, scale, out, ldo);
    else
        k_embedding_fwd<T, VEC, 4, I64><<<bg_grid_for(total, 1024, 1 << 30), 256, 0, s>>>(w, ldw, V, ids, n, nv, magic, scale, out, ldo);
    BG_LAUNCH_CHECK();
    return BG_OK;
}

template <int SRC>
void launch_sort_pass(const BwdPlan& p, const void* src, const int32_t* pos_in, int64_t n, int64_t V, int shift, int32_t* hist,
                      int32_t* total, int32_t* key_out, int32_t* pos_out, Fill f0, Fill f1, hipStream_t s) {
    const int bins = 1 << p.bits;
    const int b0 = f0.n16 ? bg_grid_for(f0.n16, kSortThreads * 4, 1024) : 0, b1 = f1.n16 ? bg_grid_for(f1.n16, kSortThreads * 4, 1024) : 0;
    const bool scanned = p.n_tiles > 64;
    if (p.rounds == 2) k_sort_hist<SRC, 2><<<p.n_tiles + b0, kSortThreads, 0, s>>>(src, n, V, shift, bins, hist, p.n_tiles, f0);
    else k_sort_hist<SRC, 8><<<p.n_tiles + b0, kSortThreads, 0, s>>>(src, n, V, shift, bins, hist, p.n_tiles, f0);
    if (scanned) k_sort_scan<<<(bins + 3) / 4, 256, 0, s>>>(hist, p.n_tiles, bins, total);
    if (p.rounds == 2)
        k_sort_place<SRC, 2, false><<<p.n_tiles + b1, kSortThreads, 0, s>>>(src, pos_in, n, V, shift, p.bits, hist, total, p.n_tiles,
                                                                           key_out, pos_out, f1);
    else if (scanned)
        k_sort_place<SRC, 8, true><<<p.n_tiles + b1, kSortThreads, 0, s>>>(src, pos_in, n, V, shift, p.bits, hist, total, p.n_tiles,
                                                                          key_out, pos_out, f1);
    else
        k_sort_place<SRC, 8, false><<<p.n_tiles + b1, kSortThreads, 0, s>>>(src, pos_in, n, V, shift, p.bits, hist, total, p.n_tiles,
                                                                           key_out, pos_out, f1);
}

__global__ void k_fill_tail(uint8_t* p, int n) { if ((int)threadIdx.x < n) p[threadIdx.x] = 0; }

}  // namespace

extern "C" int bg_embedding_fwd(int dtype, const void* weight, int64_t ldw, int64_t V, const void* ids, int ids_is_64, int64_t n,
                                int64_t D, float scale, void* out, int64_t ldo, bgStream stream) {
    const int es = bg_elem_size(dtype);
    if (!es || n < 0 || D < 0 || V < 0 || ldw < D || ldo < D) return BG_ERR_ARG;
    if (n == 0 || D == 0) return BG_OK;
    if ((V > 0 && !weight) || !ids || !out) return BG_ERR_ARG;
    if (D > kMaxWidth) return BG_ERR_SHAPE;
    auto fits = [&](int vec) {
        const uintptr_t bytes = (uintptr_t)vec * es;
        return D % vec == 0 && ldw % vec == 0 && ldo % vec == 0 && (uintptr_t)weight % bytes == 0 && (uintptr_t)out % bytes == 0;
    };
    return bg_dispatch_dtype(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        constexpr int W = 16 / sizeof(T);
        const T* w = static_cast<const T*>(weight);
        T* o = static_cast<T*>(out);
        hipStream_t s = (hipStream_t)stream;
        if (fits(W))
            return ids_is_64 ? launch_fwd<T, W, true>(w, ldw, V, ids, n, D, scale, o, ldo, s)
                             : launch_fwd<T, W, false>(w, ldw, V, ids, n, D, scale, o, ldo, s);
        return ids_is_64 ? launch_fwd<T, 1, true>(w, ldw, V, ids, n, D, scale, o, ldo, s)
                         : launch_fwd<T, 1, false>(w, ldw, V, ids, n, D, scale, o, ldo, s);
    });
}

extern "C" int64_t bg_embedding_bwd_workspace(int64_t n, int64_t V, int64_t D) {
    if (n <= 0 || V <= 0 || D <= 0 || n > ((int64_t)1 << 30) || V >= ((int64_t)1 << 31) - 1 || D > kMaxWidth) return 0;
    return bwd_plan(n, V, D).bytes;
}

extern "C" int bg_embedding_bwd(int dtype, const void* g, int64_t ldg, const void* ids, int ids_is_64, int64_t n, int64_t D, int64_t V,
                                float scale, void* dw, void* ws, int64_t ws_bytes, bgStream stream) {
    const int es = bg_elem_size(dtype);
    if (!es || n < 0 || D < 0 || V < 0 || ldg < D) return BG_ERR_ARG;
    if (V == 0 || D == 0) return BG_OK;
    if (!dw || (n > 0 && (!g || !ids || !ws))) return BG_ERR_ARG;
    if (n > ((int64_t)1 << 30) || V >= ((int64_t)1 << 31) - 1 || D > kMaxWidth) return BG_ERR_SHAPE;
    if (!bg_aligned16(dw) || (n > 0 && !bg_aligned16(ws))) return BG_ERR_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    const int64_t bytes = V * D * es, n16 = bytes / 16;
    if (bytes % 16) {
        k_fill_tail<<<1, 16, 0, s>>>(static_cast<uint8_t*>(dw) + n16 * 16, (int)(bytes % 16));
        BG_LAUNCH_CHECK();
    }
    if (n == 0) return bg_zero_bytes(dw, n16 * 16, stream);
    const BwdPlan p = bwd_plan(n, V, D);
    if (ws_bytes < p.bytes) return BG_ERR_SCRATCH;
    char* base = static_cast<char*>(ws);
    int32_t* key[2] = {reinterpret_cast<int32_t*>(base + p.key_a), reinterpret_cast<int32_t*>(base + p.key_b)};
    int32_t* pos[2] = {reinterpret_cast<int32_t*>(base + p.pos_a), reinterpret_cast<int32_t*>(base + p.pos_b)};
    int32_t* hist = reinterpret_cast<int32_t*>(base + p.hist);
    int32_t* total = reinterpret_cast<int32_t*>(base + p.total);
    float* part = reinterpret_cast<float*>(base + p.part);
    const int64_t share = (n16 + 2 * p.passes - 1) / (2 * p.passes);
    auto fill = [&](int k) {
        const int64_t a = share * k < n16 ? share * k : n16, b = share * (k + 1) < n16 ? share * (k + 1) : n16;
        return Fill{static_cast<uint4*>(dw) + a, b - a};
    };
    for (int q = 0; q < p.passes; ++q) {
        const int o = q & 1, shift = q * p.bits;
        if (q == 0 && ids_is_64) launch_sort_pass<0>(p, ids, nullptr, n, V, shift, hist, total, key[o], pos[o], fill(0), fill(1), s);
        else if (q == 0) launch_sort_pass<1>(p, ids, nullptr, n, V, shift, hist, total, key[o], pos[o], fill(0), fill(1), s);
        else launch_sort_pass<2>(p, key[1 - o], pos[1 - o], n, V, shift, hist, total, key[o], pos[o], fill(2 * q), fill(2 * q + 1), s);
        BG_LAUNCH_CHECK();
    }
    const int32_t *k = key[(p.passes - 1) & 1], *ps = pos[(p.passes - 1) & 1];
    return bg_dispatch_dtype(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        constexpr int W = 16 / sizeof(T);
        const T* gg = static_cast<const T*>(g);
        T* d = static_cast<T*>(dw);
        const bool wide = D % W == 0 && ldg % W == 0 && bg_aligned16(g);
        const int64_t pieces = (D + W - 1) / W;
        const int LG = pieces > 32 ? 64 : pieces > 16 ? 32 : pieces > 8 ? 16 : 8;
        const dim3 grid((unsigned)((p.run_tiles + 256 / LG - 1) / (256 / LG)), (unsigned)((pieces + LG - 1) / LG));
        if (wide) k_embedding_runs<T, W, true><<<grid, 256, 0, s>>>(k, ps, n, (int32_t)V, gg, ldg, D, scale, d, part, p.C, LG, p.run_tiles);
        else k_embedding_runs<T, W, false><<<grid, 256, 0, s>>>(k, ps, n, (int32_t)V, gg, ldg, D, scale, d, part, p.C, LG, p.run_tiles);
        BG_LAUNCH_CHECK();
        if (p.run_tiles > 1) {
            k_embedding_join<T><<<dim3((unsigned)p.run_tiles, (unsigned)((D + kJoinCols - 1) / kJoinCols)), kJoin * kJoinCols, 0, s>>>(
                k, n, (int32_t)V, part, p.C, p.run_tiles, D, scale, d);
            BG_LAUNCH_CHECK();
        }
        return BG_OK;
    });
}
