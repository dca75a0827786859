// Gated linear recurrence along the rows of each segment, a scan over long sequences, and its backward pass.
//
//   a = sigmoid(gate), c = 1 - a = sigmoid(-gate)          (both from one exponential, each to full relative accuracy)
//   forward :  h_t = a_t h_{t-1} + c_t x_t                 h before a segment's first row = h0 (or 0)
//   backward:  mu_t = a_t (dh_t + mu_{t+1})                mu after a segment's last row = dlast (or 0)
//              dx_t = c_t (dh_t + mu_{t+1}),  dgate_t = (dh_t + mu_{t+1}) (h_{t-1} - x_t) a_t c_t,  dh0 = mu_first
// Both are chains of maps  s -> A s + B, which compose:  (A2, B2) o (A1, B1) = (A2 A1, A2 B1 + B2).  A segment's first row
// is a CUT: the map that forgets what comes in (kept as a flag, not as A = 0: 0 * inf of another segment would leak).
// Rows are cut into tiles whatever the segments are; a workgroup composes a tile's rows in registers, the tiles are
// composed along each column, and the tile's rows are walked again from the state that comes in.
// h is never read back: the backward pass rebuilds it in registers from the fp32 state kept at the head of every tile.
#include <type_traits>
#include "common.h"

namespace {

constexpr int kTileElems = 4096;                 // rows of a tile * column groups (of 4 columns) of a tile
constexpr int kCarryCols = 32, kCarrySlices = 32;

struct Segs { const int32_t* ptr; int64_t S, N, T; };      // ptr NULL: S segments of T rows

// REV walks the rows upwards: LOGICAL row r is row N - 1 - r, logical segment j is segment S - 1 - j
template <bool REV>
__device__ __forceinline__ int64_t seg_lo(const Segs& g, int64_t j) {                // logical first row of logical segment j
    const int64_t k = REV ? g.S - j : j;
    int64_t p = g.ptr ? (int64_t)g.ptr[k] : k * g.T;
    p = p < 0 ? 0 : p > g.N ? g.N : p;
    return REV ? g.N - p : p;
}

// first[r] / last[r]: the segment whose first / last row is row r of the tile, -1: none; first[r] = -2: r is in no segment.
// The segment of the tile's first row is found by a search THREADS wide: one round for up to THREADS segments.
template <bool REV>
__device__ __forceinline__ void mark_tile(const Segs& g, int64_t row0, int rows, int32_t* first, int32_t* last) {
    const int t = threadIdx.x, threads = blockDim.x;
    const int64_t lo_all = seg_lo<REV>(g, 0), hi_all = seg_lo<REV>(g, g.S), end = row0 + rows;
    for (int r = t; r < rows; r += threads) {
        first[r] = row0 + r >= lo_all && row0 + r < hi_all ? -1 : -2;
        last[r] = -1;
    }
    int64_t lo = 0, hi = g.S;                    // lo -> how many segments begin at or before row0
    if (!g.ptr) lo = hi = g.T > 0 ? row0 / g.T + 1 : 0;
    while (lo < hi) {
        const int64_t step = (hi - lo + threads - 1) / threads, j = lo + t * step;
        const int c = __syncthreads_count(j < hi && seg_lo<REV>(g, j) <= row0);
        const int64_t nlo = c ? lo + (c - 1) * step + 1 : lo, nhi = c ? lo + c * step : lo;
        lo = nlo;
        hi = nhi < hi ? nhi : hi;
    }
    __syncthreads();
    for (int64_t j = (lo > 0 ? lo - 1 : 0) + t; j < g.S; j += threads) {
        const int64_t a = seg_lo<REV>(g, j), b = seg_lo<REV>(g, j + 1);
        if (a >= end) break;
        if (a >= b) continue;
        const int32_t s = (int32_t)(REV ? g.S - 1 - j : j);
        if (a >= row0) first[a - row0] = s;
        if (b - 1 >= row0 && b - 1 < end) last[b - 1 - row0] = s;
    }
    __syncthreads();
}

// a = sigmoid(g), c = sigmoid(-g) without cancellation: e = exp(-|g|) <= 1, r = 1 / (1 + e); one of them is r, the other e r.
// The product |g| log2(e) is carried in two parts, so e is good to ~2 ulp at any g.
__device__ __forceinline__ void gate_pair(float g, float& a, float& c) {
    const float m = fabsf(g), p = m * -1.4426950408889634f;
    const float lo = fmaf(m, -1.4426950408889634f, -p) - m * 1.9259629911266175e-8f;
    float e = __builtin_amdgcn_exp2f(p);
    e = fmaf(e, lo * 0.6931471805599453f, e);
    if (!(m < 120.f)) e = g != g ? g : 0.f;                              // (the correction term is inf * 0 for an infinite gate)
    const float r = __builtin_amdgcn_rcpf(1.f + e), er = e * r;
    a = g < 0.f ? er : r;
    c = g < 0.f ? r : er;
}

// four columns of a row: one piece (WIDE) or CG apart
template <class T, bool WIDE>
__device__ __forceinline__ void ld4(const T* __restrict__ row, int64_t c, int CG, int64_t D, float (&v)[4]) {
    if (WIDE) {
        if (c < D) {
            const BgVec<T, 4> x = *reinterpret_cast<const BgVec<T, 4>*>(row + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)x.v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (c + e * CG < D) v[e] = (float)row[c + e * CG];
    }
}
template <class T, bool WIDE>
__device__ __forceinline__ void st4(T* __restrict__ row, int64_t c, int CG, int64_t D, const float (&v)[4]) {
    if (WIDE) {
        BgVec<T, 4> x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x.v[e] = bg_round<T>(v[e]);
        if (c < D) *reinterpret_cast<BgVec<T, 4>*>(row + c) = x;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (c + e * CG < D) row[c + e * CG] = bg_round<T>(v[e]);
    }
}

struct Map4 { float A[4], B[4]; };
struct TileAgg { float* ab; int32_t* cut; };     // ab[(2 * tile + which) * D + c], cut[tile]

// The maps of the tile's row groups -> LDS; then `in` (the state that enters the tile) becomes the state that enters this
// thread's row group (from below: groups 0 .. rg - 1; from above with UP: groups RG - 1 .. rg + 1).
template <bool UP>
__device__ __forceinline__ void enter_group(const float (*sA)[4], const float (*sB)[4], const int32_t* sCut, int cg, int rg, int CG,
                                            int RG, float (&s)[4]) {
    for (int k = UP ? RG - 1 : 0; UP ? k > rg : k < rg; k += UP ? -1 : 1) {
        const bool cut = sCut[k] != 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float b = sB[k * CG + cg][e];
            s[e] = cut ? b : fmaf(sA[k * CG + cg][e], s[e], b);
        }
    }
}
template <bool UP>
__device__ __forceinline__ void write_agg(const float (*sA)[4], const float (*sB)[4], const int32_t* sCut, int cg, int CG, int RG,
                                          TileAgg agg, int64_t tile, int64_t c0, int64_t D, bool wide) {
    float A[4] = {1.f, 1.f, 1.f, 1.f}, B[4] = {0.f, 0.f, 0.f, 0.f};
    int cut_any = 0;
    for (int i = 0; i < RG; ++i) {
        const int k = UP ? RG - 1 - i : i;
        const bool cut = sCut[k] != 0;
        cut_any |= cut;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = sA[k * CG + cg][e], b = sB[k * CG + cg][e];
            B[e] = cut ? b : fmaf(a, B[e], b);
            A[e] = cut ? 0.f : a * A[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t c = wide ? c0 + cg * 4 + e : c0 + cg + e * CG;
        if (c < D) { agg.ab[2 * tile * D + c] = A[e]; agg.ab[(2 * tile + 1) * D + c] = B[e]; }
    }
    if (cg == 0 && blockIdx.y == 0) agg.cut[tile] = cut_any;
}

// ------------------------------------------------------------------------------------------------ forward
// APPLY false: the tile's map -> agg.  APPLY true: heads[tile] enters, h and h_last leave.
template <class T, int K, bool WIDE, bool REV, bool APPLY>
__global__ __launch_bounds__(256) void k_scan_fwd(const T* __restrict__ x, int64_t ldx, const T* __restrict__ gate, int64_t ldg, Segs g,
                                                  int64_t D, const float* __restrict__ h0, int CG, TileAgg agg,
                                                  const float* __restrict__ heads, T* __restrict__ h, int64_t ldh,
                                                  float* __restrict__ h_last) {
    __shared__ int32_t first[kTileElems / 8], last[kTileElems / 8];
    __shared__ float sA[256][4], sB[256][4];
    __shared__ int32_t sCut[32];
    const int RG = 256 / CG, cg = threadIdx.x & (CG - 1), rg = threadIdx.x / CG, rows = RG * K;
    const int64_t tile = blockIdx.x, row0 = tile * rows, c0 = (int64_t)blockIdx.y * (CG * 4), c = WIDE ? c0 + cg * 4 : c0 + cg;
    const int64_t r0 = row0 + rg * K;
    float a[K][4], b[K][4];
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int64_t r = r0 + i, p = REV ? g.N - 1 - r : r;
#pragma unroll
        for (int e = 0; e < 4; ++e) a[i][e] = b[i][e] = 0.f;
        if (r < g.N) {
            ld4<T, WIDE>(gate + p * ldg, c, CG, D, a[i]);
            ld4<T, WIDE>(x + p * ldx, c, CG, D, b[i]);
        }
    }
    mark_tile<REV>(g, row0, rows, first, last);
    float A[4] = {1.f, 1.f, 1.f, 1.f}, B[4] = {0.f, 0.f, 0.f, 0.f};
    uint32_t cuts = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int f = first[rg * K + i];
        float hs[4] = {0.f, 0.f, 0.f, 0.f};
        if (f >= 0 && h0) ld4<float, false>(h0 + f * D, c, WIDE ? 1 : CG, D, hs);
        if (f != -1) cuts |= 1u << i;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float ae, ce;
            gate_pair(a[i][e], ae, ce);
            float be = ce * b[i][e];
            if (f >= 0) be = fmaf(ae, hs[e], be);
            if (f == -2) be = 0.f;
            a[i][e] = ae;
            b[i][e] = be;
            B[e] = f != -1 ? be : fmaf(ae, B[e], be);
            A[e] *= ae;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) { sA[threadIdx.x][e] = A[e]; sB[threadIdx.x][e] = B[e]; }
    if (cg == 0) sCut[rg] = cuts != 0;
    __syncthreads();
    if (!APPLY) {
        if (rg == 0) write_agg<false>(sA, sB, sCut, cg, CG, RG, agg, tile, c0, D, WIDE);
        return;
    }
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    ld4<float, false>(heads + tile * D, c, WIDE ? 1 : CG, D, s);
    enter_group<false>(sA, sB, sCut, cg, rg, CG, RG, s);
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int64_t r = r0 + i, p = REV ? g.N - 1 - r : r;
        const bool cut = (cuts >> i) & 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = cut ? b[i][e] : fmaf(a[i][e], s[e], b[i][e]);
        if (r < g.N) {
            st4<T, WIDE>(h + p * ldh, c, CG, D, s);
            const int l = last[rg * K + i];
            if (l >= 0 && h_last) st4<float, false>(h_last + l * D, c, WIDE ? 1 : CG, D, s);
        }
    }
    if (h_last)                                                          // segments without rows: the state passes through
        for (int64_t k = tile; k < g.S; k += gridDim.x)
            if (seg_lo<REV>(g, k) >= seg_lo<REV>(g, k + 1) && rg == 0) {
                const int64_t sg = REV ? g.S - 1 - k : k;
                float v[4] = {0.f, 0.f, 0.f, 0.f};
                if (h0) ld4<float, false>(h0 + sg * D, c, WIDE ? 1 : CG, D, v);
                st4<float, false>(h_last + sg * D, c, WIDE ? 1 : CG, D, v);
            }
}

// ------------------------------------------------------------------------------------------------ states between the tiles
// heads[tile] = the state that enters the tile (from below, or from above with UP).  A workgroup: 32 columns, the tiles in
// 32 slices of consecutive ones.
template <bool UP>
__global__ __launch_bounds__(kCarryCols* kCarrySlices) void k_scan_carry(TileAgg agg, int64_t n_tiles, int64_t D, float* __restrict__ heads) {
    __shared__ float sA[kCarrySlices][kCarryCols], sB[kCarrySlices][kCarryCols];
    __shared__ int32_t sCut[kCarrySlices];
    const int tx = threadIdx.x % kCarryCols, ty = threadIdx.x / kCarryCols;
    const int64_t c = (int64_t)blockIdx.x * kCarryCols + tx, per = (n_tiles + kCarrySlices - 1) / kCarrySlices;
    const int64_t i0 = ty * per < n_tiles ? ty * per : n_tiles, i1 = i0 + per < n_tiles ? i0 + per : n_tiles;
    float A = 1.f, B = 0.f;
    int any = 0;
    if (c < D)
#pragma unroll 8
        for (int64_t i = i0; i < i1; ++i) {
            const int64_t t = UP ? n_tiles - 1 - i : i;
            const float a = agg.ab[2 * t * D + c], b = agg.ab[(2 * t + 1) * D + c];
            const bool cut = agg.cut[t] != 0;
            any |= cut;
            B = cut ? b : fmaf(a, B, b);
            A = cut ? 0.f : a * A;
        }
    sA[ty][tx] = A;
    sB[ty][tx] = B;
    if (tx == 0) sCut[ty] = any;
    __syncthreads();
    float s = 0.f;
    for (int k = 0; k < ty; ++k) s = sCut[k] ? sB[k][tx] : fmaf(sA[k][tx], s, sB[k][tx]);
    if (c < D)
#pragma unroll 8
        for (int64_t i = i0; i < i1; ++i) {
            const int64_t t = UP ? n_tiles - 1 - i : i;
            const float a = agg.ab[2 * t * D + c], b = agg.ab[(2 * t + 1) * D + c];
            heads[t * D + c] = s;
            s = agg.cut[t] ? b : fmaf(a, s, b);
        }
}

// ------------------------------------------------------------------------------------------------ backward
// APPLY false: the tile's map of mu -> agg.  APPLY true: heads (h below the tile) and tails (mu above it) enter.
template <class T, int K, bool WIDE, bool REV, bool APPLY>
__global__ __launch_bounds__(512) void k_scan_bwd(const T* __restrict__ x, int64_t ldx, const T* __restrict__ gate, int64_t ldg,
                                                  const T* __restrict__ dh, int64_t lddh, const float* __restrict__ dlast, Segs g,
                                                  int64_t D, const float* __restrict__ h0, int CG, TileAgg agg,
                                                  const float* __restrict__ heads, const float* __restrict__ tails, T* __restrict__ dx,
                                                  int64_t lddx, T* __restrict__ dgate, int64_t lddg, float* __restrict__ dh0) {
    __shared__ int32_t first[kTileElems / 8], last[kTileElems / 8];
    __shared__ float sA[512][4], sB[512][4];
    __shared__ int32_t sCut[64];
    const int RG = 512 / CG, cg = threadIdx.x & (CG - 1), rg = threadIdx.x / CG, rows = RG * K;
    const int64_t tile = blockIdx.x, row0 = tile * rows, c0 = (int64_t)blockIdx.y * (CG * 4), c = WIDE ? c0 + cg * 4 : c0 + cg;
    const int64_t r0 = row0 + rg * K;
    float a[K][4], cc[K][4], xx[K][4], d[K][4];
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int64_t r = r0 + i, p = REV ? g.N - 1 - r : r;
#pragma unroll
        for (int e = 0; e < 4; ++e) a[i][e] = xx[i][e] = d[i][e] = 0.f;
        if (r < g.N) {
            ld4<T, WIDE>(gate + p * ldg, c, CG, D, a[i]);
            if (dh) ld4<T, WIDE>(dh + p * lddh, c, CG, D, d[i]);
            if (APPLY) ld4<T, WIDE>(x + p * ldx, c, CG, D, xx[i]);
        }
    }
    mark_tile<REV>(g, row0, rows, first, last);
    uint32_t fcuts = 0, lcuts = 0, none = 0;
    float A[4] = {1.f, 1.f, 1.f, 1.f}, B[4] = {0.f, 0.f, 0.f, 0.f}, M[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = K - 1; i >= 0; --i) {
        const int f = first[rg * K + i], l = last[rg * K + i];
        float ds[4] = {0.f, 0.f, 0.f, 0.f};
        if (l >= 0 && dlast) ld4<float, false>(dlast + l * D, c, WIDE ? 1 : CG, D, ds);
        if (f != -1) fcuts |= 1u << i;
        if (f == -2) none |= 1u << i;
        if (l >= 0 || f == -2) lcuts |= 1u << i;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            gate_pair(a[i][e], a[i][e], cc[i][e]);
            if (l >= 0) d[i][e] += ds[e];
            if (f == -2) d[i][e] = 0.f;
            A[e] *= a[i][e];
            M[e] = a[i][e] * (l >= 0 || f == -2 ? d[i][e] : d[i][e] + M[e]);
        }
    }
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    float hp[K][4];
    if (APPLY) {
        // h before every row, from the state at the tile's head
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int f = first[rg * K + i];
            float hs[4] = {0.f, 0.f, 0.f, 0.f};
            if (f >= 0 && h0) ld4<float, false>(h0 + f * D, c, WIDE ? 1 : CG, D, hs);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hp[i][e] = hs[e];
                B[e] = fmaf(a[i][e], f == -1 ? B[e] : hs[e], cc[i][e] * xx[i][e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) { sA[threadIdx.x][e] = A[e]; sB[threadIdx.x][e] = B[e]; }
        if (cg == 0) sCut[rg] = fcuts != 0;
        __syncthreads();
        ld4<float, false>(heads + tile * D, c, WIDE ? 1 : CG, D, s);
        enter_group<false>(sA, sB, sCut, cg, rg, CG, RG, s);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const bool cut = (fcuts >> i) & 1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!cut) hp[i][e] = s[e];
                s[e] = fmaf(a[i][e], hp[i][e], cc[i][e] * xx[i][e]);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) { sA[threadIdx.x][e] = A[e]; sB[threadIdx.x][e] = M[e]; }
    if (cg == 0) sCut[rg] = lcuts != 0;
    __syncthreads();
    if (!APPLY) {
        if (rg == 0) write_agg<true>(sA, sB, sCut, cg, CG, RG, agg, tile, c0, D, WIDE);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = 0.f;
    ld4<float, false>(tails + tile * D, c, WIDE ? 1 : CG, D, s);
    enter_group<true>(sA, sB, sCut, cg, rg, CG, RG, s);
#pragma unroll
    for (int i = K - 1; i >= 0; --i) {
        const int64_t r = r0 + i, p = REV ? g.N - 1 - r : r;
        const bool cut = (lcuts >> i) & 1, out = (none >> i) & 1;
        float ox[4], og[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float lam = cut ? d[i][e] : d[i][e] + s[e];
            ox[e] = out ? 0.f : cc[i][e] * lam;
            og[e] = out ? 0.f : lam * (hp[i][e] - xx[i][e]) * (a[i][e] * cc[i][e]);
            s[e] = a[i][e] * lam;
        }
        if (r < g.N) {
            st4<T, WIDE>(dx + p * lddx, c, CG, D, ox);
            st4<T, WIDE>(dgate + p * lddg, c, CG, D, og);
            const int f = first[rg * K + i];
            if (f >= 0 && dh0) st4<float, false>(dh0 + f * D, c, WIDE ? 1 : CG, D, s);
        }
    }
    if (dh0)
        for (int64_t k = tile; k < g.S; k += gridDim.x)
            if (seg_lo<REV>(g, k) >= seg_lo<REV>(g, k + 1) && rg == 0) {
                const int64_t sg = REV ? g.S - 1 - k : k;
                float v[4] = {0.f, 0.f, 0.f, 0.f};
                if (dlast) ld4<float, false>(dlast + sg * D, c, WIDE ? 1 : CG, D, v);
                st4<float, false>(dh0 + sg * D, c, WIDE ? 1 : CG, D, v);
            }
}

// ------------------------------------------------------------------------------------------------ one row per segment
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void k_scan_step(const T* __restrict__ x, int64_t ldx, const T* __restrict__ gate, int64_t ldg,
                                                   const float* state, int64_t lds_, int64_t D, T* __restrict__ h, int64_t ldh,
                                                   float* state_out, int64_t ldso) {
    const int64_t row = blockIdx.x;
    const int64_t c0 = (int64_t)blockIdx.y * (WIDE ? 1024 : 256) + threadIdx.x * (WIDE ? 4 : 1);
    if (c0 >= D) return;
    constexpr int W = WIDE ? 4 : 1;
    const BgVec<T, W> xv = *reinterpret_cast<const BgVec<T, W>*>(x + row * ldx + c0);
    const BgVec<T, W> gv = *reinterpret_cast<const BgVec<T, W>*>(gate + row * ldg + c0);
    BgVec<float, W> sv = *reinterpret_cast<const BgVec<float, W>*>(state + row * lds_ + c0);
    BgVec<T, W> hv;
#pragma unroll
    for (int e = 0; e < W; ++e) {
        float a, c;
        gate_pair((float)gv.v[e], a, c);
        sv.v[e] = fmaf(a, sv.v[e], c * (float)xv.v[e]);
        hv.v[e] = bg_round<T>(sv.v[e]);
    }
    *reinterpret_cast<BgVec<T, W>*>(h + row * ldh + c0) = hv;
    *reinterpret_cast<BgVec<float, W>*>(state_out + row * ldso + c0) = sv;
}

// ------------------------------------------------------------------------------------------------ host side
int column_groups(int64_t D) { return D > 64 ? 32 : D > 32 ? 16 : 8; }
int64_t tile_rows(int64_t D) { return kTileElems / column_groups(D); }
int64_t tiles_of(int64_t n, int64_t D) { return (n + tile_rows(D) - 1) / tile_rows(D); }

template <class T>
bool piece_ok(const void* p, int64_t ld, int64_t D) {
    return D % 4 == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0;
}

int check_scan(int dtype, int64_t n, int64_t D, int64_t S, const int32_t* rowptr) {
    if (!bg_elem_size(dtype) || n < 0 || D < 0 || S < 0) return BG_ERR_ARG;
    if (!rowptr && (S == 0 ? n != 0 : n % S != 0)) return BG_ERR_ARG;
    if (n > INT32_MAX || S >= INT32_MAX || D > (1 << 20) || tiles_of(n, D) * 512 > UINT32_MAX) return BG_ERR_SHAPE;
    return BG_OK;
}

struct ScanWs { int64_t ab, cut, heads, bytes; };
ScanWs scan_ws(int64_t n, int64_t D) {
    const int64_t t = tiles_of(n, D);
    ScanWs w;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    w.ab = take(8 * t * D);
    w.cut = take(4 * t);
    w.heads = take(4 * t * D);
    w.bytes = at;
    return w;
}

template <class T, bool WIDE, bool REV>
void launch_scan_fwd(const T* x, int64_t ldx, const T* gate, int64_t ldg, Segs g, int64_t D, const float* h0, TileAgg agg, float* heads,
                     T* h, int64_t ldh, float* h_last, hipStream_t s) {
    const int CG = column_groups(D);
    const int64_t tiles = tiles_of(g.N, D);
    const dim3 grid((unsigned)tiles, (unsigned)((D + 4 * CG - 1) / (4 * CG)));
    k_scan_fwd<T, 16, WIDE, REV, false><<<grid, 256, 0, s>>>(x, ldx, gate, ldg, g, D, h0, CG, agg, nullptr, h, ldh, h_last);
    k_scan_carry<false><<<(unsigned)((D + kCarryCols - 1) / kCarryCols), kCarryCols * kCarrySlices, 0, s>>>(agg, tiles, D, heads);
    k_scan_fwd<T, 16, WIDE, REV, true><<<grid, 256, 0, s>>>(x, ldx, gate, ldg, g, D, h0, CG, agg, heads, h, ldh, h_last);
}
template <class T, bool WIDE, bool REV>
void launch_scan_bwd(const T* x, int64_t ldx, const T* gate, int64_t ldg, const T* dh, int64_t lddh, const float* dlast, Segs g, int64_t D,
                     const float* h0, TileAgg agg, const float* heads, float* tails, T* dx, int64_t lddx, T* dgate, int64_t lddg,
                     float* dh0, hipStream_t s) {
    const int CG = column_groups(D);
    const int64_t tiles = tiles_of(g.N, D);
    const dim3 grid((unsigned)tiles, (unsigned)((D + 4 * CG - 1) / (4 * CG)));
    k_scan_bwd<T, 8, WIDE, REV, false><<<grid, 512, 0, s>>>(x, ldx, gate, ldg, dh, lddh, dlast, g, D, h0, CG, agg, heads, tails, dx, lddx,
                                                            dgate, lddg, dh0);
    k_scan_carry<true><<<(unsigned)((D + kCarryCols - 1) / kCarryCols), kCarryCols * kCarrySlices, 0, s>>>(agg, tiles, D, tails);
    k_scan_bwd<T, 8, WIDE, REV, true><<<grid, 512, 0, s>>>(x, ldx, gate, ldg, dh, lddh, dlast, g, D, h0, CG, agg, heads, tails, dx, lddx,
                                                           dgate, lddg, dh0);
}

__global__ __launch_bounds__(256) void k_copy_or_zero(const float* __restrict__ src, float* __restrict__ dst, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) dst[i] = src ? src[i] : 0.f;
}

}  // namespace

extern "C" int64_t bg_gated_scan_heads(int64_t n_rows, int64_t D) { return n_rows > 0 && D > 0 ? tiles_of(n_rows, D) * D : 0; }

extern "C" int64_t bg_gated_scan_workspace(int64_t n_rows, int64_t D) { return n_rows > 0 && D > 0 ? scan_ws(n_rows, D).bytes : 0; }

extern "C" int bg_gated_scan_fwd(int dtype, const void* x, int64_t ldx, const void* gate, int64_t ldg, const int32_t* rowptr, int64_t n_seg,
                                 int64_t n_rows, int64_t D, const float* h0, int reverse, void* h, int64_t ldh, float* h_last,
                                 float* heads, void* ws, int64_t ws_bytes, bgStream stream) {
    const int rc = check_scan(dtype, n_rows, D, n_seg, rowptr);
    if (rc != BG_OK) return rc;
    if (ldx < D || ldg < D || ldh < D) return BG_ERR_ARG;
    if (D == 0) return BG_OK;
    hipStream_t s = (hipStream_t)stream;
    if (n_rows == 0) {                                     // no rows: the states pass through
        if (!h_last || n_seg == 0) return BG_OK;
        k_copy_or_zero<<<bg_grid_for(n_seg * D, 256, 4096), 256, 0, s>>>(h0, h_last, n_seg * D);
        BG_LAUNCH_CHECK();
        return BG_OK;
    }
    if (!x || !gate || !h || !ws) return BG_ERR_ARG;
    if (!bg_aligned16(ws)) return BG_ERR_ALIGN;
    const ScanWs w = scan_ws(n_rows, D);
    if (ws_bytes < w.bytes) return BG_ERR_SCRATCH;
    char* base = static_cast<char*>(ws);
    const TileAgg agg{reinterpret_cast<float*>(base + w.ab), reinterpret_cast<int32_t*>(base + w.cut)};
    float* hd = heads ? heads : reinterpret_cast<float*>(base + w.heads);
    const Segs g{rowptr, n_seg, n_rows, rowptr ? 0 : n_rows / n_seg};
    return bg_dispatch_dtype(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        const T *xx = static_cast<const T*>(x), *gg = static_cast<const T*>(gate);
        T* hh = static_cast<T*>(h);
        const bool wide = piece_ok<T>(x, ldx, D) && piece_ok<T>(gate, ldg, D) && piece_ok<T>(h, ldh, D);
        auto go = [&](auto W, auto R) { launch_scan_fwd<T, decltype(W)::value, decltype(R)::value>(xx, ldx, gg, ldg, g, D, h0, agg, hd, hh, ldh, h_last, s); };
        if (wide) reverse ? go(std::true_type(), std::true_type()) : go(std::true_type(), std::false_type());
        else reverse ? go(std::false_type(), std::true_type()) : go(std::false_type(), std::false_type());
        BG_LAUNCH_CHECK();
        return BG_OK;
    });
}

extern "C" int bg_gated_scan_bwd(int dtype, const void* x, int64_t ldx, const void* gate, int64_t ldg, const void* dh, int64_t lddh,
                                 const float* dlast, const int32_t* rowptr, int64_t n_seg, int64_t n_rows, int64_t D, const float* h0,
                                 int reverse, const float* heads, void* dx, int64_t lddx, void* dgate, int64_t lddg, float* dh0, void* ws,
                                 int64_t ws_bytes, bgStream stream) {
    const int rc = check_scan(dtype, n_rows, D, n_seg, rowptr);
    if (rc != BG_OK) return rc;
    if (ldx < D || ldg < D || (dh && lddh < D) || lddx < D || lddg < D) return BG_ERR_ARG;
    if (D == 0) return BG_OK;
    hipStream_t s = (hipStream_t)stream;
    if (n_rows == 0) {
        if (!dh0 || n_seg == 0) return BG_OK;
        k_copy_or_zero<<<bg_grid_for(n_seg * D, 256, 4096), 256, 0, s>>>(dlast, dh0, n_seg * D);
        BG_LAUNCH_CHECK();
        return BG_OK;
    }
    if (!x || !gate || !heads || !dx || !dgate || !ws) return BG_ERR_ARG;
    if (!bg_aligned16(ws)) return BG_ERR_ALIGN;
    const ScanWs w = scan_ws(n_rows, D);
    if (ws_bytes < w.bytes) return BG_ERR_SCRATCH;
    char* base = static_cast<char*>(ws);
    const TileAgg agg{reinterpret_cast<float*>(base + w.ab), reinterpret_cast<int32_t*>(base + w.cut)};
    float* tails = reinterpret_cast<float*>(base + w.heads);
    const Segs g{rowptr, n_seg, n_rows, rowptr ? 0 : n_rows / n_seg};
    return bg_dispatch_dtype(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        const T *xx = static_cast<const T*>(x), *gg = static_cast<const T*>(gate), *dd = static_cast<const T*>(dh);
        T *ox = static_cast<T*>(dx), *og = static_cast<T*>(dgate);
        const bool wide = piece_ok<T>(x, ldx, D) && piece_ok<T>(gate, ldg, D) && (!dh || piece_ok<T>(dh, lddh, D)) &&
                          piece_ok<T>(dx, lddx, D) && piece_ok<T>(dgate, lddg, D);
        auto go = [&](auto W, auto R) {
            launch_scan_bwd<T, decltype(W)::value, decltype(R)::value>(xx, ldx, gg, ldg, dd, lddh, dlast, g, D, h0, agg, heads, tails, ox,
                                                                       lddx, og, lddg, dh0, s);
        };
        if (wide) reverse ? go(std::true_type(), std::true_type()) : go(std::true_type(), std::false_type());
        else reverse ? go(std::false_type(), std::true_type()) : go(std::false_type(), std::false_type());
        BG_LAUNCH_CHECK();
        return BG_OK;
    });
}

extern "C" int bg_gated_scan_step(int dtype, const void* x, int64_t ldx, const void* gate, int64_t ldg, const float* state, int64_t lds,
                                  int64_t n, int64_t D, void* h, int64_t ldh, float* state_out, int64_t ldso, bgStream stream) {
    if (!bg_elem_size(dtype) || n < 0 || D < 0 || ldx < D || ldg < D || lds < D || ldh < D || ldso < D) return BG_ERR_ARG;
    if (n == 0 || D == 0) return BG_OK;
    if (!x || !gate || !state || !h || !state_out) return BG_ERR_ARG;
    if (n * 256 > UINT32_MAX || D > (1 << 20)) return BG_ERR_SHAPE;
    return bg_dispatch_dtype(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        const T *xx = static_cast<const T*>(x), *gg = static_cast<const T*>(gate);
        T* hh = static_cast<T*>(h);
        const bool wide = piece_ok<T>(x, ldx, D) && piece_ok<T>(gate, ldg, D) && piece_ok<T>(h, ldh, D) && piece_ok<float>(state, lds, D) &&
                          piece_ok<float>(state_out, ldso, D);
        const dim3 grid((unsigned)n, (unsigned)((D + (wide ? 1023 : 255)) / (wide ? 1024 : 256)));
        if (wide) k_scan_step<T, true><<<grid, 256, 0, (hipStream_t)stream>>>(xx, ldx, gg, ldg, state, lds, D, hh, ldh, state_out, ldso);
        else k_scan_step<T, false><<<grid, 256, 0, (hipStream_t)stream>>>(xx, ldx, gg, ldg, state, lds, D, hh, ldh, state_out, ldso);
        BG_LAUNCH_CHECK();
        return BG_OK;
    });
}
